// What the decoding kernels over a paged cache share: how the keys of a call's
// sequences are divided into parts, how a workgroup's waves are joined, and how
// the parts are. (attn_decode.hip: caches of float32, bf16 and float16;
// attn_fp4.hip: caches of 4-bit values.)
#pragma once

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

constexpr int DEC_WAVES = 4;         // waves of a workgroup
constexpr int DEC_KEYS = 32;         // keys of a block
constexpr int DEC_MIN = DEC_WAVES;   // fewest blocks of a part: one a wave
constexpr int DEC_ROWS = 16;         // rows of a matrix tile

struct DecodeParams {
  const unsigned char *q, *k, *v;
  long token, head;  // strides of the caches, bytes
  int page_rows;     // a page's stride in token strides
  int page, num_pages, max_pages;
  const int32_t *table, *lengths;
  void *o;
  float *lse;
  float *part;     // [slots][Hk][rows][D] unnormalised outputs
  float2 *stat;    // [slots][Hk][rows] (largest score, sum)
  int B, T, Hq, Hk, group, rows, row_tiles, window, sinks, target;
  float c;
  int negate;
};

// The keys sequence b's queries see, and its blocks.
__device__ __forceinline__ int seq_length(const DecodeParams &p, int b) {
  const int n = p.num_pages > 0 ? p.lengths[b] : 0;
  return n > 0 ? n : 0;
}
__device__ __forceinline__ KeyRange seq_keys(const DecodeParams &p, int len) {
  return key_range(len - p.T, len - 1, p.window, p.sinks);
}
__device__ __forceinline__ int len_blocks(const DecodeParams &p, int len) {
  return (seq_keys(p, len).count + DEC_KEYS - 1) / DEC_KEYS;
}
__device__ __forceinline__ int seq_blocks(const DecodeParams &p, int b) { return len_blocks(p, seq_length(p, b)); }

// The shares: every part takes `per` blocks (the last of a sequence what is
// left), a sequence at least one part. Every wave works them out for itself: the
// first 256 sequences' blocks, four a lane, are read once and together.
__device__ __forceinline__ int wave_sum_int(int x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
__device__ __forceinline__ long wave_sum_long(long x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
struct Shares {
  static constexpr int HELD = 4;
  int held[HELD];  // blocks of sequences 64 i + lane
  int per;

  __device__ __forceinline__ Shares(const DecodeParams &p, int lane) {
    if (p.B == 1) {  // one request: nothing to add up over the lanes
      held[0] = seq_blocks(p, 0);
      share(p, held[0]);
      return;
    }
    long total = 0;
    int len[HELD];  // (read by every lane, so that the four reads are in flight together)
#pragma unroll
    for (int i = 0; i < HELD; ++i) len[i] = p.lengths[64 * i + lane < p.B ? 64 * i + lane : p.B - 1];
#pragma unroll
    for (int i = 0; i < HELD; ++i) settle(len[i]);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const bool any = (64 * i + lane < p.B) & (p.num_pages > 0) & (len[i] > 0);
      held[i] = any ? len_blocks(p, len[i]) : 0;
      total += held[i];
    }
    for (int b = 64 * HELD + lane; b < p.B; b += 64) total += seq_blocks(p, b);
    share(p, wave_sum_long(total));
  }
  __device__ __forceinline__ void share(const DecodeParams &p, long total) {
    const int even = total <= 0x7fffffff - p.target
                         ? (static_cast<int>(total) + p.target - 1) / p.target
                         : static_cast<int>((total + p.target - 1) / p.target);
    const int whole = (even + DEC_MIN - 1) / DEC_MIN * DEC_MIN;
    per = uniform(whole > DEC_MIN ? whole : DEC_MIN);
  }
  __device__ __forceinline__ int parts(int blocks) const { return blocks > per ? (blocks + per - 1) / per : 1; }

  // Sequence b's parts, and its first slot.
  __device__ __forceinline__ int parts_of(const DecodeParams &p, int b, int) const { return uniform(parts(seq_blocks(p, b))); }
  __device__ __forceinline__ int first_of(const DecodeParams &p, int b, int lane) const {
    int first = 0;
    if (b > 0) {
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (64 * i + lane < b) first += parts(held[i]);
      for (int i = 64 * HELD + lane; i < b; i += 64) first += parts(seq_blocks(p, i));
      first = uniform(wave_sum_int(first));
    }
    return first;
  }
};
// Whose slot it is: a scan over the sequences, 64 at a time. seq = -1 past the last.
struct Share {
  int seq, part, parts, per;
};
__device__ __forceinline__ Share share_of_slot(const DecodeParams &p, int slot, int lane) {
  const Shares all(p, lane);
  Share s{-1, 0, 0, all.per};
  if (p.B == 1) {
    s.parts = all.parts(all.held[0]);
    s.part = slot;
    s.seq = slot < s.parts ? 0 : -1;
    return s;
  }
  int base = 0;
  const auto look = [&](int b0, int blocks) __attribute__((always_inline)) {
    const int mine = b0 + lane < p.B ? all.parts(blocks) : 0;
    int scan = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(scan, off, 64);
      if (lane >= off) scan += x;
    }
    const uint64_t past = __ballot(base + scan > slot);
    if (past) {
      const int l = __builtin_ctzll(past);
      s.seq = b0 + l;
      s.parts = __shfl(mine, l, 64);
      s.part = slot - (base + __shfl(scan, l, 64) - s.parts);
    }
    base += __shfl(scan, 63, 64);
    return past != 0;
  };
#pragma unroll
  for (int i = 0; i < Shares::HELD; ++i) {
    if (64 * i >= p.B || look(64 * i, all.held[i])) return s;
  }
  for (int b0 = 64 * Shares::HELD; b0 < p.B; b0 += 64)
    if (look(b0, b0 + lane < p.B ? seq_blocks(p, b0 + lane) : 0)) break;
  return s;
}

// max / sum over the four lanes (one of each 16) that hold a row.
__device__ __forceinline__ float max_rows(float x) {
  float a = x, b = x;
  swap16(a, b);
  a = fmaxf(a, b);
  b = a;
  swap32(a, b);
  return fmaxf(a, b);
}
// The waves' running sums o (scores' maxima m, weights' sums l) into wave 0's: the
// upper half into the lower, or one by one where JOINS is 1. With HEADS = 2 the waves of
// each parity are a head's of their own and end in waves 0 and 1. Element 4 g + i of o's
// columns j lies in element i of o[.][j]; every lane of a column holds m and l.
template <int RB, int D, int JOINS, int HEADS = 1>
__device__ __forceinline__ void join_waves(float (&merge)[JOINS][RB * DEC_ROWS * (D + 2)], float (&m)[RB], float (&l)[RB],
                                           float4_t (&o)[RB][D / 16], int wave, int lane, float pc) {
  constexpr int OT = D / 16;
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int r = 0; r < RB; ++r) l[r] = add_xor32(add_xor16(l[r]));
  static_assert(HEADS == 1 || (HEADS == 2 && JOINS == 2), "pairs of waves are joined");
  constexpr int ROUNDS = JOINS == 2 ? 3 - HEADS : DEC_WAVES - 1;
#pragma unroll
  for (int round = 0; round < ROUNDS; ++round) {
    const int from = JOINS == 2 ? DEC_WAVES / 2 >> round : round + 1, count = JOINS == 2 ? from : 1;
    if (wave >= from && wave < from + count) {
      float *dst = merge[wave - from];
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int j = 0; j < OT; ++j)
          *reinterpret_cast<float4_t *>(dst + ((r * OT + j) * 64 + lane) * 4) = o[r][j];
        if (g == 0) {
          dst[RB * DEC_ROWS * D + (r * 16 + c) * 2] = m[r];
          dst[RB * DEC_ROWS * D + (r * 16 + c) * 2 + 1] = l[r];
        }
      }
    }
    __syncthreads();
    if (wave < count) {
      const float *src = merge[wave];
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float m2 = src[RB * DEC_ROWS * D + (r * 16 + c) * 2], l2 = src[RB * DEC_ROWS * D + (r * 16 + c) * 2 + 1];
        const float top = fmaxf(m[r], m2), at = top == -INFINITY ? 0.0f : top;
        const float f1 = __builtin_amdgcn_exp2f((m[r] - at) * pc), f2 = __builtin_amdgcn_exp2f((m2 - at) * pc);
        m[r] = top;
        l[r] = l[r] * f1 + l2 * f2;
#pragma unroll
        for (int j = 0; j < OT; ++j)
          o[r][j] = o[r][j] * f1 + *reinterpret_cast<const float4_t *>(src + ((r * OT + j) * 64 + lane) * 4) * f2;
      }
    }
    __syncthreads();
  }
}

// Wave 0's rows: to the part's place, or, where it is the sequence's only one (last),
// divided by their sums to o and lse. Tile x VE + e of o holds columns VE (4 g + i) + e of
// the x-th run of 16 VE.
template <int DT, int D, int RB, int VE>
__device__ __forceinline__ void store_decoded(const DecodeParams &p, bool last, int b, int hk, int row0, int slot, int lane,
                                               const float (&m)[RB], const float (&l)[RB],
                                              const float4_t (&o)[RB][D / 16]) {
  using E = Elem<DT>;
  constexpr bool SHORT = E::BYTES == 2;
  constexpr int VLOADS = D / 16 / VE;
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + r * DEC_ROWS + c;
    if (row >= p.rows) continue;
    const float f = last && l[r] > 0.0f ? 1.0f / l[r] : 1.0f;
    const long at = last ? (static_cast<long>(b) * p.T + row / p.group) * p.Hq + hk * p.group + row % p.group
                         : (static_cast<long>(slot) * p.Hk + hk) * p.rows + row;
    if (g == 0) {
      if (!last) {
        p.stat[at] = make_float2(m[r], l[r]);
      } else if (p.lse) {
        p.lse[at] = row_lse(m[r], l[r], p.c);
      }
    }
    // element j of the lane's i-th matrix row: column VE (4 g + i) + j of a run of 16 VE
#pragma unroll
    for (int x = 0; x < VLOADS; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VE; e += 4) {
          const long d = at * D + x * 16 * VE + (4 * g + i) * VE + e;
          const float4_t y = {o[r][x * VE + e][i] * f, o[r][x * VE + e + 1][i] * f,
                              o[r][x * VE + e + 2][i] * f, o[r][x * VE + e + 3][i] * f};
          if (!last || !SHORT) {
            *reinterpret_cast<float4_t *>((last ? static_cast<float *>(p.o) : p.part) + d) = y;
          } else if constexpr (SHORT) {
            *reinterpret_cast<v2u32_t *>(static_cast<unsigned char *>(p.o) + 2 * d) =
                v2u32_t{E::pack(y[0], y[1]), E::pack(y[2], y[3])};
          }
        }
  }
}

// Joins a sequence's parts, SPLIT waves to a (sequence, query row and head),
// eight parts of a wave at a time: their outputs and their weights' statistics,
// one a lane, are fetched together. Four waves a row where there are few rows,
// one where there are many. A workgroup takes PER rows, as many of them at a time as it has
// waves for. Division says which parts they are.
template <int DT, int D, int SPLIT, int PER, typename Division>
static __global__ __launch_bounds__(256) void decode_join_kernel(const DecodeParams p) {
  constexpr int VEC = D / 64, ROWS = 4 / SPLIT, AT_ONCE = 8;  // ROWS: rows of a workgroup at a time
  static_assert(SPLIT == 1 || PER == ROWS, "a row's waves meet once");
  __shared__ float acc[SPLIT > 1 ? 4 : 1][D], stat[4][2];
  PBGDN_POISON_LDS(acc, sizeof(acc));
  PBGDN_POISON_SYNC();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), w = wave % SPLIT;
  const int tiles = (p.rows + PER - 1) / PER;
  int id = blockIdx.x;
  const int row0 = id % tiles * PER, row1 = row0 + PER < p.rows ? row0 + PER : p.rows;
  int row = row0 + wave / SPLIT;
  id /= tiles;
  const int hk = id % p.Hk, b = id / p.Hk;
  const Division all(p, lane);
  const int parts = all.parts_of(p, b, lane);
  if (parts == 1) return;  // written by the first kernel
  if (SPLIT == 1 && row >= row1) return;
  const int first = all.first_of(p, b, lane);
  do {
    float m = -INFINITY, l = 0.0f, o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = 0.0f;
    for (int i0 = w; i0 < parts; i0 += AT_ONCE * SPLIT) {  // this wave's parts: i0, i0 + SPLIT, ...
      const int count = (parts - i0 + SPLIT - 1) / SPLIT, n = count < AT_ONCE ? count : AT_ONCE;
      const long at0 = (static_cast<long>(first + i0) * p.Hk + hk) * p.rows + row;
      const long step = static_cast<long>(SPLIT) * p.Hk * p.rows;
      float x[AT_ONCE][VEC];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float *src = p.part + (at0 + (i < n ? i : 0) * step) * D + lane * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[i][e] = src[e];
      }
      const float2 s = lane < n ? p.stat[at0 + lane * step] : make_float2(-INFINITY, 0.0f);
      const float top = fmaxf(m, wave_max(s.x)), base = top == -INFINITY ? 0.0f : top;
      const float f = __builtin_amdgcn_exp2f((s.x - base) * p.c), keep = __builtin_amdgcn_exp2f((m - base) * p.c);
      m = top;
      l = l * keep + wave_sum(s.y * f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] *= keep;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i));
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] += i < n ? x[i][e] * fi : 0.0f;
      }
    }
    if constexpr (SPLIT > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[wave][lane * VEC + e] = o[e];
      if (lane == 0) {
        stat[wave][0] = m;
        stat[wave][1] = l;
      }
      __syncthreads();
      if (wave != 0) return;
#pragma unroll
      for (int i = 1; i < SPLIT; ++i) m = fmaxf(m, stat[i][0]);
      const float base = m == -INFINITY ? 0.0f : m;
      l = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < SPLIT; ++i) {
        const float f = __builtin_amdgcn_exp2f((stat[i][0] - base) * p.c);
        l += stat[i][1] * f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] += acc[i][lane * VEC + e] * f;
      }
    }
    const float inv = l > 0.0f ? 1.0f / l : l;
    const long at = (static_cast<long>(b) * p.T + row / p.group) * p.Hq + hk * p.group + row % p.group;
#pragma unroll
    for (int e = 0; e < VEC; ++e) store_elem(p.o, at * D + lane * VEC + e, DT, o[e] * inv);
    if (p.lse && lane == 0) p.lse[at] = row_lse(m, l, p.c);
    row += ROWS;
  } while (PER > ROWS && row < row1);
}

constexpr long MAX_BLOCKS = 0xffffff;  // of 256 threads: a launch has less than 2^32

// Launches the join of parts (decode_join_kernel) for a call whose parts have been: four
// waves a row (`split`), or one, of which a workgroup takes ROWS, four at a time.
inline long join_blocks(const DecodeParams &p, bool split, int rows) {
  const int per = split ? 1 : rows;
  return static_cast<long>(p.B) * p.Hk * ((p.rows + per - 1) / per);
}
template <int DT, int D, int ROWS, typename Division>
static void launch_join(const DecodeParams &p, bool split, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(join_blocks(p, split, ROWS)));
  if (split)
    hipLaunchKernelGGL((decode_join_kernel<DT, D, 4, 1, Division>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((decode_join_kernel<DT, D, 1, ROWS, Division>), grid, dim3(256), 0, stream, p);
}

// The grid of a call's parts for kernels of rb row tiles a workgroup; 0 where it
// has more workgroups or rows than a launch takes.
inline unsigned decode_blocks(DecodeParams &p, int rb) {
  p.row_tiles = (p.rows + rb * DEC_ROWS - 1) / (rb * DEC_ROWS);
  const long blocks = (static_cast<long>(p.target) + p.B) * p.Hk * p.row_tiles;
  return blocks > MAX_BLOCKS || static_cast<long>(p.B) * p.Hk * p.rows > 0x7fffffffL ? 0u : static_cast<unsigned>(blocks);
}

inline bool decode_sizes_ok(int B, int T, int Hq, int Hk, int D) {
  return B >= 0 && T >= 1 && T <= PBATTN_MAX_DRAFT && Hq > 0 && Hk > 0 && Hq % Hk == 0 && D > 0;
}

// What a decoding call's arguments make of the parameters besides the caches' addresses
// and strides: `wanted` parts over all sequences, no more than the table's pages, or the
// window, can need.
inline void decode_call(DecodeParams &p, int B, int T, int Hq, int Hk, float scale, int window, int sinks, int wanted) {
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hk = Hk;
  p.group = Hq / Hk;
  p.rows = p.group * T;
  p.window = window <= 0 || window > NO_WINDOW ? NO_WINDOW : window;
  p.sinks = sinks < NO_WINDOW ? sinks : NO_WINDOW;
  long most = static_cast<long>(p.max_pages) * p.page;
  if (most > static_cast<long>(p.window) + T + p.sinks) most = static_cast<long>(p.window) + T + p.sinks;
  most = (most + DEC_MIN * DEC_KEYS - 1) / (DEC_MIN * DEC_KEYS) * B;
  p.target = most < wanted ? static_cast<int>(most > 1 ? most : 1) : wanted;
  const float c = __builtin_fabsf(scale) * LOG2E;
  p.c = c > 1.17549435e-38f ? c : 1.17549435e-38f;
  p.negate = scale < 0.0f;
}

// The workspace's places of the parts; its bytes.
inline size_t decode_workspace(DecodeParams &p, void *workspace, int D) {
  const size_t rows = (static_cast<size_t>(p.target) + p.B) * p.Hk * p.rows;
  p.part = static_cast<float *>(workspace);
  p.stat = reinterpret_cast<float2 *>(p.part + rows * D);
  return rows * (D * sizeof(float) + sizeof(float2));
}

}  // namespace pbgdn
