// Attention of the newest tokens over a paged cache (pbattn_paged_decode) and
// the cache's writes (pbattn_paged_write).
//
// Decoding reads every visible key and value once and computes little with
// them, so the kernel is built around loads: each wave takes blocks of 32 keys
// by itself, straight from the cache into the registers the matrix
// instructions read, with no LDS in between. Scores come from 16x16 products
// S^T = K Q^T whose 16 columns are the (token, head) rows that share the key
// head. For O^T = V^T P the wave loads 8 (16-bit) whole value rows such that
// each lane holds an 8 x 8 block of V, and transposes it in place.
//
// The visible blocks of all sequences are shared out evenly from the lengths:
// every workgroup derives the same shares, so a batch of uneven contexts needs
// neither a host's knowledge of the lengths nor a list made by another kernel.
//
// Bound by the cache's bytes: 64 contexts up to 16,384 tokens, 8 key heads of 128:
// 2.12 GB in 363 us (5.86 TB/s; reading alone reaches 5.8 here, a copy 4.7). 233
// contexts, window 4,096, 2 key heads of 256: 272 us for one token (5.35 TB/s), 334
// for four (4.4 TB/s), whose parts' sums, four times as many, cost 35 us of their
// own, 18 of them in decode_join_kernel. One context of 4,097 tokens: 8 and 4 us,
// less than the host's 13 to 15.
#include <type_traits>

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

constexpr int DEC_WAVES = 4;         // waves of a workgroup
constexpr int DEC_KEYS = 32;         // keys of a block
constexpr int DEC_MIN = DEC_WAVES;   // fewest blocks of a part: one a wave
constexpr int DEC_ROWS = 16;         // rows of a matrix tile
constexpr int JOIN_SPLIT_ROWS = 2048;  // up to here four waves join a row's parts

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

template <int DT, int D>
struct Dec {
  using E = Elem<DT>;
  static constexpr bool SHORT = E::BYTES == 2;
  static constexpr int ROW = D * E::BYTES;
  static constexpr int KSTEPS = ROW / 64;           // 16-byte units a lane reads of a key
  static constexpr int VB = SHORT && D == 64 ? 8 : 16;  // bytes a lane reads of a value row at once
  static constexpr int VLOADS = ROW / 16 / VB;      // times it does
  static constexpr int VE = VB / E::BYTES;          // elements of one such read
  static constexpr int OT = D / 16;                 // 16-wide output tiles: VLOADS * VE
  // Rows up to 256 bytes: 32 keys at a time. Wider ones 16, and Q in LDS where a
  // wave has two row blocks of it (its registers hold the sums, 16 keys and their
  // values): two waves a SIMD up to 512 bytes.
  static constexpr int KG = ROW <= 256 ? 2 : 1;     // 16-key groups at a time
  static constexpr bool q_in_lds(int rb) { return ROW > 512 || (ROW == 512 && rb == 2); }
  static constexpr int OCC = ROW <= 512 ? 2 : 1;
};

// Scores of 16 keys: x += K rows (a lane's units) times Q rows.
template <int DT>
__device__ __forceinline__ float4_t key_mma(v4u32_t k, v4u32_t q, float4_t x) {
  if constexpr (DT == PBGDN_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[e]), x, 0, 0, 0);
    return x;
  } else {
    return Elem<DT>::mma16(k, q, x);
  }
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

template <int DT, int D, int RB>
__global__ __launch_bounds__(DEC_WAVES * 64, (Dec<DT, D>::OCC)) void decode_kernel(const DecodeParams p) {
  using K = Dec<DT, D>;
  using E = typename K::E;
  constexpr int KS = K::KSTEPS, OT = K::OT, KG = K::KG, KEYS = 16 * KG;
  constexpr bool Q_LDS = K::q_in_lds(RB);
  // waves joined at a time: pairs, or one after the other where two would not fit
  constexpr int JOINS = RB * D <= 256 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float merge[JOINS][RB * DEC_ROWS * (D + 2)];
  PBGDN_POISON_LDS(merge, sizeof(merge));
  PBGDN_POISON_SYNC();

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int slots = p.target + p.B, id = uniform(blockIdx.x / slots), slot = blockIdx.x - id * slots;
  const int row0 = uniform(id / p.Hk) * (RB * DEC_ROWS), hk = uniform(id % p.Hk);
  const Share share = share_of_slot(p, slot, lane);
  if (share.seq < 0) return;
  const int b = uniform(share.seq), len = uniform(seq_length(p, b));
  const KeyRange range = seq_keys(p, len);
  // this wave's KEYS-wide blocks of the part: begin + wave, then every DEC_WAVES-th
  const int blocks = (range.count + KEYS - 1) / KEYS;
  const int begin = uniform(share.part * share.per * (DEC_KEYS / KEYS));
  const int end_ = begin + share.per * (DEC_KEYS / KEYS);
  const int end = uniform(end_ < blocks ? end_ : blocks);

  // this lane's rows of Q (column c of every row block); in LDS, each wave brings in a share
  unsigned char *const ql = reinterpret_cast<unsigned char *>(&merge[0][0]);
  v4u32_t qf[Q_LDS ? 1 : RB][KS];
  int pos[RB];
  constexpr int QS = Q_LDS ? KS / DEC_WAVES : KS;  // steps of Q that a wave brings in
  const int q0 = Q_LDS ? wave * QS : 0;
  v4u32_t qs[Q_LDS ? RB : 1][QS];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + r * DEC_ROWS + c;
    const int rr = row < p.rows ? row : p.rows - 1;
    const int t = rr / p.group;
    pos[r] = len - p.T + t;
    const unsigned char *src = p.q + ((static_cast<long>(b) * p.T + t) * p.Hq + hk * p.group + rr - t * p.group) * K::ROW;
    v4u32_t *x = Q_LDS ? qs[r] : qf[r];
#pragma unroll
    for (int s = 0; s < QS; ++s) x[s] = *reinterpret_cast<const v4u32_t *>(src + (4 * (q0 + s) + g) * 16);
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    v4u32_t *x = Q_LDS ? qs[r] : qf[r];
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      if (p.negate) x[s] ^= K::SHORT ? 0x80008000u : 0x80000000u;
      if constexpr (Q_LDS)
        *reinterpret_cast<v4u32_t *>(ql + (r * DEC_ROWS + c) * K::ROW + ((4 * (q0 + s) + g) ^ c) * 16) = x[s];
    }
  }
  if constexpr (Q_LDS) __syncthreads();
  float m[RB], l[RB];
  float4_t o[RB][OT];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int j = 0; j < OT; ++j) o[r][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const unsigned char *kbase = p.k + hk * p.head, *vbase = p.v + hk * p.head;
  const int32_t *table = p.table + static_cast<long>(b) * p.max_pages;
  // Key `lane` (modulo KEYS) of a block: its page, and its place there (-1: there is none); then its row in the cache.
  const auto lookup = [&](int blk, int &page, int &place) __attribute__((always_inline)) {
    const uint32_t u = static_cast<uint32_t>(blk) * KEYS + lane % KEYS, last = range.count - 1;  // (past a range's end too)
    const int v = static_cast<int>(u < last ? u : last), j = v < range.sinks ? v : v + range.delta;
    const int pg = j / p.page;
    page = table[pg < p.max_pages ? pg : p.max_pages - 1];
    place = ((u <= last) & (pg < p.max_pages)) ? j - pg * p.page : -1;
  };
  const auto cache_row = [&](int page, int place) __attribute__((always_inline)) {
    return ((place >= 0) & (page >= 0) & (page < p.num_pages)) ? page * p.page_rows + place : -1;
  };
  // The cache is read once: past the caches (non-temporal), 4 to 9% faster where
  // it is larger than they are.
  v4u32_t kf[KG][KS];
  uint32_t vf[4 * KG][K::VLOADS][K::VB / 4];
  const auto load_keys = [&](int rows) __attribute__((always_inline)) {
    const int safe = rows >= 0 ? rows : 0;
#pragma unroll
    for (int kb = 0; kb < KG; ++kb) {
      const unsigned char *src = kbase + static_cast<long>(__shfl(safe, 16 * kb + c, 64)) * p.token;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        kf[kb][s] = __builtin_nontemporal_load(reinterpret_cast<const v4u32_t *>(src + (4 * s + g) * 16));
    }
  };
  const auto load_values = [&](int rows) __attribute__((always_inline)) {
    const int safe = rows >= 0 ? rows : 0;
#pragma unroll
    for (int i = 0; i < 4 * KG; ++i) {
      const unsigned char *src = vbase + static_cast<long>(__shfl(safe, i / 4 * 16 + 4 * g + i % 4, 64)) * p.token;
#pragma unroll
      for (int x = 0; x < K::VLOADS; ++x) {
        if constexpr (K::VB == 16) {
          const v4u32_t w = __builtin_nontemporal_load(reinterpret_cast<const v4u32_t *>(src + x * 16 * K::VB + c * K::VB));
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[i][x][e] = w[e];
        } else {
          const v2u32_t w = __builtin_nontemporal_load(reinterpret_cast<const v2u32_t *>(src + x * 16 * K::VB + c * K::VB));
#pragma unroll
          for (int e = 0; e < 2; ++e) vf[i][x][e] = w[e];
        }
      }
    }
  };
  // A block's keys are fetched while the one before is weighed, its values while
  // the scores are formed: the registers of either are free again by then. The
  // pages of the block after are asked for before those values: loads come back
  // in order, and the next keys' addresses would otherwise wait for them all.
  int valid = -1, page = -1, place = -1;
  if (begin + wave < end) {
    lookup(begin + wave, page, place);
    valid = cache_row(page, place);
    lookup(begin + wave + DEC_WAVES, page, place);
    load_keys(valid);
    load_values(valid);
  }
  const auto step = [&](int blk, auto last) __attribute__((always_inline)) {
    constexpr bool more = !decltype(last)::value;
    const bool all = __ballot(valid >= 0) == ~0ull;
    float4_t sc[RB][KG];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < KG; ++kb) sc[r][kb] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t qat = opaque(c * K::ROW + (g ^ c) * 16);  // unit g of row c: unit 4 s + g is 64 s from it, by exclusive or
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        v4u32_t q;
        if constexpr (Q_LDS) {
          const uint32_t lo = (4 * k) % 16 * 16, hi = (4 * k) / 16 * 256;
          q = *reinterpret_cast<const v4u32_t *>(ql + r * DEC_ROWS * K::ROW + (qat ^ lo) + hi);
        } else {
          q = qf[r][k];
        }
#pragma unroll
        for (int kb = 0; kb < KG; ++kb) sc[r][kb] = key_mma<DT>(kf[kb][k], q, sc[r][kb]);
      }
    if constexpr (!K::SHORT && !more) {
      // nothing stands between the last products and the reads of their results, which the
      // compiler may put closer than the ten cycles they take to be there
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_nop 1");
    }
    const int next = more ? cache_row(page, place) : -1;
    if constexpr (more) load_keys(next);
    if (!all) {  // values of absent keys: zeros, whatever the row they were read from holds
#pragma unroll
      for (int i = 0; i < 4 * KG; ++i) {
        const bool in = __shfl(valid, i / 4 * 16 + 4 * g + i % 4, 64) >= 0;
#pragma unroll
        for (int x = 0; x < K::VLOADS; ++x)
#pragma unroll
          for (int e = 0; e < K::VB / 4; ++e) vf[i][x][e] = in ? vf[i][x][e] : 0u;
      }
    }
    const int u0 = blk * KEYS;
    const int j0 = u0 < range.sinks ? u0 : u0 + range.delta, j1 = u0 + KEYS - 1 + range.delta;
    const bool whole = all && u0 >= range.sinks && j1 <= len - p.T && j0 > len - 1 - p.window;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float4_t (&s)[KG] = sc[r];
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4 * KG; ++i) {
          const int key = i / 4 * 16 + 4 * g + i % 4, u = u0 + key;
          const int j = u < range.sinks ? u : u + range.delta;
          const bool seen = (__shfl(valid, key, 64) >= 0) & sees(pos[r], j, p.window, p.sinks);
          s[i / 4][i % 4] = seen ? s[i / 4][i % 4] : -INFINITY;
        }
      }
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 4 * KG; ++i) mx = fmaxf(mx, s[i / 4][i % 4]);
      mx = max_rows(mx);
      if (__any((mx - m[r]) * p.c > LAG)) {
        const float top = fmaxf(m[r], mx);
        const float alpha = __builtin_amdgcn_exp2f((m[r] - (top == -INFINITY ? 0.0f : top)) * p.c);
        m[r] = top;
        l[r] *= alpha;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[r][j] *= alpha;
      }
      const float base = m[r] == -INFINITY ? 0.0f : m[r], at = base * p.c;
      const bool far = __any(fabsf(at) > EXACT_SCORES);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * KG; ++i) {
        const float x = s[i / 4][i % 4];
        s[i / 4][i % 4] = __builtin_amdgcn_exp2f(far ? (x - base) * p.c : __builtin_fmaf(x, p.c, -at));
        sum += s[i / 4][i % 4];
      }
      l[r] += sum;
    }
    // O^T += V^T P; element e of the lane's value rows makes output tile x VE + e
    if constexpr (K::SHORT) {
      using Half = std::conditional_t<KG == 2, v4u32_t, v2u32_t>;
      Half w[RB];
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int i = 0; i < 2 * KG; ++i) w[r][i] = E::pack(sc[r][i / 2][2 * (i % 2)], sc[r][i / 2][2 * (i % 2) + 1]);
#pragma unroll
      for (int x = 0; x < K::VLOADS; ++x)
#pragma unroll
        for (int e = 0; e < K::VE; ++e) {
          Half a;
#pragma unroll
          for (int i = 0; i < 2 * KG; ++i)
            a[i] = __builtin_amdgcn_perm(vf[2 * i + 1][x][e / 2], vf[2 * i][x][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int r = 0; r < RB; ++r) o[r][x * K::VE + e] = E::mma16(a, w[r], o[r][x * K::VE + e]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * KG; ++i)
#pragma unroll
        for (int x = 0; x < K::VLOADS; ++x)
#pragma unroll
          for (int e = 0; e < K::VE; ++e)
#pragma unroll
            for (int r = 0; r < RB; ++r)
              o[r][x * K::VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __uint_as_float(vf[i][x][e]), sc[r][i / 4][i % 4], o[r][x * K::VE + e], 0, 0, 0);
    }
    if constexpr (more) {
      lookup(blk + 2 * DEC_WAVES, page, place);
      load_values(next);
      valid = next;
    }
  };
  // The last block apart: loads on some ways through the loop only would have its
  // values wait for the next keys.
  int blk = begin + wave;
  for (; blk + DEC_WAVES < end; blk += DEC_WAVES) step(blk, std::false_type{});
  if (blk < end) step(blk, std::true_type{});
  // A value that some tokens see and others do not (a later draft's, one the
  // window has passed) enters all rows' products, with weight zero where it is not
  // seen: harmless unless it is infinite or NaN. Outputs that end so are worked
  // out again, key by key, from what their token sees alone.
  if (p.T > 1) {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float nought = 0.0f;
#pragma unroll
      for (int j = 0; j < OT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) nought = __builtin_fmaf(o[r][j][i], 0.0f, nought);  // zero, or NaN
      if (!__any(nought != 0.0f)) continue;
#pragma unroll
      for (int j = 0; j < OT; ++j) o[r][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const int row = row0 + r * DEC_ROWS + c, rr = row < p.rows ? row : p.rows - 1, t = rr / p.group;
      const unsigned char *qrow =
          p.q + ((static_cast<long>(b) * p.T + t) * p.Hq + hk * p.group + rr - t * p.group) * K::ROW;
      const float base = m[r] == -INFINITY ? 0.0f : m[r], sign = p.negate ? -1.0f : 1.0f;
      for (int at = begin + wave; at < end; at += DEC_WAVES) {
        int pg, place_;
        lookup(at, pg, place_);
        const int rows = cache_row(pg, place_);
        for (int key = 0; key < KEYS; ++key) {
          const int slot_ = __shfl(rows, key, 64), u = at * KEYS + key, j = u < range.sinks ? u : u + range.delta;
          if (slot_ < 0) continue;
          const unsigned char *kr = kbase + static_cast<long>(slot_) * p.token, *vr = vbase + static_cast<long>(slot_) * p.token;
          float dot = 0.0f;
          for (int d = g * (D / 4); d < (g + 1) * (D / 4); ++d) dot += load_elem(kr, d, DT) * load_elem(qrow, d, DT);
          dot = add_xor32(add_xor16(dot)) * sign;
          if (!sees(pos[r], j, p.window, p.sinks)) continue;
          const float w = __builtin_amdgcn_exp2f((dot - base) * p.c);
#pragma unroll
          for (int x = 0; x < K::VLOADS; ++x)
#pragma unroll
            for (int e = 0; e < K::VE; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[r][x * K::VE + e][i] += w * load_elem(vr, (x * 16 + 4 * g + i) * K::VE + e, DT);
        }
      }
    }
  }
  if constexpr (Q_LDS) __syncthreads();  // Q's place is the joins'

#pragma unroll
  for (int r = 0; r < RB; ++r) l[r] = add_xor32(add_xor16(l[r]));
  // join the waves into wave 0: the upper half into the lower, or one by one
  constexpr int ROUNDS = JOINS == 2 ? 2 : DEC_WAVES - 1;
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
        const float f1 = __builtin_amdgcn_exp2f((m[r] - at) * p.c), f2 = __builtin_amdgcn_exp2f((m2 - at) * p.c);
        m[r] = top;
        l[r] = l[r] * f1 + l2 * f2;
#pragma unroll
        for (int j = 0; j < OT; ++j)
          o[r][j] = o[r][j] * f1 + *reinterpret_cast<const float4_t *>(src + ((r * OT + j) * 64 + lane) * 4) * f2;
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;

#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + r * DEC_ROWS + c;
    if (row >= p.rows) continue;
    const bool last = share.parts == 1;
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
    for (int x = 0; x < K::VLOADS; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < K::VE; e += 4) {
          const long d = at * D + x * 16 * K::VE + (4 * g + i) * K::VE + e;
          const float4_t y = {o[r][x * K::VE + e][i] * f, o[r][x * K::VE + e + 1][i] * f,
                              o[r][x * K::VE + e + 2][i] * f, o[r][x * K::VE + e + 3][i] * f};
          if (!last || !K::SHORT) {
            *reinterpret_cast<float4_t *>((last ? static_cast<float *>(p.o) : p.part) + d) = y;
          } else if constexpr (K::SHORT) {
            *reinterpret_cast<v2u32_t *>(static_cast<unsigned char *>(p.o) + 2 * d) =
                v2u32_t{E::pack(y[0], y[1]), E::pack(y[2], y[3])};
          }
        }
  }
}

// Joins a sequence's parts, SPLIT waves to a (sequence, query row and head),
// eight parts of a wave at a time: their outputs and their weights' statistics,
// one a lane, are fetched together. Four waves a row where there are few rows,
// one where there are many.
template <int DT, int D, int SPLIT>
__global__ __launch_bounds__(256) void decode_join_kernel(const DecodeParams p) {
  constexpr int VEC = D / 64, ROWS = 4 / SPLIT, AT_ONCE = 8;  // ROWS: rows of a workgroup
  __shared__ float acc[SPLIT > 1 ? 4 : 1][D], stat[4][2];
  PBGDN_POISON_LDS(acc, sizeof(acc));
  PBGDN_POISON_SYNC();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), w = wave % SPLIT;
  const int tiles = (p.rows + ROWS - 1) / ROWS;
  int id = blockIdx.x;
  const int row = id % tiles * ROWS + wave / SPLIT;
  id /= tiles;
  const int hk = id % p.Hk, b = id / p.Hk;
  const Shares all(p, lane);
  const int parts = uniform(all.parts(seq_blocks(p, b)));
  if (parts == 1) return;  // written by the first kernel
  if (SPLIT == 1 && row >= p.rows) return;
  int first = 0;  // the sequence's first slot
  if (b > 0) {
#pragma unroll
    for (int i = 0; i < Shares::HELD; ++i)
      if (64 * i + lane < b) first += all.parts(all.held[i]);
    for (int i = 64 * Shares::HELD + lane; i < b; i += 64) first += all.parts(seq_blocks(p, i));
    first = uniform(wave_sum_int(first));
  }
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
}

// ---------------------------------------------------------------------------
// Writes into the pages: 16 bytes a thread, the threads of a token together.
// ---------------------------------------------------------------------------
struct WriteParams {
  const unsigned char *k, *v;
  long k_token, k_head, v_token, v_head;
  unsigned char *kc, *vc;
  long page_stride, token, head;
  const int64_t *slots;
  long total;
  int page, units, N, Hk;  // 16-byte units of a head
};
// 19,001 tokens of 2 heads of 256, bf16: 13.3 us for 78 MB (5.8 TB/s); 64 tokens:
// 2.7 us, the host's call 8.
__global__ __launch_bounds__(256) void paged_write_kernel(const WriteParams p) {
  const int per = p.Hk * p.units;  // units of a token, of one cache
  const long n = static_cast<long>(p.N) * per;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) {
    const int tok = static_cast<int>(i / per), x = static_cast<int>(i - static_cast<long>(tok) * per);
    const int64_t slot = p.slots[tok];
    if (slot < 0 || slot >= p.total) continue;
    const int hd = x / p.units, u = x - hd * p.units;
    const int64_t pg = slot / p.page;
    const long to = pg * p.page_stride + (slot - pg * p.page) * p.token + hd * p.head + u * 16;
    const v4u32_t a = *reinterpret_cast<const v4u32_t *>(p.k + tok * p.k_token + hd * p.k_head + u * 16);
    const v4u32_t b = *reinterpret_cast<const v4u32_t *>(p.v + tok * p.v_token + hd * p.v_head + u * 16);
    *reinterpret_cast<v4u32_t *>(p.kc + to) = a;
    *reinterpret_cast<v4u32_t *>(p.vc + to) = b;
  }
}

template <int DT, int D>
static int launch_decode(DecodeParams &p, hipStream_t stream) {
  const long slots = static_cast<long>(p.target) + p.B;
  const auto run = [&](auto kernel, int rb) {
    p.row_tiles = (p.rows + rb * DEC_ROWS - 1) / (rb * DEC_ROWS);
    const long blocks = slots * p.Hk * p.row_tiles;
    if (blocks > 0x7fffffffL || static_cast<long>(p.B) * p.Hk * p.rows > 0x7fffffffL) return false;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(DEC_WAVES * 64), 0, stream, p);
    return true;
  };
  const bool ok = p.rows <= DEC_ROWS ? run(decode_kernel<DT, D, 1>, 1) : run(decode_kernel<DT, D, 2>, 2);
  if (!ok) return PBGDN_ERR_UNSUPPORTED;
  const long rows = static_cast<long>(p.B) * p.Hk * p.rows;
  if (rows <= JOIN_SPLIT_ROWS) {
    hipLaunchKernelGGL((decode_join_kernel<DT, D, 4>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, p);
  } else {
    const unsigned blocks = static_cast<unsigned>(p.B * p.Hk * ((p.rows + 3) / 4));
    hipLaunchKernelGGL((decode_join_kernel<DT, D, 1>), dim3(blocks), dim3(256), 0, stream, p);
  }
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

template <int DT>
static int dispatch_decode(DecodeParams &p, int D, hipStream_t stream) {
  switch (D) {
    case 64: return launch_decode<DT, 64>(p, stream);
    case 128: return launch_decode<DT, 128>(p, stream);
    case 256: return launch_decode<DT, 256>(p, stream);
    default: return PBGDN_ERR_UNSUPPORTED;
  }
}

// Parts wanted over all sequences: enough workgroups to even out the GPU, few
// enough that the parts' sums stay small beside the cache. Eight a CU for rows up
// to 256 bytes (three at a time; 64 contexts up to 16,384 tokens, 128 wide: 364 us,
// with four 400, with two 459), four for wider ones (two at a time; 233 contexts,
// 256 wide, 32 query rows: 337 us, with eight 349, with two 343).
static int decode_target(int Hk, int rows, int row_bytes) {
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  const int tiles = (rows + 2 * DEC_ROWS - 1) / (2 * DEC_ROWS);
  const int t = (row_bytes <= 256 ? 8 : 4) * shape.cus / (Hk * tiles);
  return t > 1 ? t : 1;
}
static bool decode_sizes_ok(int B, int T, int Hq, int Hk, int D) {
  return B >= 0 && T >= 1 && T <= PBATTN_MAX_DRAFT && Hq > 0 && Hk > 0 && Hq % Hk == 0 && D > 0;
}

// The cache's strides in bytes; false when they cannot be.
static bool cache_strides(const int64_t *s, int bytes, int page_size, int num_pages, long out[3]) {
  for (int a = 0; a < 3; ++a) {
    if (s[a] < 0 || s[a] * bytes % 16 != 0) return false;
    out[a] = s[a] * bytes;
  }
  return true;
}

}  // namespace pbgdn

extern "C" size_t pbattn_paged_decode_workspace_size(int B, int T, int Hq, int Hk, int D) {
  using namespace pbgdn;
  if (!decode_sizes_ok(B, T, Hq, Hk, D)) return 0;
  const int rows = Hq / Hk * T;
  const size_t slots = static_cast<size_t>(decode_target(Hk, rows, 0)) + B;  // the most of any type
  return slots * Hk * rows * (D * sizeof(float) + sizeof(float2));
}

extern "C" int pbattn_paged_decode(const void *q, const void *k_cache, const void *v_cache, int dtype,
                                   const int64_t *strides, int page_size, int num_pages, const int32_t *page_table,
                                   int max_pages, const int32_t *lengths, void *o, float *lse, int B, int T, int Hq,
                                   int Hk, int D, float scale, int window, int sinks, void *workspace,
                                   size_t workspace_bytes, void *stream) {
  using namespace pbgdn;
  if (!decode_sizes_ok(B, T, Hq, Hk, D) || !attn_dtype(dtype) || !strides || page_size <= 0 || num_pages < 0 ||
      max_pages < 0 || sinks < 0 || !(scale - scale == 0.0f)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (B == 0) return PBGDN_OK;
  if (!q || !o || !lengths || (max_pages > 0 && !page_table) || (num_pages > 0 && (!k_cache || !v_cache)) || !workspace ||
      !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o) || !aligned16(workspace)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  long st[3];
  if (!cache_strides(strides, attn_bytes(dtype), page_size, num_pages, st)) return PBGDN_ERR_INVALID_ARGUMENT;
  if (num_pages > 1 || page_size > 1) {
    if (st[1] <= 0 || st[0] % st[1] != 0) return PBGDN_ERR_INVALID_ARGUMENT;
  }
  const long page_rows = st[1] > 0 ? st[0] / st[1] : 0;
  if (page_rows * (num_pages > 0 ? num_pages - 1 : 0) + page_size > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  if (workspace_bytes < pbattn_paged_decode_workspace_size(B, T, Hq, Hk, D)) return PBGDN_ERR_INVALID_ARGUMENT;
  DecodeParams p{};
  p.q = static_cast<const unsigned char *>(q);
  p.k = static_cast<const unsigned char *>(k_cache);
  p.v = static_cast<const unsigned char *>(v_cache);
  p.token = st[1];
  p.head = st[2];
  p.page_rows = static_cast<int>(page_rows);
  p.page = page_size;
  p.num_pages = max_pages > 0 ? num_pages : 0;  // (no table: no keys)
  p.max_pages = max_pages;
  p.table = page_table;
  p.lengths = lengths;
  p.o = o;
  p.lse = lse;
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hk = Hk;
  p.group = Hq / Hk;
  p.rows = p.group * T;
  p.window = window <= 0 || window > NO_WINDOW ? NO_WINDOW : window;
  p.sinks = sinks < NO_WINDOW ? sinks : NO_WINDOW;
  // (no more parts than the table's pages, or the window, can need)
  long most = static_cast<long>(max_pages) * page_size;
  if (most > static_cast<long>(p.window) + T + p.sinks) most = static_cast<long>(p.window) + T + p.sinks;
  most = (most + DEC_MIN * DEC_KEYS - 1) / (DEC_MIN * DEC_KEYS) * B;
  const int wanted = decode_target(Hk, p.rows, D * attn_bytes(dtype));
  p.target = most < wanted ? static_cast<int>(most > 1 ? most : 1) : wanted;
  const float c = __builtin_fabsf(scale) * LOG2E;
  p.c = c > 1.17549435e-38f ? c : 1.17549435e-38f;
  p.negate = scale < 0.0f;
  const size_t rows = (static_cast<size_t>(p.target) + B) * Hk * p.rows;
  p.part = static_cast<float *>(workspace);
  p.stat = reinterpret_cast<float2 *>(p.part + rows * D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  debug_poison(o, static_cast<size_t>(B) * T * Hq * D * attn_bytes(dtype), s);
  if (lse) debug_poison(lse, static_cast<size_t>(B) * T * Hq * sizeof(float), s);
  debug_poison(workspace, rows * (D * sizeof(float) + sizeof(float2)), s);
  switch (dtype) {
    case PBGDN_F32: return dispatch_decode<PBGDN_F32>(p, D, s);
    case PBGDN_BF16: return dispatch_decode<PBGDN_BF16>(p, D, s);
    default: return dispatch_decode<PBGDN_F16>(p, D, s);
  }
}

extern "C" int pbattn_paged_write(const void *k, const void *v, int dtype, const int64_t *kv_strides, void *k_cache,
                                  void *v_cache, const int64_t *strides, int page_size, int num_pages,
                                  const int64_t *slots, int N, int Hk, int D, void *stream) {
  using namespace pbgdn;
  if (N < 0 || Hk <= 0 || D <= 0 || !attn_dtype(dtype) || !kv_strides || !strides || page_size <= 0 || num_pages < 0) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (N == 0 || num_pages == 0) return PBGDN_OK;
  const int bytes = attn_bytes(dtype);
  if (D * bytes % 16 != 0) return PBGDN_ERR_UNSUPPORTED;
  if (!k || !v || !k_cache || !v_cache || !slots || !aligned16(k) || !aligned16(v) || !aligned16(k_cache) ||
      !aligned16(v_cache)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  long st[3];
  if (!cache_strides(strides, bytes, page_size, num_pages, st)) return PBGDN_ERR_INVALID_ARGUMENT;
  for (int a = 0; a < 4; ++a)
    if (kv_strides[a] < 0 || kv_strides[a] * bytes % 16 != 0) return PBGDN_ERR_INVALID_ARGUMENT;
  WriteParams p{};
  p.k = static_cast<const unsigned char *>(k);
  p.v = static_cast<const unsigned char *>(v);
  p.k_token = kv_strides[0] * bytes;
  p.k_head = kv_strides[1] * bytes;
  p.v_token = kv_strides[2] * bytes;
  p.v_head = kv_strides[3] * bytes;
  p.kc = static_cast<unsigned char *>(k_cache);
  p.vc = static_cast<unsigned char *>(v_cache);
  p.page_stride = st[0];
  p.token = st[1];
  p.head = st[2];
  p.slots = slots;
  p.total = static_cast<long>(num_pages) * page_size;
  p.page = page_size;
  p.units = D * bytes / 16;
  p.N = N;
  p.Hk = Hk;
  const long want = (static_cast<long>(N) * Hk * p.units + 255) / 256;
  hipLaunchKernelGGL(paged_write_kernel, dim3(static_cast<unsigned>(want < 65536 ? want : 65536)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}
