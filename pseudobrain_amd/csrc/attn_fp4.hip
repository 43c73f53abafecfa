// The cache held in 4 bits (attn_fp4.hpp): decoding over it (pbattn_fp4_decode),
// its writes (pbattn_fp4_write) and its reading back (pbattn_fp4_read).
//
// Decoding reads 17 bytes for 32 values instead of 64, so what a bfloat16 cache's kernel
// does beside its loads would cost as much as they do. Codes become bfloat16 operands by
// one conversion for two values, scale included; a value row's codes are fetched as they
// lie and transposed by byte permutations after it. Distances of rows and scales are
// worked out once, a lane for each key, and go through LDS to the lanes that need them.
// A block's loads go out a whole block ahead, and page table entries one before that.
//
// 64 contexts up to 16,384 tokens, 32 heads of 128 on 8, bf16: 99 us, 5.7 TB/s; reading
// alone reaches 5.9 (a bfloat16 cache takes 365). 233 contexts behind a window of
// 4,096, 16 heads of 256 on 2, four drafted tokens: 130 us for 79 us of bytes, bound by
// issue: both tiles of 16 rows unpack the cache for themselves (one drafted token: 77).
// Two tiles a workgroup leave one wave a SIMD or spill: 126 to 128 us for the 136 of the
// whole call (weights in one part), but float16 rows 79 for 58 and float32 rows 110 for 64
// (64 contexts).
#include <type_traits>

#include "attn_decode.hpp"
#include "attn_fp4.hpp"
#include "pages.hpp"

namespace pbgdn {

struct Fp4DecodeParams {
  DecodeParams d;                          // k, v, head: the codes'
  const unsigned char *k_scale, *v_scale;  // laid out as the codes are, a sixteenth of every stride
  uint32_t page_step, token_step;          // a page's and a token's stride of the codes in 16 bytes, of the scales in bytes
  uint32_t page_mul;                       // j / page = (2 j page_mul) >> 32 >> page_shift for 0 <= j < 2^31
  int page_shift;
};

// How the work is divided: the keys of all sequences, in order, are one line of quads
// (four blocks of keys, one for each wave of a workgroup; a sequence that sees no key has
// one too), of which workgroup w of a (row tile, key head) takes `per` from w per on,
// whatever sequences they belong to. Its piece of sequence b is part w + b: the pairs
// (w, b) that meet follow each other, and w + b rises from each to the next. So as many
// workgroups as fit the GPU at once share the work evenly, and each starts once.
__device__ __forceinline__ long uniform_long(long x) {
  return static_cast<long>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(x >> 32)))) << 32 |
                           static_cast<uint32_t>(uniform(static_cast<int>(x))));
}
struct Walk {
  static constexpr int HELD = 4;
  int held[HELD];  // quads of sequences 64 i + lane
  long per, total;

  __device__ __forceinline__ static int quads_of(const DecodeParams &p, int len) {
    const int n = (len_blocks(p, len) + DEC_WAVES - 1) / DEC_WAVES;
    return n > 1 ? n : 1;
  }
  __device__ __forceinline__ static int quads(const DecodeParams &p, int b) { return quads_of(p, seq_length(p, b)); }

  __device__ __forceinline__ Walk(const DecodeParams &p, int lane) {
    if (p.B == 1) {  // one request: nothing to add up over the lanes
      held[0] = quads(p, 0);
      total = held[0];
    } else {
      total = 0;
      int len[HELD];  // (read by every lane, so that the four reads are in flight together)
#pragma unroll
      for (int i = 0; i < HELD; ++i) len[i] = p.lengths[64 * i + lane < p.B ? 64 * i + lane : p.B - 1];
#pragma unroll
      for (int i = 0; i < HELD; ++i) settle(len[i]);
#pragma unroll
      for (int i = 0; i < HELD; ++i) {
        held[i] = 64 * i + lane < p.B ? quads_of(p, ((p.num_pages > 0) & (len[i] > 0)) ? len[i] : 0) : 0;
        total += held[i];
      }
      for (int b = 64 * HELD + lane; b < p.B; b += 64) total += quads(p, b);
      total = wave_sum_long(total);
    }
    total = uniform_long(total);
    const long target = p.target;
    per = uniform_long(total <= 0x7fffffff - target ? (static_cast<int>(total) + p.target - 1) / p.target
                                                    : (total + target - 1) / target);
  }
  // Whose quad x < total is, and where that sequence starts.
  __device__ __forceinline__ int find(const DecodeParams &p, long x, int lane, long &start) const {
    start = 0;
    if (p.B == 1) return 0;
    int found = 0;
    const auto look = [&](int b0, int mine) __attribute__((always_inline)) {
      int scan = mine;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(scan, off, 64);
        if (lane >= off) scan += y;
      }
      const uint64_t past = __ballot(start + scan > x);
      if (past) {
        const int l = __builtin_ctzll(past);
        found = b0 + l;
        start += __shfl(scan, l, 64) - __shfl(mine, l, 64);
        return true;
      }
      start += __shfl(scan, 63, 64);
      return false;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (64 * i >= p.B || look(64 * i, held[i])) return found;
    for (int b0 = 64 * HELD; b0 < p.B; b0 += 64)
      if (look(b0, b0 + lane < p.B ? quads(p, b0 + lane) : 0)) break;
    return found;
  }
  // Sequence b's first quad.
  __device__ __forceinline__ long start_of(const DecodeParams &p, int b, int lane) const {
    if (b == 0) return 0;
    long x = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (64 * i + lane < b) x += held[i];
    for (int i = 64 * HELD + lane; i < b; i += 64) x += quads(p, i);
    return wave_sum_long(x);
  }
  __device__ __forceinline__ int workgroup_of(long x) const {
    return x <= 0x7fffffff && per <= 0x7fffffff ? static_cast<int>(x) / static_cast<int>(per) : static_cast<int>(x / per);
  }
  // Sequence b's parts, and its first slot.
  __device__ __forceinline__ int parts_of(const DecodeParams &p, int b, int lane) const {
    const long first = start_of(p, b, lane);
    return uniform(workgroup_of(first + quads(p, b) - 1) - workgroup_of(first) + 1);
  }
  __device__ __forceinline__ int first_of(const DecodeParams &p, int b, int lane) const {
    return uniform(workgroup_of(start_of(p, b, lane))) + b;
  }
};

// Q and the weights enter bfloat16 products as one, two or three parts that sum up to
// them. Q: bfloat16 rows as they are, float16 rows in two, float32 rows in three, all of
// them exactly. The weights: two parts, which round them to 16 bits (2^-16: small beside a
// 16-bit result's own rounding, and to either side), and for float32 rows three, which are
// all of their 24 bits. (One part for bfloat16 rows takes 107 us for 113 with 64 contexts up
// to 16,384 tokens, and leaves an error of 2^-9 in every weight: 0.0021 to 0.0023 against 64
// bits, for the 0.0017 of the result's own rounding.)
// So the cache's values, exact in bfloat16, meet every type of row in the same kernel.
template <int DT>
struct Parts {
  static constexpr int N = DT == PBGDN_BF16 ? 1 : DT == PBGDN_F16 ? 2 : 3;
  static constexpr int WEIGHT = DT == PBGDN_F32 ? 3 : 2;
};
// The upper halves of two words.
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
// Two values as N pairs of bfloat16: all but the last cut, not rounded (no part passes the
// type's range), the last, what is left, rounded to nearest.
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t *out) {
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    out[i] = upper_halves(a, b);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
  out[N - 1] = Elem<PBGDN_BF16>::pack(x, y);
}

// Eight values from src as float32.
template <int DT>
__device__ __forceinline__ void load8(const unsigned char *src, float *x) {
  if constexpr (DT == PBGDN_F32) {
    const float4_t a = *reinterpret_cast<const float4_t *>(src), b = *reinterpret_cast<const float4_t *>(src + 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = a[e];
      x[4 + e] = b[e];
    }
  } else {
    const v4u32_t a = *reinterpret_cast<const v4u32_t *>(src);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = Elem<DT>::low(a[e]);
      x[2 * e + 1] = Elem<DT>::high(a[e]);
    }
  }
}

// Read past the caches (ONCE) or through them.
template <bool ONCE, typename T>
__device__ __forceinline__ T load_keys(const T *p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  return *p;
}

template <int DT, int D>
struct Fp4 {
  static constexpr int N = Parts<DT>::N, W = Parts<DT>::WEIGHT;
  static constexpr int ROW = D / 2;           // bytes of a key's codes
  static constexpr int SROW = D / FP4_BLOCK;  // and of its scales
  static constexpr int KSTEPS = D / 32;       // matrix steps of a score
  static constexpr int KW = ROW / 16;         // words a lane reads of a key: one a step
  static constexpr int KSCALES = D == 256 ? 2 : 1;  // and of its scales
  static constexpr int OT = D / 16;           // output tiles: values a lane reads of a value row
  static constexpr int VW = D == 64 ? 1 : OT / 8;   // words that hold them
  static constexpr int KG = 2, KEYS = 16 * KG;      // keys at a time
  static constexpr int SW = SROW / 4 > 0 ? SROW / 4 : 1;  // words that hold a key's scales
  // First of the eight columns that lane group g takes in matrix step s.
  __device__ static constexpr int column(int g, int s) {
    return D == 64 ? 16 * g + 8 * s : 128 * (s / 4) + 32 * g + 8 * (s % 4);
  }
};

// A wave's own LDS accesses before this come before those after it.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Which of 16 keys is row m of their matrix product, so that the values of keys 4 i ..
// 4 i + 3, next to each other where their rows are, are those of element i of the
// result's lane groups.
__device__ __forceinline__ int key_of(int m) { return 4 * (m % 4) + m / 4; }

// Workgroups of a CU at once (waves of a SIMD), by the registers that the sums of RB row
// tiles and two blocks of keys and values take. Four at D = 64 spill 2 to 5 registers (64
// contexts up to 8,192 tokens, 24 heads on 8: heads before tokens 49 us, 52 with three and
// no spill; float16, two drafted tokens 52.5 and 54; tokens first 50 and 48).
constexpr int fp4_held(int D, int RB) { return RB == 2 || D == 256 ? 2 : D == 128 ? 3 : 4; }

// NEAR: the caches' offsets fit 32 bits. ONCE: no other workgroup reads the same lines, so
// that keys are loaded past the caches (values not: a row's are fetched in pieces). HEADS:
// key heads of a workgroup, whose waves they share by parity: two where the rows of
// neighbouring heads lie side by side, and are so fetched together.
template <int DT, int D, int RB, bool NEAR, bool ONCE, int HEADS>
__global__ __launch_bounds__(DEC_WAVES * 64, (fp4_held(D, RB))) void fp4_decode_kernel(const Fp4DecodeParams pp) {
  using K = Fp4<DT, D>;
  using E = Elem<PBGDN_BF16>;
  constexpr int KS = K::KSTEPS, OT = K::OT, KG = K::KG, KEYS = K::KEYS, N = K::N, W = K::W;
  constexpr int JOINS = RB * D <= 256 ? 2 : 1, HW = DEC_WAVES / HEADS;  // HW: waves of a head
  __shared__ __attribute__((aligned(16))) float merge[JOINS][RB * DEC_ROWS * (D + 2)];
  __shared__ v4u32_t q_of[HEADS][RB * N * KS * 64];  // [row tile][part][step][lane]
  __shared__ struct {
    __attribute__((aligned(16))) uint32_t at[KEYS];
    unsigned char scales[2 * KEYS * K::SROW];  // of the keys, then of the values
  } lds_keys[DEC_WAVES];
  PBGDN_POISON_LDS(merge, sizeof(merge));
  PBGDN_POISON_LDS(q_of, sizeof(q_of));
  PBGDN_POISON_LDS(lds_keys, sizeof(lds_keys));
  PBGDN_POISON_SYNC();
  const DecodeParams &p = pp.d;

  const int thread = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  // Workgroups go to the XCDs in turn: the heads and row tiles of a piece follow each
  // other on one XCD, whose L2 they share (rows of a token next to each other lie in one
  // line; row tiles read the same ones).
  const int groups = p.Hk / HEADS, pieces = groups * p.row_tiles, turn = blockIdx.x >> 3;
  const int w = uniform(turn / pieces * 8 + (blockIdx.x & 7)), id = turn - turn / pieces * pieces;
  const int row0 = uniform(id / groups) * (RB * DEC_ROWS), hk = uniform(id % groups * HEADS + wave % HEADS);
  const int hw = wave / HEADS;  // this wave among its head's
  v4u32_t *const q_lds = q_of[wave % HEADS];
  const Walk walk(p, thread);
  const long x_end = (w + 1) * walk.per < walk.total ? (w + 1) * walk.per : walk.total;
  long x_at = w * walk.per, start;
  if (w >= p.target || x_at >= walk.total) return;
  int b = uniform(walk.find(p, x_at, thread, start));
  start = uniform_long(start);
  for (; x_at < x_end && b < p.B; ++b) {
    // (opaque: what follows from the lane is worked out where it is used, for each part
    // again, instead of being kept in registers that the main loop needs)
    const int lane = static_cast<int>(opaque(thread)), c = lane & 15, g = lane >> 4;
    const int len = uniform(seq_length(p, b));
    const KeyRange range = seq_keys(p, len);
    const int quads = uniform(Walk::quads_of(p, len));
    const int quad0 = uniform(static_cast<int>(x_at - start));
    const int quad1 = uniform(static_cast<int>(x_end - start < quads ? x_end - start : quads));
    const bool alone = quad0 == 0 && quad1 == quads;  // the sequence's only part
    const int slot = w + b;
    x_at = start + quad1;
    start += quads;
    // this wave's KEYS-wide blocks of the part: begin + hw, then every HW-th
    static_assert(KEYS == DEC_KEYS, "quads are of such blocks");
    const int blocks = (range.count + KEYS - 1) / KEYS, begin = quad0 * DEC_WAVES;
    const int end = uniform(quad1 * DEC_WAVES < blocks ? quad1 * DEC_WAVES : blocks);

    // this lane's rows of Q (column c of every row tile), in parts; each wave brings in a share
    int pos[RB];
    constexpr int QB = DT == PBGDN_F32 ? 4 : 2;  // bytes of an element of Q
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int row = row0 + r * DEC_ROWS + c;
      const int rr = row < p.rows ? row : p.rows - 1;
      const int t = rr / p.group;
      pos[r] = len - p.T + t;
      const unsigned char *src = p.q + ((static_cast<long>(b) * p.T + t) * p.Hq + hk * p.group + rr - t * p.group) * (D * QB);
      for (int s = hw; s < KS; s += HW) {
        const unsigned char *eight = src + K::column(g, s) * QB;
        v4u32_t part[N];
        if constexpr (DT == PBGDN_BF16) {
          part[0] = *reinterpret_cast<const v4u32_t *>(eight);
          if (p.negate) part[0] ^= 0x80008000u;
        } else {
          float x[8];
          load8<DT>(eight, x);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            uint32_t y[N];
            split_pair<N>(p.negate ? -x[e] : x[e], p.negate ? -x[e + 1] : x[e + 1], y);
#pragma unroll
            for (int i = 0; i < N; ++i) part[i][e / 2] = y[i];
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) q_lds[((r * N + i) * KS + s) * 64 + lane] = part[i];
      }
    }
    __syncthreads();
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
    const unsigned char *ksbase = pp.k_scale + hk * (p.head / 16), *vsbase = pp.v_scale + hk * (p.head / 16);
    const int32_t *table = p.table + static_cast<long>(b) * p.max_pages;
    // Where a block's keys lie, key lane % KEYS a lane: its page and its place there (-1:
    // there is none), and then its row's distance from the caches' bases (of a row that
    // exists, in any case).
    struct Place {
      int page, place;
    };
    const auto lookup = [&](int blk) __attribute__((always_inline)) {
      const uint32_t u = static_cast<uint32_t>(blk) * KEYS + lane % KEYS, last = range.count - 1;  // (past a range's end too)
      const int v = static_cast<int>(u < last ? u : last), j = v < range.sinks ? v : v + range.delta;
      const int pg = static_cast<int>(__umulhi(2u * j, pp.page_mul) >> pp.page_shift);
      return Place{table[pg < p.max_pages ? pg : p.max_pages - 1], ((u <= last) & (pg < p.max_pages)) ? j - pg * p.page : -1};
    };
    const auto exists = [&](const Place &x) __attribute__((always_inline)) {
      return (x.place >= 0) & (x.page >= 0) & (x.page < p.num_pages);
    };
    const auto distance = [&](const Place &x) __attribute__((always_inline)) {
      return exists(x) ? (x.page * pp.page_step + x.place * pp.token_step) << (NEAR ? 4 : 0) : 0u;
    };
    // A block as a lane takes it: unit g of key 16 kb + c of every group of keys, columns
    // OT c .. of the values that its weights belong to, and the scales of one key (lanes
    // below KEYS) or value. The scales and the distances go to their users through LDS,
    // where a wave has a place of its own.
    struct Block {
      uint32_t k[KG][K::KW], v[4 * KG][K::VW], scales[K::SW];
      bool held;  // key lane % KEYS exists
    };
    uint32_t *const at = lds_keys[wave].at;
    unsigned char *const scales = lds_keys[wave].scales;
    const auto publish = [&](const Place &x) __attribute__((always_inline)) {
      const uint32_t d = distance(x);
      wave_lds_order();
      if (lane < KEYS) at[lane] = d;
      wave_lds_order();
      return d;
    };
    const unsigned char *const my_scales = lane < KEYS ? ksbase : vsbase;
    const auto codes = [&](const unsigned char *base, uint32_t d, uint32_t lane_at) __attribute__((always_inline)) {
      return NEAR ? base + (d + lane_at) : base + lane_at + (static_cast<uint64_t>(d) << 4);
    };
    const auto load = [&](Block &x, const Place &pl) __attribute__((always_inline)) {
      x.held = exists(pl);
      const unsigned char *ss = my_scales + (publish(pl) >> (NEAR ? 4 : 0));
      if constexpr (D == 64) {
        x.scales[0] = *reinterpret_cast<const uint16_t *>(ss);
      } else if constexpr (D == 128) {
        x.scales[0] = *reinterpret_cast<const uint32_t *>(ss);
      } else {
        const v2u32_t w = *reinterpret_cast<const v2u32_t *>(ss);
        x.scales[0] = w[0];
        x.scales[1] = w[1];
      }
#pragma unroll
      for (int kb = 0; kb < KG; ++kb) {
        const unsigned char *src = codes(kbase, at[16 * kb + key_of(c)], g * (D == 64 ? 8 : 16));
        if constexpr (D == 64) {
          const v2u32_t w = load_keys<ONCE>(reinterpret_cast<const v2u32_t *>(src));
          x.k[kb][0] = w[0];
          x.k[kb][1] = w[1];
        } else {
#pragma unroll
          for (int h = 0; h < D / 128; ++h) {
            const v4u32_t w = load_keys<ONCE>(reinterpret_cast<const v4u32_t *>(src + h * 64));
#pragma unroll
            for (int e = 0; e < 4; ++e) x.k[kb][4 * h + e] = w[e];
          }
        }
      }
#pragma unroll
      for (int kb = 0; kb < KG; ++kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned char *src = codes(vbase, at[16 * kb + 4 * i + g], c * (OT / 2));
          if constexpr (D == 64) {
            x.v[4 * kb + i][0] = *reinterpret_cast<const uint16_t *>(src);
          } else if constexpr (D == 128) {
            x.v[4 * kb + i][0] = *reinterpret_cast<const uint32_t *>(src);
          } else {
            const v2u32_t w = *reinterpret_cast<const v2u32_t *>(src);
            x.v[4 * kb + i][0] = w[0];
            x.v[4 * kb + i][1] = w[1];
          }
        }
      }
    };
    // One block of keys, cur; the next one's loads go out before it is worked on, and
    // before them the page table's entries of the one after: loads come back in order.
    Place pl{-1, -1};  // of the next block
    const auto step = [&](int blk, Block &cur, Block &next, auto last) __attribute__((always_inline)) {
      constexpr bool more = !decltype(last)::value;
      if constexpr (more) {
        const Place after = lookup(blk + 2 * HW);
        load(next, pl);
        pl = after;
      }
      // absent keys get a scale of one: finite values, whatever the row they were read from
      // holds, which their weights of zero cancel
#pragma unroll
      for (int i = 0; i < K::SW; ++i) cur.scales[i] = cur.held ? cur.scales[i] : 0x7f7f7f7fu;
      wave_lds_order();
      if constexpr (D == 64) {
        reinterpret_cast<uint16_t *>(scales)[lane] = static_cast<uint16_t>(cur.scales[0]);
      } else {
#pragma unroll
        for (int i = 0; i < K::SW; ++i) reinterpret_cast<uint32_t *>(scales)[K::SW * lane + i] = cur.scales[i];
      }
      wave_lds_order();
      const uint64_t held = __ballot(cur.held);
      float4_t sc[RB][KG];
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int kb = 0; kb < KG; ++kb) sc[r][kb] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      float ks[KG][K::KSCALES];
#pragma unroll
      for (int kb = 0; kb < KG; ++kb)
#pragma unroll
        for (int h = 0; h < K::KSCALES; ++h)
          ks[kb][h] = fp4_scale(scales[(16 * kb + key_of(c)) * K::SROW + (D == 64 ? g / 2 : 4 * h + g)]);
      float vs[4 * KG];
#pragma unroll
      for (int i = 0; i < 4 * KG; ++i)
        vs[i] = fp4_scale(scales[(KEYS + i / 4 * 16 + 4 * (i % 4) + g) * K::SROW + c * OT / FP4_BLOCK]);
      // Q's parts are read a matrix step ahead where there are registers for them (64 contexts up
      // to 8,192 tokens, 32 heads of 128, eight drafted tokens: 93.2 and 90.5 us; 256-wide float32
      // 67.8 and 64.4).
      constexpr int AHEAD = N == 1 || D == 256 ? 2 : 1;
      v4u32_t qs[AHEAD][N * RB];
      const auto read_q = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N * RB; ++i) qs[s % AHEAD][i] = q_lds[((i % RB * N + i / RB) * KS + s) * 64 + lane];
      };
#pragma unroll
      for (int s = 0; s < AHEAD - 1; ++s) read_q(s);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (s + AHEAD - 1 < KS) read_q(s + AHEAD - 1);
        v4u32_t a[KG];
#pragma unroll
        for (int kb = 0; kb < KG; ++kb) a[kb] = fp4_unpack8(cur.k[kb][s], ks[kb][D == 256 ? s / 4 : 0]);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            const v4u32_t q = qs[s % AHEAD][i * RB + r];
#pragma unroll
            for (int kb = 0; kb < KG; ++kb) sc[r][kb] = E::mma16(a[kb], q, sc[r][kb]);
          }
      }
      const int u0 = blk * KEYS;
      const int j0 = u0 < range.sinks ? u0 : u0 + range.delta, j1 = u0 + KEYS - 1 + range.delta;
      const bool whole = held == ~0ull && u0 >= range.sinks && j1 <= len - p.T && j0 > len - 1 - p.window;
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        float4_t (&s)[KG] = sc[r];
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4 * KG; ++i) {
            const int key = i / 4 * 16 + 4 * (i % 4) + g, u = u0 + key;
            const int j = u < range.sinks ? u : u + range.delta;
            const bool seen = ((held >> key) & 1) & sees(pos[r], j, p.window, p.sinks);
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
        float sum = 0.0f;
        if (__any(fabsf(at) > EXACT_SCORES)) {
#pragma unroll
          for (int i = 0; i < 4 * KG; ++i) s[i / 4][i % 4] = (s[i / 4][i % 4] - base) * p.c;
        } else {
#pragma unroll
          for (int i = 0; i < 4 * KG; ++i) s[i / 4][i % 4] = __builtin_fmaf(s[i / 4][i % 4], p.c, -at);
        }
#pragma unroll
        for (int i = 0; i < 4 * KG; ++i) {
          s[i / 4][i % 4] = __builtin_amdgcn_exp2f(s[i / 4][i % 4]);
          sum += s[i / 4][i % 4];
        }
        l[r] += sum;
      }
      // O^T += V^T P; element e of the lane's values makes output tile e
      v4u32_t w[RB][KG / 2][W];
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int h = 0; h < KG / 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = sc[r][2 * h + i / 2][2 * (i % 2)], y = sc[r][2 * h + i / 2][2 * (i % 2) + 1];
            uint32_t part[W];
            split_pair<W>(x, y, part);
#pragma unroll
            for (int n = 0; n < W; ++n) w[r][h][n][i] = part[n];
          }
      const auto pair_of_tiles = [&](auto E0) __attribute__((always_inline)) {  // tiles 2 e and 2 e + 1
        constexpr int e = decltype(E0)::value;
#pragma unroll
        for (int h = 0; h < KG / 2; ++h) {
          uint32_t x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = fp4_pair<e % 4>(cur.v[8 * h + i][e / 4], vs[8 * h + i]);
          v4u32_t lo, hi;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
            hi[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
          }
#pragma unroll
          for (int n = 0; n < W; ++n)
#pragma unroll
            for (int r = 0; r < RB; ++r) {
              o[r][2 * e] = E::mma16(lo, w[r][h][n], o[r][2 * e]);
              o[r][2 * e + 1] = E::mma16(hi, w[r][h][n], o[r][2 * e + 1]);
            }
        }
      };
      pair_of_tiles(std::integral_constant<int, 0>{});
      pair_of_tiles(std::integral_constant<int, 1>{});
      if constexpr (OT >= 8) {
        pair_of_tiles(std::integral_constant<int, 2>{});
        pair_of_tiles(std::integral_constant<int, 3>{});
      }
      if constexpr (OT >= 16) {
        pair_of_tiles(std::integral_constant<int, 4>{});
        pair_of_tiles(std::integral_constant<int, 5>{});
        pair_of_tiles(std::integral_constant<int, 6>{});
        pair_of_tiles(std::integral_constant<int, 7>{});
      }
    };
    if (begin + hw < end) {
      Block x, y;
      const Place first = lookup(begin + hw);
      pl = lookup(begin + hw + HW);
      load(x, first);
      int blk = begin + hw;
      for (; blk + 2 * HW < end; blk += 2 * HW) {
        step(blk, x, y, std::false_type{});
        step(blk + HW, y, x, std::false_type{});
      }
      if (blk + HW < end) {
        step(blk, x, y, std::false_type{});
        step(blk + HW, y, x, std::true_type{});
      } else {
        step(blk, x, y, std::true_type{});
      }
    }
    // A value that some tokens see and others do not enters all rows' products, with
    // weight zero where it is not seen: harmless unless its scale is that of NaN (or
    // infinite). Outputs that end so are worked out again, key by key, from what their
    // token sees alone.
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
        const unsigned char *qrow = p.q + ((static_cast<long>(b) * p.T + t) * p.Hq + hk * p.group + rr - t * p.group) * (D * QB);
        const float base = m[r] == -INFINITY ? 0.0f : m[r], sign = p.negate ? -1.0f : 1.0f;
        for (int at = begin + hw; at < end; at += HW) {
          const Place mine = lookup(at);
          const uint64_t held = __ballot(exists(mine));
          const int steps = static_cast<int>(distance(mine));
          for (int key = 0; key < KEYS; ++key) {
            const uint64_t sr = static_cast<uint32_t>(__shfl(steps, key, 64)) >> (NEAR ? 4 : 0), cr = sr << 4;
            const int u = at * KEYS + key, j = u < range.sinks ? u : u + range.delta;
            if (!((held >> key) & 1)) continue;
            float dot = 0.0f;
#pragma unroll 1
            for (int d = g * (D / 4); d < (g + 1) * (D / 4); d += 8) {
              const v4u32_t k = fp4_unpack8(*reinterpret_cast<const uint32_t *>(kbase + cr + d / 2),
                                            fp4_scale(ksbase[sr + d / FP4_BLOCK]));
              float x[8];
              load8<DT>(qrow + d * QB, x);
#pragma unroll
              for (int e = 0; e < 4; ++e) dot += E::low(k[e]) * x[2 * e] + E::high(k[e]) * x[2 * e + 1];
            }
            dot = add_xor32(add_xor16(dot)) * sign;
            if (!sees(pos[r], j, p.window, p.sinks)) continue;
            const float w = __builtin_amdgcn_exp2f((dot - base) * p.c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d = (4 * g + i) * OT;
              const float vs = fp4_scale(vsbase[sr + d / FP4_BLOCK]);
#pragma unroll
              for (int e = 0; e < OT; e += 8) {
                const unsigned char *src = vbase + cr + (d + e) / 2;
                uint32_t word;
                if constexpr (D == 64)
                  word = *reinterpret_cast<const uint16_t *>(src);
                else
                  word = *reinterpret_cast<const uint32_t *>(src);
                const v4u32_t v = fp4_unpack8(word, vs);
#pragma unroll
                for (int x = 0; x < 8 && e + x < OT; ++x)
                  o[r][e + x][i] += w * (x % 2 ? E::high(v[x / 2]) : E::low(v[x / 2]));
              }
              __builtin_amdgcn_sched_barrier(0);  // (not all the values at once, in so many registers)
            }
          }
        }
      }
    }
    const int lane_ = static_cast<int>(opaque(thread));
    join_waves<RB, D, JOINS, HEADS>(merge, m, l, o, wave, lane_, p.c);
    if (wave < HEADS) store_decoded<DT, D, RB, OT>(p, alone, b, hk, row0, slot, lane_, m, l, o);
  }
}

// ---------------------------------------------------------------------------
// Writes: eight values of a key and of a value a thread, four threads a scale. Bound by
// bytes: 19,001 tokens of two 256-wide heads, bf16, 10.4 us (4.7 TB/s read and written);
// 64 tokens of eight heads 2.8 us, the launch.
// ---------------------------------------------------------------------------
struct Fp4Cache {
  unsigned char *k, *v, *k_scale, *v_scale;
  long page_stride, token, head;  // of the codes, bytes; the scales': a sixteenth
  long total;                     // slots
  int page;
};
struct Fp4WriteParams {
  const unsigned char *k, *v;
  long k_token, k_head, v_token, v_head;
  Fp4Cache cache;
  const int64_t *slots;
  int eighths, N, Hk;  // groups of eight values of a head
};

// Codes of the eight values of each of four neighbouring lanes, and their scale.
__device__ __forceinline__ uint32_t quantise(const float *x, uint32_t &scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t a = __float_as_uint(x[e]) & 0x7fffffffu;
    top = a > top ? a : top;
  }
  uint32_t other = __builtin_amdgcn_mov_dpp(top, 0xb1, 0xf, 0xf, false);
  top = other > top ? other : top;
  other = __builtin_amdgcn_mov_dpp(top, 0x4e, 0xf, 0xf, false);
  top = other > top ? other : top;
  scale = fp4_scale_of(top);
  return fp4_pack8(x, fp4_scale(scale));
}

template <int DT>
__global__ __launch_bounds__(256) void fp4_write_kernel(const Fp4WriteParams p) {
  constexpr int BYTES = DT == PBGDN_F32 ? 4 : 2;
  const int per = p.Hk * p.eighths;  // of a token (a multiple of 8: the lanes of a scale stay together)
  const long n = static_cast<long>(p.N) * per;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) {
    const int tok = static_cast<int>(i / per), x = static_cast<int>(i - static_cast<long>(tok) * per);
    const int64_t slot = p.slots[tok];
    if (slot < 0 || slot >= p.cache.total) continue;
    const int hd = x / p.eighths, u = x - hd * p.eighths;
    const int64_t pg = slot / p.cache.page;
    const long row = pg * p.cache.page_stride + (slot - pg * p.cache.page) * p.cache.token + hd * p.cache.head;
    float k[8], v[8];
    load8<DT>(p.k + tok * p.k_token + hd * p.k_head + u * (8 * BYTES), k);
    load8<DT>(p.v + tok * p.v_token + hd * p.v_head + u * (8 * BYTES), v);
    uint32_t ks, vs;
    const uint32_t kc = quantise(k, ks), vc = quantise(v, vs);
    *reinterpret_cast<uint32_t *>(p.cache.k + row + u * 4) = kc;
    *reinterpret_cast<uint32_t *>(p.cache.v + row + u * 4) = vc;
    if (u % 4 == 0) {
      p.cache.k_scale[row / 16 + u / 4] = static_cast<unsigned char>(ks);
      p.cache.v_scale[row / 16 + u / 4] = static_cast<unsigned char>(vs);
    }
  }
}

// ---------------------------------------------------------------------------
// Reading back: sequences packed in their order, eight values of a key and of a
// value a thread. Every workgroup adds up the lengths for itself, finds the cache
// rows of its tokens, and copies them, four pieces a thread in flight. Bound by bytes:
// 41,600 tokens of two 256-wide heads as bf16 in 24 us (4.5 TB/s read and written).
// ---------------------------------------------------------------------------
constexpr int READ_TOKENS = 64;  // most tokens of a workgroup

struct Fp4ReadParams {
  Fp4Cache cache;
  const int32_t *table, *lengths;
  void *k, *v;
  int32_t *cu;
  int B, max_pages, tokens, Hk, eighths, num_pages, per_block;
};

// Eight values of a word as DT at dst.
template <int DT>
__device__ __forceinline__ void store8(unsigned char *dst, uint32_t w, float scale) {
  const v4u32_t x = fp4_unpack8(w, scale);
  if constexpr (DT == PBGDN_BF16) {
    *reinterpret_cast<v4u32_t *>(dst) = x;
  } else if constexpr (DT == PBGDN_F16) {
    v4u32_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = Elem<PBGDN_F16>::pack(Elem<PBGDN_BF16>::low(x[e]), Elem<PBGDN_BF16>::high(x[e]));
    *reinterpret_cast<v4u32_t *>(dst) = y;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float4_t *>(dst + 16 * h) =
          float4_t{Elem<PBGDN_BF16>::low(x[2 * h]), Elem<PBGDN_BF16>::high(x[2 * h]),
                   Elem<PBGDN_BF16>::low(x[2 * h + 1]), Elem<PBGDN_BF16>::high(x[2 * h + 1])};
  }
}

template <int DT>
__global__ __launch_bounds__(SCAN_THREADS) void fp4_read_kernel(const Fp4ReadParams p) {
  constexpr int BYTES = DT == PBGDN_F32 ? 4 : 2, AT_ONCE = 4;
  __shared__ int start[MAX_REQUESTS];
  __shared__ long waves[SCAN_WAVES], rows[READ_TOKENS];
  PBGDN_POISON_LDS(start, sizeof(start));
  PBGDN_POISON_LDS(rows, sizeof(rows));
  PBGDN_POISON_SYNC();
  const int each = (p.B + SCAN_THREADS - 1) / SCAN_THREADS, b0 = threadIdx.x * each;
  long mine = 0, total;
  for (int b = b0; b < b0 + each && b < p.B; ++b) mine += p.lengths[b] > 0 ? p.lengths[b] : 0;
  long at = block_scan(mine, waves, total);
  for (int b = b0; b < b0 + each && b < p.B; ++b) {
    start[b] = static_cast<int>(at < p.tokens ? at : p.tokens);
    if (blockIdx.x == 0) p.cu[b] = start[b];
    at += p.lengths[b] > 0 ? p.lengths[b] : 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.cu[p.B] = static_cast<int>(total < p.tokens ? total : p.tokens);
  __syncthreads();

  const int first = blockIdx.x * p.per_block, n = p.tokens - first < p.per_block ? p.tokens - first : p.per_block;
  if (static_cast<int>(threadIdx.x) < n) {
    const int t = first + threadIdx.x;
    long row = -1;  // (tokens past the last sequence have none)
    if (t < total) {
      const int b = sequence_of(start, p.B, t), j = t - start[b], i = j / p.cache.page;
      const int pg = i < p.max_pages ? p.table[static_cast<long>(b) * p.max_pages + i] : -1;
      if (pg >= 0 && pg < p.num_pages) row = pg * p.cache.page_stride + (j - i * p.cache.page) * p.cache.token;
    }
    rows[threadIdx.x] = row;
  }
  __syncthreads();
  const int per = p.Hk * p.eighths, end = n * per;
  for (int i0 = threadIdx.x; i0 < end; i0 += AT_ONCE * SCAN_THREADS) {
    uint32_t k[AT_ONCE], v[AT_ONCE], ks[AT_ONCE], vs[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int i = i0 + j * SCAN_THREADS, tok = i < end ? i / per : 0, x = i - tok * per;
      const int hd = x / p.eighths, u = x - hd * p.eighths;
      const long row = i < end ? rows[tok] : -1;
      k[j] = v[j] = 0;
      ks[j] = vs[j] = 127;
      if (row >= 0) {
        const long from = row + hd * p.cache.head, scales = from / 16 + u / 4;
        k[j] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p.cache.k + from + u * 4));
        v[j] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p.cache.v + from + u * 4));
        ks[j] = p.cache.k_scale[scales];
        vs[j] = p.cache.v_scale[scales];
      }
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int i = i0 + j * SCAN_THREADS;
      if (i >= end) break;
      const long to = (static_cast<long>(first) * per + i) * (8 * BYTES);
      store8<DT>(static_cast<unsigned char *>(p.k) + to, k[j], fp4_scale(ks[j]));
      store8<DT>(static_cast<unsigned char *>(p.v) + to, v[j], fp4_scale(vs[j]));
    }
  }
}

// Row tiles of 16 that a workgroup takes at once: two where that keeps its registers
// within those of two waves a SIMD.
static int fp4_row_tiles(int D, int rows) { return rows > DEC_ROWS && D < 256 ? 2 : 1; }

// Key heads of a workgroup: two where the rows of neighbouring heads lie side by side and
// are shorter than a line. Rows in token order, times with one head and with two: 64
// contexts up to 8,192 tokens, 8 heads of 64, 66 and 49 us; 16 up to 4,000, 16 heads of
// 128, 38.5 and 33; 64 up to 16,384, 8 heads of 128, 155 and 152 (142 with four, which took
// 4% longer in the others; heads before tokens 106: memory gives more in longer runs).
static int fp4_heads(int Hk, int rows, int D, bool beside) {
  return beside && D < 256 && rows <= DEC_ROWS && Hk % 2 == 0 ? 2 : 1;
}

// Workgroups of a row tile and `heads` key heads: together as many as the GPU holds at once.
static int fp4_target(int Hk, int rows, int D, int heads) {
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  const int rb = fp4_row_tiles(D, rows), tiles = (rows + rb * DEC_ROWS - 1) / (rb * DEC_ROWS);
  const long t = static_cast<long>(fp4_held(D, rb)) * shape.cus / (static_cast<long>(Hk / heads) * tiles);
  return t > 1 ? static_cast<int>(t) : 1;
}

template <int DT, int D, bool NEAR>
static int launch_fp4(Fp4DecodeParams &p, int heads, hipStream_t stream) {
  // A line that holds rows of several heads is read by the workgroups of all of them: through the
  // caches (64 contexts up to 8,192 tokens, token by token: 3 heads of 128 past them 41.3 us, through
  // them 37.7; 3 of 64 34.6 and 32.5; 8 of 64, eight drafted tokens 79.5 and 76.4).
  const bool own_lines = p.d.Hk == 1 || p.d.head >= 128;
  const int rb = fp4_row_tiles(D, p.d.rows);
  p.d.row_tiles = (p.d.rows + rb * DEC_ROWS - 1) / (rb * DEC_ROWS);
  const long blocks = (p.d.target + 7L) / 8 * 8 * (p.d.Hk / heads) * p.d.row_tiles;
  // Joined by four waves a row where a sequence may have more parts than one fetches at once;
  // else eight rows a workgroup, which all take the same sums over the lengths.
  const bool split = p.d.target > 8L * p.d.B;
  if (blocks > MAX_BLOCKS || join_blocks(p.d, split, 8) > MAX_BLOCKS ||
      static_cast<long>(p.d.B) * p.d.Hk * p.d.rows > 0x7fffffffL) {
    return PBGDN_ERR_UNSUPPORTED;
  }
  const auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(DEC_WAVES * 64), 0, stream, p);
  };
  if constexpr (D == 256) {
    if (p.d.row_tiles == 1 && NEAR)
      run(fp4_decode_kernel<DT, D, 1, NEAR, NEAR, 1>);
    else
      run(fp4_decode_kernel<DT, D, 1, NEAR, false, 1>);
  } else {
    if (NEAR && heads == 2)
      run(fp4_decode_kernel<DT, D, 1, NEAR, false, NEAR ? 2 : 1>);
    else if (rb == 1 && own_lines && NEAR)
      run(fp4_decode_kernel<DT, D, 1, NEAR, NEAR, 1>);
    else if (rb == 1)
      run(fp4_decode_kernel<DT, D, 1, NEAR, false, 1>);
    else if (p.d.row_tiles == 1 && own_lines && NEAR)
      run(fp4_decode_kernel<DT, D, 2, NEAR, NEAR, 1>);
    else
      run(fp4_decode_kernel<DT, D, 2, NEAR, false, 1>);
  }
  launch_join<DT, D, 8, Walk>(p.d, split, stream);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

template <int DT, bool NEAR>
static int dispatch_fp4(Fp4DecodeParams &p, int D, int heads, hipStream_t stream) {
  switch (D) {
    case 64: return launch_fp4<DT, 64, NEAR>(p, heads, stream);
    case 128: return launch_fp4<DT, 128, NEAR>(p, heads, stream);
    default: return launch_fp4<DT, 256, NEAR>(p, heads, stream);
  }
}
template <int DT>
static int dispatch_fp4(Fp4DecodeParams &p, int D, bool near, int heads, hipStream_t stream) {
  return near ? dispatch_fp4<DT, true>(p, D, heads, stream) : dispatch_fp4<DT, false>(p, D, heads, stream);
}

static bool fp4_width(int D) { return D == 64 || D == 128 || D == 256; }

// Strides (page, token, head) of the codes in bytes, each a multiple of a row, so that
// the scales' sixteenths of them are whole rows too. The tokens of a page are evenly
// spaced and a page is a whole number of them away from the next.
static int fp4_cache(Fp4Cache &c, const void *k, const void *v, const void *ks, const void *vs, const int64_t *strides,
                     int page_size, int num_pages, int D) {
  const int64_t row = D / 2;
  for (int a = 0; a < 3; ++a)
    if (strides[a] < 0 || strides[a] % row != 0) return PBGDN_ERR_INVALID_ARGUMENT;
  if ((num_pages > 1 || page_size > 1) && (strides[1] <= 0 || strides[0] % strides[1] != 0)) return PBGDN_ERR_INVALID_ARGUMENT;
  if (num_pages > 0 && (!k || !v || !ks || !vs || !aligned16(k) || !aligned16(v) || !aligned16(ks) || !aligned16(vs)))
    return PBGDN_ERR_INVALID_ARGUMENT;
  c.k = static_cast<unsigned char *>(const_cast<void *>(k));
  c.v = static_cast<unsigned char *>(const_cast<void *>(v));
  c.k_scale = static_cast<unsigned char *>(const_cast<void *>(ks));
  c.v_scale = static_cast<unsigned char *>(const_cast<void *>(vs));
  c.page_stride = strides[0];
  c.token = strides[1];
  c.head = strides[2];
  c.total = static_cast<long>(num_pages) * page_size;
  c.page = page_size;
  return PBGDN_OK;
}

}  // namespace pbgdn

extern "C" size_t pbattn_fp4_decode_workspace_size(int B, int T, int Hq, int Hk, int D) {
  using namespace pbgdn;
  if (!decode_sizes_ok(B, T, Hq, Hk, D) || !fp4_width(D)) return 0;
  const int rows = Hq / Hk * T;
  const size_t slots = static_cast<size_t>(fp4_target(Hk, rows, D, fp4_heads(Hk, rows, D, true))) + B;
  return slots * Hk * rows * (D * sizeof(float) + sizeof(float2));
}

extern "C" int pbattn_fp4_decode(const void *q, int dtype, const void *k_cache, const void *v_cache, const void *k_scale,
                                 const void *v_scale, const int64_t *strides, int page_size, int num_pages,
                                 const int32_t *page_table, int max_pages, const int32_t *lengths, void *o, float *lse,
                                 int B, int T, int Hq, int Hk, int D, float scale, int window, int sinks, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  using namespace pbgdn;
  if (!decode_sizes_ok(B, T, Hq, Hk, D) || !attn_dtype(dtype) || !strides || page_size <= 0 || num_pages < 0 ||
      max_pages < 0 || sinks < 0 || !(scale - scale == 0.0f)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (!fp4_width(D)) return PBGDN_ERR_UNSUPPORTED;
  if (B == 0) return PBGDN_OK;
  if (!q || !o || !lengths || (max_pages > 0 && !page_table) || !workspace || !aligned16(q) || !aligned16(o) ||
      !aligned16(workspace)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  Fp4Cache cache;
  const int status = fp4_cache(cache, k_cache, v_cache, k_scale, v_scale, strides, page_size, num_pages, D);
  if (status != PBGDN_OK) return status;
  const long pages = num_pages > 0 ? num_pages - 1 : 0;
  const long reach = (cache.page_stride / 16) * pages + (cache.token / 16) * (page_size - 1L);
  if (reach > 0xffffffffL) return PBGDN_ERR_UNSUPPORTED;
  const bool near = reach < (1L << 28) - D / 32;  // (a row's own bytes within 4 GiB, too)
  const int heads = fp4_heads(Hk, Hq / Hk * T, D, near && cache.head == D / 2);
  if (workspace_bytes < pbattn_fp4_decode_workspace_size(B, T, Hq, Hk, D)) return PBGDN_ERR_INVALID_ARGUMENT;
  Fp4DecodeParams pp{};
  DecodeParams &p = pp.d;
  p.q = static_cast<const unsigned char *>(q);
  p.k = cache.k;
  p.v = cache.v;
  pp.k_scale = cache.k_scale;
  pp.v_scale = cache.v_scale;
  p.head = cache.head;
  pp.page_step = static_cast<uint32_t>(pages > 0 ? cache.page_stride / 16 : 0);
  pp.token_step = static_cast<uint32_t>(page_size > 1 ? cache.token / 16 : 0);
  // with 2^(s - 1) < page <= 2^s, floor(2^(31 + s) / page) + 1 is 2^(31 + s) / page and at
  // most one more, which adds less than 1 / page to any quotient below 2^31 / page
  while ((1L << pp.page_shift) < page_size) ++pp.page_shift;
  pp.page_mul = static_cast<uint32_t>((1ULL << (31 + pp.page_shift)) / page_size + 1);
  p.page = page_size;
  p.num_pages = max_pages > 0 ? num_pages : 0;  // (no table: no keys)
  p.max_pages = max_pages;
  p.table = page_table;
  p.lengths = lengths;
  p.o = o;
  p.lse = lse;
  decode_call(p, B, T, Hq, Hk, scale, window, sinks, fp4_target(Hk, Hq / Hk * T, D, heads));
  const size_t used = decode_workspace(p, workspace, D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  debug_poison(o, static_cast<size_t>(B) * T * Hq * D * attn_bytes(dtype), s);
  if (lse) debug_poison(lse, static_cast<size_t>(B) * T * Hq * sizeof(float), s);
  debug_poison(workspace, used, s);
  switch (dtype) {
    case PBGDN_F32: return dispatch_fp4<PBGDN_F32>(pp, D, near, heads, s);
    case PBGDN_BF16: return dispatch_fp4<PBGDN_BF16>(pp, D, near, heads, s);
    default: return dispatch_fp4<PBGDN_F16>(pp, D, near, heads, s);
  }
}

extern "C" int pbattn_fp4_write(const void *k, const void *v, int dtype, const int64_t *kv_strides, void *k_cache,
                                void *v_cache, void *k_scale, void *v_scale, const int64_t *strides, int page_size,
                                int num_pages, const int64_t *slots, int N, int Hk, int D, void *stream) {
  using namespace pbgdn;
  if (N < 0 || Hk <= 0 || D <= 0 || !attn_dtype(dtype) || !kv_strides || !strides || page_size <= 0 || num_pages < 0) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (!fp4_width(D) || static_cast<long>(Hk) * D > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  if (N == 0 || num_pages == 0) return PBGDN_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return PBGDN_ERR_INVALID_ARGUMENT;
  const int bytes = attn_bytes(dtype);
  for (int a = 0; a < 4; ++a)
    if (kv_strides[a] < 0 || kv_strides[a] * bytes % 16 != 0) return PBGDN_ERR_INVALID_ARGUMENT;
  Fp4WriteParams p{};
  const int status = fp4_cache(p.cache, k_cache, v_cache, k_scale, v_scale, strides, page_size, num_pages, D);
  if (status != PBGDN_OK) return status;
  p.k = static_cast<const unsigned char *>(k);
  p.v = static_cast<const unsigned char *>(v);
  p.k_token = kv_strides[0] * bytes;
  p.k_head = kv_strides[1] * bytes;
  p.v_token = kv_strides[2] * bytes;
  p.v_head = kv_strides[3] * bytes;
  p.slots = slots;
  p.eighths = D / 8;
  p.N = N;
  p.Hk = Hk;
  const long want = (static_cast<long>(N) * Hk * p.eighths + 255) / 256;
  const dim3 grid(static_cast<unsigned>(want < 65536 ? want : 65536));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case PBGDN_F32: hipLaunchKernelGGL(fp4_write_kernel<PBGDN_F32>, grid, dim3(256), 0, s, p); break;
    case PBGDN_BF16: hipLaunchKernelGGL(fp4_write_kernel<PBGDN_BF16>, grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL(fp4_write_kernel<PBGDN_F16>, grid, dim3(256), 0, s, p); break;
  }
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

extern "C" int pbattn_fp4_read(const void *k_cache, const void *v_cache, const void *k_scale, const void *v_scale,
                               const int64_t *strides, int page_size, int num_pages, const int32_t *page_table,
                               int max_pages, const int32_t *lengths, void *k, void *v, int dtype, int32_t *cu_seqlens,
                               int B, int tokens, int Hk, int D, void *stream) {
  using namespace pbgdn;
  if (B < 0 || tokens < 0 || Hk <= 0 || D <= 0 || !attn_dtype(dtype) || !strides || page_size <= 0 || num_pages < 0 ||
      max_pages < 0) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (!fp4_width(D) || B > MAX_REQUESTS || static_cast<long>(Hk) * D > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  if (!cu_seqlens || (B > 0 && !lengths) || (B > 0 && max_pages > 0 && !page_table) ||
      (tokens > 0 && (!k || !v || !aligned16(k) || !aligned16(v)))) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  Fp4ReadParams p{};
  const int status = fp4_cache(p.cache, k_cache, v_cache, k_scale, v_scale, strides, page_size, num_pages, D);
  if (status != PBGDN_OK) return status;
  p.table = page_table;
  p.lengths = lengths;
  p.k = k;
  p.v = v;
  p.cu = cu_seqlens;
  p.B = B;
  p.max_pages = max_pages;
  p.tokens = tokens;
  p.Hk = Hk;
  p.eighths = D / 8;
  p.num_pages = num_pages;
  // Tokens of a workgroup: as many as leave the GPU eight workgroups a CU, READ_TOKENS at most.
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  const long even = (tokens + 8L * shape.cus - 1) / (8L * shape.cus);
  p.per_block = static_cast<int>(even < 1 ? 1 : even > READ_TOKENS ? READ_TOKENS : even);
  while (p.per_block > 1 && static_cast<long>(p.per_block) * Hk * p.eighths > 0x3fffffffL) p.per_block /= 2;  // (32-bit counts)
  const long blocks = (tokens + static_cast<long>(p.per_block) - 1) / p.per_block;
  if (blocks > MAX_BLOCKS) return PBGDN_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks > 0 ? blocks : 1));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t bytes = static_cast<size_t>(tokens) * Hk * D * attn_bytes(dtype);
  debug_poison(k, bytes, s);
  debug_poison(v, bytes, s);
  debug_poison(cu_seqlens, (B + 1) * sizeof(int32_t), s);
  switch (dtype) {
    case PBGDN_F32: hipLaunchKernelGGL(fp4_read_kernel<PBGDN_F32>, grid, dim3(SCAN_THREADS), 0, s, p); break;
    case PBGDN_BF16: hipLaunchKernelGGL(fp4_read_kernel<PBGDN_BF16>, grid, dim3(SCAN_THREADS), 0, s, p); break;
    default: hipLaunchKernelGGL(fp4_read_kernel<PBGDN_F16>, grid, dim3(SCAN_THREADS), 0, s, p); break;
  }
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}
