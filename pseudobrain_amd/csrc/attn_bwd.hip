// Windowed attention, backward (pbattn_window_bwd).
//
// Four kernels, none with an atomic sum:
//   range_kernel  float16: the maxima that bound ds
//   dq_kernel     the forward's walk over keys: S^T, dP^T, dS^T, dQ^T += K^T dS^T;
//                 before it, per row, lse in powers of two and delta = do . o - dlse
//                 (made exact where rows see few keys), which it keeps for
//                 dkdv_kernel by (batch, key head) in the row order of the tiles
//   dkdv_kernel   a wave owns 32 keys, with K and V rows and the sums of dK^T
//                 and dV^T in registers, and walks the queries that see them
//                 (all heads of the group): S = Q K^T, P, dV^T += dO^T P,
//                 dP = dO V^T, dS, dK^T += Q^T dS. Long or few walks are split
//                 into parts; the sinks, which every later query sees, are
//                 always walked in parts beyond their window
//   join_kernel   sums of parts, in a fixed order
// Recomputing S and dP on both sides costs two products of seven, and saves
// float32 sums of dQ in memory and their atomics.
//
// Forward and backward of 8,192 tokens, 32 heads of 128 on 8, float16, take 2.46
// to 2.59 ms: 740 to 780 TFLOP/s of the formulas' flops, 950 to 1,000 with the two
// products formed twice, where a large product reaches 1,296. In it the forward
// takes 600 us, range_kernel 25, dq_kernel 800 (matrix unit busy 65%), dkdv_kernel
// 1,180 (54%), join_kernel 27.
#include <atomic>

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

// Weights are exp2(s c - lse), with lse in powers of two as one float32: off by up to
// 2^-23 |lse|. In rows whose |lse| (natural) is beyond this, where that would reach
// 2^-13, dq_kernel finds the largest score and the sum again; the largest is then the
// row's origin, which its scores lose before they are scaled, and lse the sum's
// logarithm alone. Workgroups that meet such rows (`has_large`) go the masked tiles'
// way throughout, and take the origins off there.
constexpr float LARGE_LSE = 1024.0f;

// float16: dkdv_kernel's weights, at most 1, are held times 2^14, for beside many
// keys they are small: 1.5 million alike came out 1.6% off in dV as multiples of 2^-24.
constexpr int F16_WEIGHTS = 14;

constexpr int QR = 32;            // rows of a query tile of dkdv_kernel
constexpr int DQ_WAVES = 4, DQ_ROWS = 32 * DQ_WAVES;  // waves and rows of a workgroup of dq_kernel
// Rows (or a token's heads if more) of one part of the sinks' walk, by how many
// sinks there are: a part's sums, two float32 rows a sink, against the rows of Q and
// dO that each 32 sinks read. 16 rows a sink keep what the sums write to an eighth of
// one such reading in 16 bits; past 256 sinks, where a part stays 4,096 rows, the sums
// grow with the sinks (to twice one reading at 4,096), and so does the number of
// readings.
constexpr int tail_rows(int sinks) { return sinks < 8 ? 128 : sinks < 256 ? 16 * sinks : 4096; }
constexpr int MAX_PARTS = 16;     // parts of an ordinary key tile's walk

struct BwdParams {
  WindowParams f;
  const void *grad_o, *o;
  const float *lse, *grad_lse;
  void *dq, *dk, *dv;
  float2 *stat;       // [B][Hk][Tq G]: (lse log2(e), for float16 less F16_WEIGHTS; delta); +inf for a row that sees nothing
  float *origin;      // as stat: zero but for rows of large scores
  int *has_large;     // [B][Hk][f.slots]: a tile of dq_kernel has such a row
  uint32_t *range;    // float16: bits of max |do|, |v|, |dlse|
  float *part;        // [2][parts][B][Hk][Tk][D] when parts > 1
  float *tail;        // [2][tail slots][Hk][sinks][D]
  float scale;
  int B, D;
  int parts;          // parts of a key tile's walk
  int key_slots;      // key tiles of a (batch, key head)
  int sinks;          // keys that stay visible, 0 when no query is beyond their window
  int tail_tokens;    // query tokens of one part of the sinks' walk
  int tail_slots;     // parts of the sinks' walk over all long sequences, and slot 0 of each: the window's own part
  // query tiles: `heads` heads of `tokens` tokens each, `splits` tiles for the heads of a token
  int heads, tokens, splits;
};

// The sinks' parts belong to the long sequences, those of more keys than the window
// (in the others no query is beyond it). In a packed call a long sequence's number is
// at most its place, and at most the windows' worths of keys before it: it has no
// other's number, whose sequence would lie a window and a key further on.
__device__ __forceinline__ bool is_long(const WindowParams &f, const Seq &sq) { return sq.nk > f.window; }
__device__ __forceinline__ int long_number(const WindowParams &f, int seq) {
  if (!f.cu_q) return seq;
  const int before = boundary(f.cu_k ? f.cu_k : f.cu_q, seq, f.Tk) / (f.window + 1);
  return seq < before ? seq : before;
}
inline int long_most(const WindowParams &f) {
  const int most = f.Tk / (f.window + 1);
  return f.cu_q && most < f.nseq ? most : f.nseq;
}
// A long sequence's slots: the window's part, then one per tail_tokens tokens.
__device__ __forceinline__ int tail_start(const BwdParams &p, int seq) {
  if (!p.f.cu_q) return seq * ((p.f.Tq + p.tail_tokens - 1) / p.tail_tokens + 1);
  return boundary(p.f.cu_q, seq, p.f.Tq) / p.tail_tokens + 2 * long_number(p.f, seq);
}
inline long tail_slot_count(const WindowParams &f, int tokens) {
  return f.cu_q ? f.Tq / tokens + 2L * long_most(f) : f.nseq * ((f.Tq + tokens - 1L) / tokens + 1);
}

// The last of the boundaries 0 .. n that is no further than `token`: its sequence, or n past the last.
__device__ __forceinline__ int last_at(const int32_t *cu, int n, int total, int token) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (boundary(cu, mid, total) <= token)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// float16's range: o is a mean of the values its row sees, so |delta| and |dp| are
// at most D max |do| max |v| (and max |dlse|), and ds their sum; a power of two
// brings that bound to 2^14.
// ---------------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ float range_scale(const uint32_t *range) {
  if constexpr (DT != PBGDN_F16) return 1.0f;
  const float bound = 2.0f * D * __uint_as_float(range[0]) * __uint_as_float(range[1]) + __uint_as_float(range[2]);
  if (!(bound > 0.0f && bound < 1e30f)) return 1.0f;
  int e;
  frexpf(bound, &e);
  e = 14 - e;
  e = e > 100 ? 100 : e < -100 ? -100 : e;
  return ldexpf(1.0f, e);
}

__global__ void range_zero_kernel(uint32_t *range) {
  if (threadIdx.x < 4) range[threadIdx.x] = 0;
}

// A workgroup's maximum into a word of `range`: one atomic, and none when the
// word holds as much (maxima do not depend on their order).
__device__ __forceinline__ void range_max(float x, uint32_t *word) {
  __shared__ float top[4];
  x = wave_max(x);
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t bits = __float_as_uint(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
    if (bits > __hip_atomic_load(word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(word, bits);
  }
  __syncthreads();
}

// max |do|, |dlse| and |v| of what takes part: the queries that see a key and the
// keys that a query sees. Infinities (and NaN) are left out: what they reach is not
// finite by any scale, and the rest keeps its own. Three quarters of the workgroups
// read grad_o, the rest v, a run of tokens each (8,192 tokens, 32 heads of 128 on 8:
// 84 MB in 22 to 27 us).
template <int D>
__global__ __launch_bounds__(256) void range_kernel(const BwdParams p) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;  // lanes of a row, rows of a workgroup
  const WindowParams &f = p.f;
  const int split = gridDim.x * 3 / 4, unit = threadIdx.x % LPR * 16, first = threadIdx.x / LPR;
  const auto finite = [](float x) { return x < INFINITY ? x : 0.0f; };
  const auto largest = [&](const unsigned char *src, float top) {
    const half8_t x = *reinterpret_cast<const half8_t *>(src + unit);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, finite(fabsf(static_cast<float>(x[i]))));
    return top;
  };
  float top = 0.0f, top_dlse = 0.0f;
  if (static_cast<int>(blockIdx.x) < split) {
    const long rows = static_cast<long>(p.B) * f.Tq * f.Hq;
    for (long r = blockIdx.x * static_cast<long>(RPB) + first; r < rows; r += split * static_cast<long>(RPB)) {
      if (p.lse[r] == -INFINITY) continue;
      top = largest(static_cast<const unsigned char *>(p.grad_o) + r * D * 2, top);
      if (p.grad_lse && unit == 0) top_dlse = fmaxf(top_dlse, finite(fabsf(p.grad_lse[r])));
    }
    range_max(top, p.range);
    if (p.grad_lse) range_max(top_dlse, p.range + 2);
    return;
  }
  const long tokens = static_cast<long>(p.B) * f.Tk, blocks = gridDim.x - split;
  const long per = (tokens + blocks - 1) / blocks, t0 = (blockIdx.x - split) * per;
  const long t1 = t0 + per < tokens ? t0 + per : tokens;
  int seq = 0;
  for (long r = t0 * f.Hk + first; r < t1 * f.Hk; r += RPB) {
    const long bt = r / f.Hk, b = bt / f.Tk;
    int key = static_cast<int>(bt - b * f.Tk);
    const unsigned char *src = f.v.base + b * f.v.batch + key * f.v.token + (r - bt * f.Hk) * f.v.head;
    if (f.cu_q) {
      const int32_t *cu = f.cu_k ? f.cu_k : f.cu_q;
      if (r < t0 * f.Hk + RPB) seq = last_at(cu, f.nseq, f.Tk, key);
      while (seq < f.nseq && boundary(cu, seq + 1, f.Tk) <= key) ++seq;
      if (seq == f.nseq) break;  // this token and those after belong to no sequence
    } else {
      seq = static_cast<int>(b);
    }
    const Seq sq = sequence<true>(f.cu_q, f.cu_k, seq, f.nseq, f.Tq, f.Tk);
    key -= sq.k0;
    if (sq.nq > 0 && (key > sq.nk - sq.nq - f.window || key < f.sinks)) top = largest(src, top);
  }
  range_max(top, p.range + 1);
}

// ---------------------------------------------------------------------------
// dK and dV. TAIL: the sinks' keys against the queries beyond their window.
//
// Four waves share a staged tile of 32 rows of Q and dO (LDS reads of it feed all
// four products), each with 32 keys of its own. Up to D = 128 in 16 bits two
// workgroups fit a CU, two waves a SIMD; at D = 256 the sums alone take 256
// registers and one wave has a SIMD to itself, so its waits are not covered: 4 x
// 2,048 tokens, 32 heads of 128 on 8, window 1,024: 270 to 300 us (700 TFLOP/s,
// the matrix unit busy 38%); 6,011 tokens in 7 sequences, 16 heads of 256 on 2,
// window 512: 182 to 190 us (390 TFLOP/s, 20%). The sinks' walk reads all of Q and
// dO again for a few keys: 26 us there, 28 to 31 us for 4 x 2,048 tokens.
// ---------------------------------------------------------------------------
template <int DT, int D, int NW>
struct Dkdv {
  using L = Tile<DT, D>;
  static constexpr int BN = 32 * NW, TILE = QR * L::ROW, STAT = QR * 16, BUF = 2 * TILE + STAT, LDS = 2 * BUF;
  static constexpr int LOADS = QR / L::PER_DMA;  // of one tensor, all waves
  // Registers hold the sums, and K and V rows where they find room beside them
  // (two waves a SIMD up to D = 128 in 16 bits): otherwise LDS does.
  static constexpr bool HELD = L::ROW <= 512, V_HELD = HELD && (D != 128 || L::E::BYTES == 4);
  static constexpr int VS = HELD ? 0 : BN * L::ROW, KV = VS + (V_HELD ? 0 : BN * L::ROW);  // V's place, both sizes
  static constexpr int BUFS = KV + 2 * BUF <= 160 * 1024 ? 2 : 1;
  static constexpr int BYTES = KV + BUFS * BUF;
};

template <int DT, int D, int NW, bool TAIL, int WAVES>
__global__ __launch_bounds__(NW * 64, WAVES) void dkdv_kernel(const BwdParams p) {
  using K = Dkdv<DT, D, NW>;
  using L = typename K::L;
  using E = typename L::E;
  constexpr int S = L::STEPS, MB = L::MB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  PBGDN_POISON_LDS(lds, K::BYTES);
  PBGDN_POISON_SYNC();

  const WindowParams &f = p.f;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5, G = f.group;

  // which keys, which part of their queries
  int b, hk, seq, tile, part, slot = 0;
  if constexpr (TAIL) {
    int id = blockIdx.x;
    const int sink_tiles = (p.sinks + 31) / 32;
    tile = uniform(id % sink_tiles);
    id /= sink_tiles;
    hk = uniform(id % f.Hk);
    slot = uniform(id / f.Hk);
    // bisection over the sequences' first slots: a long one's are past those of all before it
    int lo = 0, hi = f.nseq - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tail_start(p, mid) <= slot)
        lo = mid;
      else
        hi = mid - 1;
    }
    seq = uniform(lo);
    b = f.cu_q ? 0 : seq;
    part = slot - tail_start(p, seq) - 1;
  } else {
    const int groups = gridDim.x / (p.key_slots * p.parts);
    int grp, s;
    place(blockIdx.x, groups, p.key_slots * p.parts, grp, s);
    s = p.key_slots * p.parts - 1 - s;  // the first keys, which most queries see, first
    b = uniform(grp / f.Hk);
    hk = grp - b * f.Hk;
    tile = uniform(s / p.parts);
    part = s - tile * p.parts;
    seq = b;
    const int32_t *cu = f.cu_k ? f.cu_k : f.cu_q;
    if (f.cu_q) {
      seq = slot_sequence(cu, f.nseq, f.Tk, 1, K::BN, tile);
      tile = uniform(tile - slot_start(cu, seq, f.Tk, 1, K::BN));
    }
  }
  const Seq sq = sequence<true>(f.cu_q, f.cu_k, seq, f.nseq, f.Tq, f.Tk);
  const int j0 = tile * K::BN;
  if (part < 0 || tile < 0 || j0 >= sq.nk || (TAIL && !is_long(f, sq))) return;
  const int off = sq.nk - sq.nq;  // position of query token 0

  // the query tokens [t0, t1) of this part
  int t0, t1;
  if constexpr (TAIL) {
    t0 = j0 + f.window - off;  // the first beyond the window of the tile's first key
    t0 = t0 > 0 ? t0 : 0;
    const int from = part * p.tail_tokens;
    if (from >= sq.nq) return;
    t0 = t0 > from ? t0 : from;
    t1 = sq.nq - from > p.tail_tokens ? from + p.tail_tokens : sq.nq;
  } else {
    const int jl = (j0 + K::BN < sq.nk ? j0 + K::BN : sq.nk) - 1;
    t0 = j0 - off > 0 ? j0 - off : 0;
    t1 = jl < sq.nk - f.window ? jl + f.window - off : sq.nq;
    t1 = t1 < 0 ? 0 : t1;
    if (p.parts > 1) {
      int step = (t1 - t0 + p.parts - 1) / p.parts;
      step = uniform((step + p.tokens - 1) / p.tokens * p.tokens);
      t0 = t0 + part * step;
      t1 = t1 < t0 + step ? t1 : t0 + step;
    }
  }
  const int tiles = uniform(t1 > t0 ? (t1 - t0 + p.tokens - 1) / p.tokens * p.splits : 0);

  // whether the tiles of dq_kernel that those tokens' rows lie in have rows of large scores
  int some_large = 0;
  if (tiles > 0) {
    const int *flags = p.has_large + (static_cast<long>(b) * f.Hk + hk) * f.slots +
                       (f.cu_q ? slot_start(f.cu_q, seq, f.Tq, G, DQ_ROWS) : 0);
    const int last = (t1 * G - 1) / DQ_ROWS;
    int s = t0 * G / DQ_ROWS + lane;
    if (s <= last) some_large = flags[s];
    if (uniform(s) + 64 <= last) {
      for (s += 64; s <= last; s += 64) some_large |= flags[s];
    }
  }

  // this wave's keys
  const int key = j0 + wave * 32 + n;
  const int kc = key < sq.nk ? key : sq.nk - 1;
  const unsigned char *krow = f.k.base + b * f.k.batch + hk * f.k.head + (sq.k0 + kc) * f.k.token;
  const unsigned char *vrow = f.v.base + b * f.v.batch + hk * f.v.head + (sq.k0 + kc) * f.v.token;
  v4u32_t kf[K::HELD ? S : 1], vf[K::V_HELD ? S : 1];
  unsigned char *const kl = lds + wave * 32 * L::ROW, *const vl = kl + K::VS;
  uint32_t rbase = L::rows_base(n, h), cbase = L::cols_base(lane);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    v4u32_t x = *reinterpret_cast<const v4u32_t *>(krow + (2 * s + h) * 16);
    if (f.negate) x ^= E::BYTES == 2 ? 0x80008000u : 0x80000000u;  // (K here serves the scores alone)
    const v4u32_t y = *reinterpret_cast<const v4u32_t *>(vrow + (2 * s + h) * 16);
    const uint32_t at = (rbase ^ ((2 * s) % 16 * 16)) + (2 * s) / 16 * 256;
    if constexpr (K::HELD)
      kf[s] = x;
    else
      *reinterpret_cast<v4u32_t *>(kl + at) = x;
    if constexpr (K::V_HELD)
      vf[s] = y;
    else
      *reinterpret_cast<v4u32_t *>(vl + at) = y;
  }

  if constexpr (K::HELD) {
#pragma unroll
    for (int s = 0; s < S; ++s) settle(kf[s]);
  }
  if constexpr (K::V_HELD) {
#pragma unroll
    for (int s = 0; s < S; ++s) settle(vf[s]);
  }
  some_large = __any(some_large);
  float16_t dk[MB], dv[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) dk[m] = dv[m] = zero16();
  const float unit = DT == PBGDN_F16 ? ldexpf(1.0f, -F16_WEIGHTS) : 1.0f, scale16 = range_scale<DT, D>(p.range);
  const float range = scale16 * unit;  // of dS, beside the weights' own

  // Staging of the query tiles in turn: `tokens` tokens of `heads` heads, or the
  // heads of a token in `splits` tiles. A lane's offsets into a tile do not change;
  // a lane past the tile's tokens (or heads, where they are split) stages zeros.
  const uint32_t inv = 65536 / p.heads + 1;  // row / heads = row inv >> 16 for rows below 32
  const long g_token = static_cast<long>(f.Hq) * L::ROW;
  constexpr int PER_WAVE = (K::LOADS + NW - 1) / NW;
  const auto offsets = [&](int lane, int w, uint32_t &q_at, uint32_t &g_at, int &index) __attribute__((always_inline)) {
    const int row = (wave + NW * w) * L::PER_DMA + lane / L::UNITS;
    const int tt = static_cast<int>((row * inv) >> 16), gg = row - tt * p.heads;
    const uint32_t unit = ((lane % L::UNITS) ^ L::swz(row)) * 16;
    q_at = tt * static_cast<uint32_t>(f.q.token) + gg * static_cast<uint32_t>(f.q.head) + unit;
    g_at = tt * static_cast<uint32_t>(g_token) + gg * L::ROW + unit;
    index = p.splits == 1 ? tt : gg;
  };
  constexpr bool AT_HELD = K::HELD && PER_WAVE <= 2;  // kept in registers, or worked out at each tile
  uint32_t q_at[AT_HELD ? PER_WAVE : 1], g_at[AT_HELD ? PER_WAVE : 1];
  int index[AT_HELD ? PER_WAVE : 1];
  if constexpr (AT_HELD) {
#pragma unroll
    for (int w = 0; w < PER_WAVE; ++w) offsets(lane, w, q_at[w], g_at[w], index[w]);
  }
  const unsigned char *qp = f.q.base + b * f.q.batch + (sq.q0 + t0) * f.q.token + hk * G * f.q.head;
  const unsigned char *gp = static_cast<const unsigned char *>(p.grad_o) +
                            ((static_cast<long>(b) * f.Tq + sq.q0 + t0) * f.Hq + hk * G) * static_cast<long>(L::ROW);
  const float2 *sp = p.stat + ((static_cast<long>(b) * f.Hk + hk) * f.Tq + sq.q0 + t0) * G;
  const long q_size = (p.tokens - 1) * f.q.token + (p.heads - 1) * f.q.head + L::ROW;
  const long g_size = (p.tokens - 1) * g_token + p.heads * L::ROW;
  int st = t0, split = 0;  // of the tile to stage next
  unsigned char *const bufs = lds + K::KV;
  const auto stage = [&](int i) __attribute__((always_inline)) {
    const uint32_t to = uniform(lds_address(bufs + (K::BUFS == 2 ? (i & 1) * K::BUF : 0)));
    const int left = p.splits == 1 ? t1 - st : G - split * QR, most = p.splits == 1 ? p.tokens : QR;
    const int limit = left < most ? left : most;
    const v4u32_t dq_ = dma_desc(qp, q_size), dg_ = dma_desc(gp, g_size);
    const int lane_ = AT_HELD ? 0 : opaque(threadIdx.x & 63);
#pragma unroll
    for (int w = 0; w < PER_WAVE; ++w) {
      const int inst = wave + NW * w;
      uint32_t qa, ga;
      int x;
      if constexpr (AT_HELD)
        qa = q_at[w], ga = g_at[w], x = index[w];
      else
        offsets(lane_, w, qa, ga, x);
      const bool in = x < limit;
      dma(dq_, in ? qa : OUT_OF_RANGE, to + inst * 1024);
      dma(dg_, in ? ga : OUT_OF_RANGE, to + K::TILE + inst * 1024);
    }
    const long rows = limit * (p.splits == 1 ? G : 1);
    if (wave == 0) dma4(dma_desc(sp, rows * 8), lane * 4, to + 2 * K::TILE);
    if (wave == NW - 1) dma4(dma_desc(p.origin + (sp - p.stat), rows * 4), lane * 4, to + 2 * K::TILE + QR * 8);
    // on to the next
    if (++split == p.splits) {
      split = 0;
      st += p.tokens;
      qp += p.tokens * f.q.token - (p.splits - 1) * QR * f.q.head;
      gp += p.tokens * g_token - (p.splits - 1) * QR * L::ROW;
      sp += p.tokens * G - (p.splits - 1) * QR;
    } else {
      qp += QR * f.q.head;
      gp += QR * L::ROW;
      sp += QR;
    }
  };

  // Each wave computes with the tiles [lead, mine) whose queries see any of its
  // keys, in a loop without a way around the products (around one, the compiler
  // moves every accumulator between register files), and keeps step with the
  // others' staging before and after.
  const int w_lo = j0 + wave * 32, w_hi = w_lo + 31;
  int lead = 0, mine = tiles;
  if constexpr (TAIL) {
    if (w_lo >= f.sinks) mine = 0;
  } else {
    const int before = w_lo - off - t0, after = w_hi - t0 - off;  // tokens before the first that sees w_lo
    lead = uniform(before > 0 ? before / p.tokens * p.splits : 0);
    if (after < t1 - t0 - f.window) {  // tokens from after + window on see none
      const int n = (after + f.window + p.tokens - 1) / p.tokens * p.splits;
      mine = uniform(n < 0 ? 0 : n < tiles ? n : tiles);
    }
  }
  if (tiles > 0 && K::BUFS == 2) stage(0);
  const auto advance = [&](int i) __attribute__((always_inline)) {
    if constexpr (K::BUFS == 2) {
      wait_dma<0>();
      block_sync();
      if (i + 1 < tiles) stage(i + 1);
    } else {
      block_sync();
      stage(i);
      wait_dma<0>();
      block_sync();
    }
  };
  int i = 0;
  for (; i < lead && i < tiles; ++i) advance(i);
  for (; i < mine; ++i) {
    advance(i);
    const unsigned char *qt = bufs + (K::BUFS == 2 ? (i & 1) * K::BUF : 0), *gt = qt + K::TILE;
    const float4_t *stat = reinterpret_cast<const float4_t *>(qt + 2 * K::TILE);
    const int tok = t0 + (p.splits == 1 ? i : uniform(i / p.splits)) * p.tokens;
    const int p_lo = tok + off, p_hi = (tok + p.tokens < t1 ? tok + p.tokens : t1) - 1 + off;
    const bool whole = TAIL ? w_hi < f.sinks && w_hi <= p_lo - f.window : w_hi <= p_lo && w_lo > p_hi - f.window;

    rbase = opaque(rbase);
    cbase = opaque(cbase);
    float16_t x, y;
    if constexpr (K::HELD)
      L::template rows_product<1>(qt, rbase, kf, &x);
    else
      x = L::rows_product_lds(qt, kl, rbase);
    if constexpr (K::V_HELD)
      L::template rows_product<1>(gt, rbase, vf, &y);
    else
      y = L::rows_product_lds(gt, vl, rbase);
    if (!whole || some_large) {
      if (some_large) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4_t a = stat[QR / 2 + (2 * e + 4 * h) / 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) x[e + r] -= a[r];
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int pos = p_lo + static_cast<int>((acc_row(e, h) * inv) >> 16);
        const bool seen = TAIL ? (key < f.sinks) & (key <= pos - f.window) : (key <= pos) & (key > pos - f.window);
        x[e] = seen ? x[e] : -INFINITY;
        y[e] = seen ? y[e] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      // rows 2 e + 4 h .. + 3: (lse, delta) pairs
      const float4_t a = stat[e + 2 * h], c = stat[e + 2 * h + 1];
      const float lse[4] = {a[0], a[2], c[0], c[2]}, delta[4] = {a[1], a[3], c[1], c[3]};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[e + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e + r], f.c, -lse[r]));
        float d = y[e + r] - delta[r];
        if constexpr (DT == PBGDN_F16) d *= range;
        y[e + r] = x[e + r] * d;
      }
    }
    const typename L::Operand xo = L::operand(x), yo = L::operand(y);
    L::template cols_product<1>(gt, cbase, &xo, dv);
    L::template cols_product<1>(qt, cbase, &yo, dk);
  }
  for (; i < tiles; ++i) advance(i);

  if (key >= sq.nk || (TAIL && key >= p.sinks)) return;
  const float fk = p.scale / scale16;
  const long row = (static_cast<long>(b) * f.Tk + sq.k0 + key) * f.Hk + hk;
  if constexpr (TAIL) {
    const long at = ((static_cast<long>(slot) * f.Hk + hk) * p.sinks + key) * D;
    const long half = static_cast<long>(p.tail_slots) * f.Hk * p.sinks * D;
    store_row<PBGDN_F32, D>(p.tail + at, dk, h, fk);
    store_row<PBGDN_F32, D>(p.tail + half + at, dv, h, unit);
  } else if (p.parts > 1) {
    const long half = static_cast<long>(p.B) * f.Tk * f.Hk * D;
    store_row<PBGDN_F32, D>(p.part + part * half + row * D, dk, h, fk);
    store_row<PBGDN_F32, D>(p.part + (p.parts + part) * half + row * D, dv, h, unit);
  } else if (key < p.sinks && seq < f.nseq && is_long(f, sq)) {
    const long at = ((static_cast<long>(tail_start(p, seq)) * f.Hk + hk) * p.sinks + key) * D;
    const long half = static_cast<long>(p.tail_slots) * f.Hk * p.sinks * D;
    store_row<PBGDN_F32, D>(p.tail + at, dk, h, fk);
    store_row<PBGDN_F32, D>(p.tail + half + at, dv, h, unit);
  } else {
    store_row<DT, D>(static_cast<unsigned char *>(p.dk) + row * L::ROW, dk, h, fk);
    store_row<DT, D>(static_cast<unsigned char *>(p.dv) + row * L::ROW, dv, h, unit);
  }
}

// Sums the parts of dk and dv, in a fixed order. The first `sink_blocks`
// workgroups take a sink each (of a long sequence and key head): its threads, four
// elements of the row each, split the many parts and join through LDS. The rest
// take the other keys where p.parts > 1, four elements a thread. Bound by the
// parts' reads (5 parts of 6,011 keys, 2 heads of 256: 123 MB in 23 us).
template <int DT>
__device__ __forceinline__ void store4(void *dst, long at, float4_t x) {
  using E = Elem<DT>;
  if constexpr (E::BYTES == 2)
    reinterpret_cast<v2u32_t *>(dst)[at / 4] = v2u32_t{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
  else
    reinterpret_cast<float4_t *>(dst)[at / 4] = x;
}
template <int DT, int D>
__global__ __launch_bounds__(256) void join_kernel(const BwdParams p, int sink_blocks) {
  const WindowParams &f = p.f;
  constexpr int TPR = D / 4, GROUPS = 256 / TPR;
  __shared__ __attribute__((aligned(16))) float sums[GROUPS][D];
  const long half = static_cast<long>(p.B) * f.Tk * f.Hk * D;
  if (static_cast<int>(blockIdx.x) < sink_blocks) {
    int id = blockIdx.x;
    const int key = id % p.sinks;
    id /= p.sinks;
    const int hk = id % f.Hk, number = id / f.Hk;
    int seq = number;
    if (f.cu_q) {  // the last sequence that has no higher number, if it is the long one of this
      int lo = 0, hi = f.nseq - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (long_number(f, mid) <= number)
          lo = mid;
        else
          hi = mid - 1;
      }
      seq = lo;
    }
    const Seq sq = sequence<true>(f.cu_q, f.cu_k, seq, f.nseq, f.Tq, f.Tk);
    if (key >= sq.nk || !is_long(f, sq) || long_number(f, seq) != number) return;
    const long row = ((f.cu_q ? 0 : static_cast<long>(seq) * f.Tk) + sq.k0 + key) * f.Hk + hk;
    const int tails = (sq.nq + p.tail_tokens - 1) / p.tail_tokens;
    const int d = threadIdx.x % TPR * 4, group = threadIdx.x / TPR;
    const long tail_half = static_cast<long>(p.tail_slots) * f.Hk * p.sinks * D;
    const long tail = ((static_cast<long>(tail_start(p, seq)) * f.Hk + hk) * p.sinks + key) * D + d;
    const long step = static_cast<long>(f.Hk) * p.sinks * D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.parts > 1)
        for (int a = group; a < p.parts; a += GROUPS)
          sum += *reinterpret_cast<const float4_t *>(p.part + (which * p.parts + a) * half + row * D + d);
#pragma unroll 4
      for (int a = group + (p.parts > 1); a <= tails; a += GROUPS)  // (slot 0: the window's, where it has no parts)
        sum += *reinterpret_cast<const float4_t *>(p.tail + which * tail_half + tail + a * step);
      __syncthreads();
      *reinterpret_cast<float4_t *>(&sums[group][d]) = sum;
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int g = 1; g < GROUPS; ++g) sum += *reinterpret_cast<const float4_t *>(&sums[g][d]);
        store4<DT>(which ? p.dv : p.dk, row * D + d, sum);
      }
    }
    return;
  }
  const long n = static_cast<long>(p.B) * f.Tk * f.Hk * TPR, blocks = gridDim.x - sink_blocks;
  for (long i = (blockIdx.x - sink_blocks) * 256L + threadIdx.x; i < n; i += blocks * 256L) {
    const long row = i / TPR;
    const int d = static_cast<int>(i - row * TPR) * 4;
    if (p.sinks) {  // the sinks are taken above
      const long token = row / f.Hk;
      int seq = static_cast<int>(token / f.Tk), key = static_cast<int>(token - static_cast<long>(seq) * f.Tk);
      if (f.cu_q) {
        const int32_t *cu = f.cu_k ? f.cu_k : f.cu_q;
        seq = last_at(cu, f.nseq, f.Tk, key);
        key -= boundary(cu, seq, f.Tk);
      }
      if (key < p.sinks && seq < f.nseq && is_long(f, sequence<true>(f.cu_q, f.cu_k, seq, f.nseq, f.Tq, f.Tk))) continue;
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for (int a = 0; a < p.parts; ++a)
        sum += *reinterpret_cast<const float4_t *>(p.part + (which * p.parts + a) * half + row * D + d);
      store4<DT>(which ? p.dv : p.dk, row * D + d, sum);
    }
  }
}

// ---------------------------------------------------------------------------
// dQ: the forward's rows and walk.
//
// delta = do . o is taken from an o that the forward rounded to 16 bits, after
// weights of 16 bits: with few keys, whose weights are large, that is as much as
// the rounding of dS itself (17 keys, bf16: dq 0.0029 of its norm off, with an
// exact delta 0.0024; 1,024 keys 0.0025 and 0.0024). As the sum of dS over a
// row's keys is dlse, what it comes to instead is delta's error. Where a walk is
// of 128 keys at most, the rows walk once for that sum, and again with the delta
// corrected by it, which is kept for dkdv_kernel, so this kernel comes first.
//
// 4 x 2,048 tokens, 32 heads of 128 on 8, window 1,024: 187 to 211 us (770
// TFLOP/s, the matrix unit busy 46%); 6,011 tokens in 7 sequences, 16 heads of 256
// on 2, window 512: 122 to 127 us at one wave a SIMD (430 TFLOP/s, 21%). Reading o for
// delta takes 4 to 15 us of it; a pass of its own over o and grad_o took 18 to 37.
// ---------------------------------------------------------------------------
template <int DT, int D, int NW, int BN>
struct Dq {
  using L = Tile<DT, D>;
  static constexpr int BM = 32 * NW, TILE = BN * L::ROW, LDS = 4 * TILE;
  static constexpr int EXACT_TILES = DT == PBGDN_F32 ? 0 : 128 / BN;  // walks whose delta is corrected
};

template <int DT, int D, int NW, int BN, int WAVES>
__global__ __launch_bounds__(NW * 64, WAVES) void dq_kernel(const BwdParams p) {
  using F = Dq<DT, D, NW, BN>;
  using L = typename F::L;
  using E = typename L::E;
  constexpr int S = L::STEPS, MB = L::MB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  PBGDN_POISON_LDS(lds, F::LDS);
  PBGDN_POISON_SYNC();

  const WindowParams &f = p.f;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5, G = f.group;
  const int groups = gridDim.x / f.slots;
  int grp, slot;
  place(blockIdx.x, groups, f.slots, grp, slot);
  int *const has_large = p.has_large + grp * static_cast<long>(f.slots) + slot;
  const int b = uniform(grp / f.Hk), hk = grp - b * f.Hk;
  int seq = b;
  if (f.cu_q) {
    seq = slot_sequence(f.cu_q, f.nseq, f.Tq, G, F::BM, slot);
    slot = uniform(slot - slot_start(f.cu_q, seq, f.Tq, G, F::BM));
  }
  const Seq sq = sequence<false>(f.cu_q, f.cu_k, seq, f.nseq, f.Tq, f.Tk);
  const int total = sq.nq * G, row0 = slot * F::BM;
  if (slot < 0 || row0 >= total) return;
  const int off = sq.nk - sq.nq;
  const auto position = [&](int row) __attribute__((always_inline)) {
    return uniform((row < total ? row : total - 1) / G) + off;
  };
  const KeyRange range = key_range(position(row0), position(row0 + F::BM - 1), f.window, f.sinks);
  const int wrow = row0 + wave * 32;
  const int w_first = position(wrow), w_last = position(wrow + 31);

  const unsigned char *kb_ = f.k.base + b * f.k.batch + hk * f.k.head + sq.k0 * f.k.token;
  const unsigned char *vb_ = f.v.base + b * f.v.batch + hk * f.v.head + sq.k0 * f.v.token;
  const KeyStage<DT, D, BN, NW> stage(kb_, f.k.token, vb_, f.v.token, range, wave, lane);
  const int tiles = (range.count + BN - 1) / BN;
  if (tiles > 0) stage.tile(0, lds);

  const int row = wrow + n, r = row < total ? row : total - 1;
  const int t = r / G, head = hk * G + (r - t * G), pos = t + off;
  const long out = (static_cast<long>(b) * f.Tq + sq.q0 + t) * f.Hq + head;
  const unsigned char *qrow = f.q.base + b * f.q.batch + (sq.q0 + t) * f.q.token + head * f.q.head;
  const unsigned char *grow = static_cast<const unsigned char *>(p.grad_o) + out * L::ROW;
  v4u32_t qf[S], gf[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    qf[s] = *reinterpret_cast<const v4u32_t *>(qrow + (2 * s + h) * 16);
    gf[s] = *reinterpret_cast<const v4u32_t *>(grow + (2 * s + h) * 16);
    if (f.negate) qf[s] ^= E::BYTES == 2 ? 0x80008000u : 0x80000000u;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    settle(qf[s]);
    settle(gf[s]);
  }
  float2 st;
  float origin = 0.0f;
  bool large;
  {
    const unsigned char *orow = static_cast<const unsigned char *>(p.o) + out * L::ROW;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const v4u32_t x = *reinterpret_cast<const v4u32_t *>(orow + (2 * s + h) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (E::BYTES == 2)
          sum += E::low(x[i]) * E::low(gf[s][i]) + E::high(x[i]) * E::high(gf[s][i]);
        else
          sum += __uint_as_float(x[i]) * __uint_as_float(gf[s][i]);
      }
    }
    sum = add_xor32(sum);
    const float lse = p.lse[out], dlse = p.grad_lse ? p.grad_lse[out] : 0.0f;
    const bool empty = lse == -INFINITY;
    large = fabsf(lse) > LARGE_LSE && fabsf(lse) < INFINITY;
    st = make_float2(empty ? INFINITY : lse * LOG2E, empty ? 0.0f : sum - dlse);
  }
  settle(st.x);
  settle(st.y);
  const int wave_large = __any(large);
  const float scale16 = range_scale<DT, D>(p.range);
  float16_t dq[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) dq[m] = zero16();

  const uint32_t rbase = L::rows_base(n, h), cbase = L::cols_base(lane);
  const auto advance = [&](int it) __attribute__((always_inline)) {
    wait_dma<0>();
    block_sync();
    if (it + 1 < tiles) stage.tile(it + 1, lds + ((it + 1) & 1) * F::TILE);
  };
  // Scores (and dP) of 32 keys, those from u0 on of the range; `whole`: every row sees all of them.
  const auto scores = [&](const unsigned char *kt, int u0, bool whole, float16_t &x) __attribute__((always_inline)) {
    L::template rows_product<1>(kt, rbase, qf, &x);
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int u = u0 + acc_row(i, h);
        x[i] = sees(pos, u < range.sinks ? u : u + range.delta, f.window, f.sinks) ? x[i] : -INFINITY;
      }
    }
  };
  const auto products = [&](const unsigned char *kt, const unsigned char *vt, int u0, bool whole, float16_t &x,
                            float16_t &y) __attribute__((always_inline)) {
    L::template rows_product<1>(kt, rbase, qf, &x);
    L::template rows_product<1>(vt, rbase, gf, &y);
    if (!whole || wave_large) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int u = u0 + acc_row(i, h);
        const bool seen = sees(pos, u < range.sinks ? u : u + range.delta, f.window, f.sinks);
        x[i] = seen ? x[i] - origin : -INFINITY;
        y[i] = seen ? y[i] : 0.0f;
      }
    }
  };
  const int mine = wave_tiles(range, tiles, w_last, BN);
  int it = 0;
  const auto again = [&]() __attribute__((always_inline)) {  // the walk from its start
    for (; it < tiles; ++it) advance(it);
    it = 0;
    block_sync();
    stage.tile(0, lds);
  };
  // Rows of large scores: their largest, and the sum of the weights against it, once more.
  __shared__ int any_large[NW];
  if (lane == 0) any_large[wave] = wave_large;
  block_sync();
  int walk_large = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) walk_large |= any_large[w];
  walk_large = uniform(walk_large);
  if (threadIdx.x == 0) *has_large = walk_large;
  if (walk_large && tiles > 0) {
    float m = -INFINITY, l = 0.0f;
    for (; it < mine; ++it) {
      advance(it);
      const unsigned char *kt = lds + (it & 1) * F::TILE;
      const bool whole = whole_tile(range, it * BN, BN, w_first, w_last, f.window);
#pragma unroll 1
      for (int kb = 0; kb < BN / 32; ++kb) {
        float16_t x;
        scores(kt + 32 * kb * L::ROW, it * BN + 32 * kb, whole, x);
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, x[i]);
        most = fmaxf(m, max_xor32(most));
        const float base = most == -INFINITY ? 0.0f : most;
        l *= __builtin_amdgcn_exp2f((m - base) * f.c);
#pragma unroll
        for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f((x[i] - base) * f.c);
        m = most;
      }
    }
    l += __shfl_xor(l, 32, 64);
    if (large) {
      origin = m;
      st.x = __builtin_amdgcn_logf(l);
    }
    again();
  }
  if constexpr (F::EXACT_TILES > 0) {
    if (tiles > 0 && tiles <= F::EXACT_TILES) {
      float sum = 0.0f;
      for (; it < mine; ++it) {
        advance(it);
        const unsigned char *kt = lds + (it & 1) * F::TILE, *vt = kt + 2 * F::TILE;
        const bool whole = whole_tile(range, it * BN, BN, w_first, w_last, f.window);
#pragma unroll 1
        for (int kb = 0; kb < BN / 32; ++kb) {
          float16_t x, y;
          products(kt + 32 * kb * L::ROW, vt + 32 * kb * L::ROW, it * BN + 32 * kb, whole, x, y);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sum = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], f.c, -st.x)), y[i] - st.y, sum);
          }
        }
      }
      sum += __shfl_xor(sum, 32, 64);
      if (st.x != INFINITY) st.y += p.grad_lse ? sum - p.grad_lse[out] : sum;
      settle(st.y);
      again();
    }
  }
  if (h == 0 && row < total) {
    const long at = ((static_cast<long>(b) * f.Hk + hk) * f.Tq + sq.q0) * G + r;
    p.stat[at] = make_float2(DT == PBGDN_F16 ? st.x - F16_WEIGHTS : st.x, st.y);
    p.origin[at] = origin;
  }
  for (; it < mine; ++it) {
    advance(it);
    const unsigned char *kt = lds + (it & 1) * F::TILE, *vt = kt + 2 * F::TILE;
    const int u0 = it * BN;
    const bool whole = whole_tile(range, u0, BN, w_first, w_last, f.window);
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      float16_t x, y;
      products(kt + 32 * kb * L::ROW, vt + 32 * kb * L::ROW, u0 + 32 * kb, whole, x, y);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float d = y[i] - st.y;
        if constexpr (DT == PBGDN_F16) d *= scale16;
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], f.c, -st.x)) * d;
      }
      const typename L::Operand w = L::operand(x);
      L::template cols_product<1>(kt + 32 * kb * L::ROW, cbase, &w, dq);
    }
  }
  for (; it < tiles; ++it) advance(it);
  if (row < total) store_row<DT, D>(static_cast<unsigned char *>(p.dq) + out * L::ROW, dq, h, p.scale / scale16);
}

// ---------------------------------------------------------------------------
// Launches.
// ---------------------------------------------------------------------------
// Waves (of 32 keys) of a workgroup of dkdv_kernel.
template <int DT, int D>
constexpr int dkdv_waves() { return DT != PBGDN_F32 ? 4 : D == 256 ? 1 : 2; }

static bool sinks_beyond(const WindowParams &f) { return f.sinks > 0 && f.window < f.Tk; }
static int sink_count(const WindowParams &f) { return !sinks_beyond(f) ? 0 : f.sinks < f.Tk ? f.sinks : f.Tk; }

// Parts of a key tile's walk, none shorter than about 16 query tiles. Within a
// window, whose walks are equal: as many as keep the workgroups to twice the CUs,
// for every further part costs its sums' way through memory (8,000 tokens, window
// 1,000, 2 key heads: 359 us with four parts, with five 391; 8,028 tokens, window
// 128, 8 key heads: 293 us with one, with two 343; 4 x 2,048 tokens, window 1,024:
// with one 650 us, with two 690). Without one, where the first keys' walks are
// the longest: at least four workgroups a CU (8,192 tokens: 2,565 us, with half as many 3,145).
static int walk_parts(const WindowParams &f, int B, int bn, int cus) {
  const long tiles = (static_cast<long>(f.Tk) * (f.cu_q ? 1 : B) + bn - 1) / bn * f.Hk;
  const long walk = (f.window < f.Tq ? static_cast<long>(f.window) + bn : f.Tq) * f.group / QR;
  const long want = (f.window < f.Tq ? 2L : 4L) * cus;
  long parts = tiles > 0 ? (f.window < f.Tq ? want : want + tiles - 1) / tiles : 1;
  if (parts > walk / 16) parts = walk / 16;
  return parts < 2 ? 1 : parts > MAX_PARTS ? MAX_PARTS : static_cast<int>(parts);
}

template <int DT, int D>
static int launch_bwd(BwdParams &p, hipStream_t stream) {
  WindowParams &f = p.f;
  const int nb = f.cu_q ? 1 : p.B;
  DeviceShape shape;
  if (!device_shape(shape)) return PBGDN_ERR_LAUNCH;
  if constexpr (DT == PBGDN_F16) {
    hipLaunchKernelGGL(range_zero_kernel, dim3(1), dim3(64), 0, stream, p.range);
    hipLaunchKernelGGL((range_kernel<D>), dim3(shape.cus * 8), dim3(256), 0, stream, p);
  }
  {
    constexpr int DQ_BN = DT == PBGDN_F32 ? (D == 64 ? 64 : 32) : D == 256 ? 32 : 64;
    constexpr int W = DT != PBGDN_F32 && D <= 128 ? 2 : 1;
    using F = Dq<DT, D, DQ_WAVES, DQ_BN>;
    static std::atomic<bool> flags[MAX_DEVICES];
    const auto kernel = dq_kernel<DT, D, DQ_WAVES, DQ_BN, W>;
    if (!smem_configured(reinterpret_cast<const void *>(kernel), F::LDS, flags)) return PBGDN_ERR_LAUNCH;
    static_assert(F::BM == DQ_ROWS);
    const long slots = window_slots(f, DQ_ROWS), blocks = slots * nb * f.Hk;
    if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
    f.slots = static_cast<int>(slots);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(DQ_WAVES * 64), F::LDS, stream, p);
  }

  constexpr int NW = dkdv_waves<DT, D>(), BN = 32 * NW;
  if (f.Tk > 0) {
    {
      using K = Dkdv<DT, D, NW>;
      constexpr int W = DT != PBGDN_F32 && D <= 128 ? 2 : 1;
      static std::atomic<bool> flags[MAX_DEVICES];
      const auto kernel = dkdv_kernel<DT, D, NW, false, W>;
      if (!smem_configured(reinterpret_cast<const void *>(kernel), K::BYTES, flags)) return PBGDN_ERR_LAUNCH;
      const long slots = f.cu_q ? f.Tk / BN + f.nseq + 1 : (f.Tk + BN - 1) / BN;
      const long blocks = slots * p.parts * nb * f.Hk;
      if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
      p.key_slots = static_cast<int>(slots);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(NW * 64), K::BYTES, stream, p);
    }
    if (p.sinks) {
      using K = Dkdv<DT, D, 1>;
      static std::atomic<bool> flags[MAX_DEVICES];
      const auto kernel = dkdv_kernel<DT, D, 1, true, DT != PBGDN_F32 && D <= 128 ? 2 : 1>;
      if (!smem_configured(reinterpret_cast<const void *>(kernel), K::BYTES, flags)) return PBGDN_ERR_LAUNCH;
      const long blocks = static_cast<long>(p.tail_slots) * f.Hk * ((p.sinks + 31) / 32);
      if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64), K::BYTES, stream, p);
    }
    if (p.parts > 1 || p.sinks) {
      const long sinks = p.sinks ? static_cast<long>(long_most(f)) * f.Hk * p.sinks : 0;
      const long want = p.parts > 1 ? (static_cast<long>(p.B) * f.Tk * f.Hk * (D / 4) + 255) / 256 : 0;
      const long blocks = sinks + (want < 65536 ? want : 65536);
      if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
      hipLaunchKernelGGL((join_kernel<DT, D>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p,
                         static_cast<int>(sinks));
    }
  }
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

// The workspace: statistics, the float16 range, the parts.
struct Plan {
  size_t stat, origin, has_large, range, part, tail, bytes;
  int parts, sinks, tail_tokens, tail_slots;
};
static int key_tile(int dtype, int D) {
  return 32 * (dtype != PBGDN_F32 ? 4 : D == 256 ? 1 : 2);
}
static bool plan(Plan &w, const WindowParams &f, int dtype, int B, int D) {
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;  // sizes are asked for without a device too
  w.parts = walk_parts(f, B, key_tile(dtype, D), shape.cus);
  w.sinks = sink_count(f);
  w.tail_tokens = (tail_rows(w.sinks) + f.group - 1) / f.group;
  const long slots = w.sinks ? tail_slot_count(f, w.tail_tokens) : 0;
  if (slots > 0x7fffffffL) return false;
  w.tail_slots = static_cast<int>(slots);
  const auto round = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  w.stat = 0;
  w.origin = round(static_cast<size_t>(B) * f.Tq * f.Hq * sizeof(float2));
  w.has_large = w.origin + round(static_cast<size_t>(B) * f.Tq * f.Hq * sizeof(float));
  w.range = w.has_large + round(static_cast<size_t>(B) * f.Hk * window_slots(f, DQ_ROWS) * sizeof(int));
  w.part = w.range + 256;
  w.tail = w.part + round(w.parts > 1 ? 2 * sizeof(float) * w.parts * B * f.Tk * f.Hk * static_cast<size_t>(D) : 0);
  w.bytes = w.tail + round(2 * sizeof(float) * slots * f.Hk * w.sinks * static_cast<size_t>(D));
  return true;
}

}  // namespace pbgdn

extern "C" size_t pbattn_window_bwd_workspace_size(int B, int Tq, int Tk, int Hq, int Hk, int D, int num_seqs,
                                                   int dtype, int packed, int window, int sinks) {
  using namespace pbgdn;
  if (B < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk != 0 || num_seqs < 0 || sinks < 0 ||
      !attn_dtype(dtype) || (D != 64 && D != 128 && D != 256)) {
    return 0;
  }
  WindowParams f{};
  const int32_t some = 0;
  f.cu_q = packed ? &some : nullptr;
  f.nseq = num_seqs;
  f.Tq = Tq;
  f.Tk = Tk;
  f.Hq = Hq;
  f.Hk = Hk;
  f.group = Hq / Hk;
  f.window = window <= 0 || window > NO_WINDOW ? NO_WINDOW : window;
  f.sinks = sinks < NO_WINDOW ? sinks : NO_WINDOW;
  Plan w;
  return plan(w, f, dtype, B, D) ? w.bytes : 0;
}

extern "C" int pbattn_window_bwd(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                                 const int32_t *cu_q, const int32_t *cu_k, int num_seqs, const void *o,
                                 const float *lse, const void *grad_o, const float *grad_lse, void *dq, void *dk,
                                 void *dv, int B, int Tq, int Tk, int Hq, int Hk, int D, float scale, int window,
                                 int sinks, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace pbgdn;
  BwdParams p{};
  const int status = window_params(p.f, q, k, v, dtype, strides, cu_q, cu_k, num_seqs, B, Tq, Tk, Hq, Hk, D, scale,
                                   window, sinks);
  if (status != PBGDN_OK || p.f.nseq == 0) return status;
  if (!o || !lse || !grad_o || !dq || (Tk > 0 && (!dk || !dv)) || !workspace) return PBGDN_ERR_INVALID_ARGUMENT;
  if (!aligned16(o) || !aligned16(grad_o) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
      !aligned16(workspace)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  Plan w;
  if (!plan(w, p.f, dtype, B, D)) return PBGDN_ERR_UNSUPPORTED;
  if (workspace_bytes < w.bytes) return PBGDN_ERR_INVALID_ARGUMENT;
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  p.o = o;
  p.lse = lse;
  p.grad_o = grad_o;
  p.grad_lse = grad_lse;
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.stat = reinterpret_cast<float2 *>(ws + w.stat);
  p.origin = reinterpret_cast<float *>(ws + w.origin);
  p.has_large = reinterpret_cast<int *>(ws + w.has_large);
  p.range = reinterpret_cast<uint32_t *>(ws + w.range);
  p.part = reinterpret_cast<float *>(ws + w.part);
  p.tail = reinterpret_cast<float *>(ws + w.tail);
  p.scale = scale;
  p.B = B;
  p.D = D;
  p.parts = w.parts;
  p.sinks = w.sinks;
  p.tail_tokens = w.tail_tokens;
  p.tail_slots = w.tail_slots;
  p.heads = p.f.group < QR ? p.f.group : QR;
  p.tokens = QR / p.heads;
  p.splits = (p.f.group + QR - 1) / QR;
  // dkdv_kernel's tiles are staged by 32-bit offsets into a buffer resource, and OUT_OF_RANGE has to be past its end
  const long row = static_cast<long>(D) * attn_bytes(dtype);
  const long q_head = p.heads > 1 ? p.f.q.head : 0;
  const long g_span = (p.tokens - 1L) * Hq * row + p.heads * row;
  if (q_head > OUT_OF_RANGE || (p.tokens - 1) * p.f.q.token + (p.heads - 1) * q_head + row > OUT_OF_RANGE ||
      g_span > OUT_OF_RANGE) {
    return PBGDN_ERR_UNSUPPORTED;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  debug_poison(dq, static_cast<size_t>(B) * Tq * Hq * D * attn_bytes(dtype), st);
  debug_poison(dk, static_cast<size_t>(B) * Tk * Hk * D * attn_bytes(dtype), st);
  debug_poison(dv, static_cast<size_t>(B) * Tk * Hk * D * attn_bytes(dtype), st);
  debug_poison(workspace, w.bytes, st);
#define PBATTN_BWD(T)                                    \
  switch (D) {                                           \
    case 64: return launch_bwd<T, 64>(p, st);            \
    case 128: return launch_bwd<T, 128>(p, st);          \
    default: return launch_bwd<T, 256>(p, st);           \
  }
  switch (dtype) {
    case PBGDN_F32: PBATTN_BWD(PBGDN_F32)
    case PBGDN_BF16: PBATTN_BWD(PBGDN_BF16)
    default: PBATTN_BWD(PBGDN_F16)
  }
#undef PBATTN_BWD
}
