// Windowed attention, forward (pbattn_window_fwd).
//
// A workgroup owns BM rows of one (sequence, key head): a row is a (query
// token, head of the key head's group) pair, tokens outermost, so that the
// heads that share keys also share the tile's one pass over them, and a tile
// of BM / G tokens overhangs its window by that little. It walks the union of
// its rows' keys (the sinks, then the window) in tiles of BN, staged by
// direct-to-LDS loads one tile ahead, with the running maximum and sum of an
// online softmax held by the lanes that hold the scores.
//
// Scores are formed as S^T = K Q^T and outputs as O^T = V^T P^T, so that a lane
// of either product holds one row, its maximum and sum stay in the lane pair,
// and the score accumulators are the second product's operand as they stand.
// K and V keep their order in LDS (V's columns come from transposing reads).
//
// Bound by the issue of a SIMD's two waves: 32,768 tokens, 32 heads of 128 on 8,
// window 4,096, take 1.94 to 2.07 ms (1,000 to 1,060 TFLOP/s; a large bf16
// product reaches 1,353 here), of which the matrix unit is busy 54% and the
// softmax's vector instructions take 38%; LDS is busy 27%, without conflicts.
// Shorter key tiles, other waits and wave priorities measured the same. 19,001
// tokens in 24 sequences, 16 heads of 256 on 2: 208 us (711 TFLOP/s), the edges
// of windows and sequences and the last round of workgroups making up the rest.
#include <atomic>

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

// Where a workgroup's BM rows lie: their sequence, its keys, and a run of rows'
// positions.
struct Place {
  int b, hk, off;
  int total, row0;
  Seq sq;
  bool empty;
  const unsigned char *k, *v;
};
template <int BM>
__device__ __forceinline__ Place place_rows(const WindowParams &p) {
  Place w;
  int grp, slot;
  place(blockIdx.x, gridDim.x / p.slots, p.slots, grp, slot);
  w.b = uniform(grp / p.Hk);
  w.hk = grp - w.b * p.Hk;
  int seq = w.b;
  if (p.cu_q) {
    seq = slot_sequence(p.cu_q, p.nseq, p.Tq, p.group, BM, slot);
    slot = uniform(slot - slot_start(p.cu_q, seq, p.Tq, p.group, BM));
  }
  w.sq = sequence<false>(p.cu_q, p.cu_k, seq, p.nseq, p.Tq, p.Tk);
  w.total = w.sq.nq * p.group;
  w.row0 = slot * BM;
  w.empty = slot < 0 || w.row0 >= w.total;
  w.off = w.sq.nk - w.sq.nq;
  w.k = p.k.base + w.b * p.k.batch + w.hk * p.k.head + w.sq.k0 * p.k.token;
  w.v = p.v.base + w.b * p.v.batch + w.hk * p.v.head + w.sq.k0 * p.v.token;
  return w;
}
__device__ __forceinline__ int position(const Place &w, int row, int group) {
  return uniform((row < w.total ? row : w.total - 1) / group) + w.off;
}

// The 32 rows of a wave: lane (n, h) has row n's query units 2 s + h, its softmax
// state and the rows 8 (i / 4) + 4 h + i % 4 of every 32 of its output.
template <int DT, int D>
struct WaveRows {
  using L = Tile<DT, D>;
  using E = typename L::E;
  static constexpr int S = L::STEPS, MB = L::MB;
  v4u32_t q[S];
  int pos;
  long out;  // (token, head) index of the row, or -1
  float m, l;
  float16_t o[MB];
  uint32_t rbase, cbase;
  int h;

  __device__ __forceinline__ void load(const WindowParams &p, const Place &w, int row, int lane) {
    h = lane >> 5;
    row += lane & 31;
    const int r = row < w.total ? row : w.total - 1;
    const int t = r / p.group, head = w.hk * p.group + (r - t * p.group);
    pos = t + w.off;
    out = row < w.total ? (static_cast<long>(w.b) * p.Tq + w.sq.q0 + t) * p.Hq + head : -1;
    const unsigned char *src = p.q.base + w.b * p.q.batch + (w.sq.q0 + t) * p.q.token + head * p.q.head;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      q[s] = *reinterpret_cast<const v4u32_t *>(src + (2 * s + h) * 16);
      if (p.negate) q[s] ^= E::BYTES == 2 ? 0x80008000u : 0x80000000u;
    }
#pragma unroll
    for (int s = 0; s < S; ++s) settle(q[s]);
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < MB; ++i) o[i] = zero16();
    rbase = L::rows_base(lane & 31, h);
    cbase = L::cols_base(lane);
  }

  // Scores of a tile's KB x 32 keys, those from u0 on of the range; `whole`: every
  // row sees all of them.
  template <int KB>
  __device__ __forceinline__ void scores(const WindowParams &p, const KeyRange &range, const unsigned char *tile, int u0,
                                         bool whole, float16_t *sc) const {
    L::template rows_product<KB>(tile, L::ROW < 512 ? rbase : opaque(rbase), q, sc);
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int u = u0 + 32 * kb + acc_row(i, h);
          sc[kb][i] = sees(pos, u < range.sinks ? u : u + range.delta, p.window, p.sinks) ? sc[kb][i] : -INFINITY;
        }
    }
  }

  // Scores to weights, against a reference m that lags behind the maximum.
  template <int KB>
  __device__ __forceinline__ void weights(float c, float16_t *sc) {
    float mx = sc[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
    mx = max_xor32(mx);
    if (__any((mx - m) * c > LAG)) {
      const float top = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f((m - (top == -INFINITY ? 0.0f : top)) * c);
      m = top;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
    }
    const float base = m == -INFINITY ? 0.0f : m, at = base * c;
    if (__any(fabsf(at) > EXACT_SCORES)) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kb][i] = __builtin_amdgcn_exp2f((sc[kb][i] - base) * c);
    } else {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][i], c, -at));
    }
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += sc[kb][i];
    l += sum;
  }

  template <int KB>
  __device__ __forceinline__ void values(const unsigned char *tile, const float16_t *sc) {
    typename L::Operand w[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) w[kb] = L::operand(sc[kb]);
    L::template cols_product<KB>(tile, L::ROW < 512 ? cbase : opaque(cbase), w, o);
  }

  // A value that some rows of a tile see and others do not (a later token's, one
  // the window has passed) enters the products of them all, with weight zero where
  // it is not seen: harmless unless it is infinite or NaN. Rows that end so are
  // worked out again, key by key, from what they see alone. Uniform over the wave.
  __device__ __forceinline__ bool spoiled() const {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x = __builtin_fmaf(o[i][e], 0.0f, x);  // zero, or NaN
    return __any(x != 0.0f);
  }
  __device__ __forceinline__ void redo(const WindowParams &p, const KeyRange &range, const unsigned char *k,
                                                 const unsigned char *v) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < MB; ++i) o[i] = zero16();
    for (int u = 0; u < range.count; ++u) {
      const long j = u < range.sinks ? u : u + range.delta;
      const unsigned char *kr = k + j * p.k.token, *vr = v + j * p.v.token;
      float dot = 0.0f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const v4u32_t x = *reinterpret_cast<const v4u32_t *>(kr + (2 * s + h) * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (E::BYTES == 2)
            dot += E::low(x[i]) * E::low(q[s][i]) + E::high(x[i]) * E::high(q[s][i]);
          else
            dot += __uint_as_float(x[i]) * __uint_as_float(q[s][i]);
        }
      }
      dot = add_xor32(dot);
      if (!sees(pos, static_cast<int>(j), p.window, p.sinks)) continue;
      const float top = fmaxf(m, dot), base = top == -INFINITY ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f((m - base) * p.c), w = __builtin_amdgcn_exp2f((dot - base) * p.c);
      m = top;
      l = l * keep + w;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int d = 32 * i + acc_row(e, h);
          const float x = load_elem(vr, d, DT);
          o[i][e] = o[i][e] * keep + w * x;
        }
    }
  }

  // o and lse of the wave's rows; l summed over the lane halves.
  __device__ __forceinline__ void store(const WindowParams &p) const {
    const float inv = l > 0.0f ? 1.0f / l : l;  // no key seen: zeros (a NaN stays)
    if (out < 0) return;
    if (p.lse && h == 0) p.lse[out] = row_lse(m, l, p.c);
    store_row<DT, D>(static_cast<unsigned char *>(p.o) + out * L::ROW, o, h, inv);
  }
};

template <int DT, int D, int NW, int BN>
struct Fwd {
  static constexpr int BM = 32 * NW, KB = BN / 32, TILE = BN * Tile<DT, D>::ROW, LDS = 4 * TILE;
};

template <int DT, int D, int NW, int BN, int WAVES>
__global__ __launch_bounds__(NW * 64, WAVES) void window_fwd_kernel(const WindowParams p) {
  using F = Fwd<DT, D, NW, BN>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  PBGDN_POISON_LDS(lds, F::LDS);
  PBGDN_POISON_SYNC();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const Place w = place_rows<F::BM>(p);
  if (w.empty) return;
  // the keys of the workgroup's rows, and this wave's first and last position
  const KeyRange range =
      key_range(position(w, w.row0, p.group), position(w, w.row0 + F::BM - 1, p.group), p.window, p.sinks);
  const int row = w.row0 + wave * 32;
  const int w_first = position(w, row, p.group), w_last = position(w, row + 31, p.group);
  const KeyStage<DT, D, BN, NW, (Tile<DT, D>::ROW < 512)> stage(w.k, p.k.token, w.v, p.v.token, range, wave, lane);
  const int tiles = (range.count + BN - 1) / BN;
  if (tiles > 0) stage.tile(0, lds);
  WaveRows<DT, D> r;
  r.load(p, w, row, lane);

  const auto advance = [&](int it) __attribute__((always_inline)) {
    wait_dma<0>();
    block_sync();
    if (it + 1 < tiles) stage.tile(it + 1, lds + ((it + 1) & 1) * F::TILE);
  };
  const int mine = wave_tiles(range, tiles, w_last, BN);
  int it = 0;
  for (; it < mine; ++it) {
    advance(it);
    const unsigned char *kt = lds + (it & 1) * F::TILE, *vt = kt + 2 * F::TILE;
    float16_t sc[F::KB];
    r.template scores<F::KB>(p, range, kt, it * BN, whole_tile(range, it * BN, BN, w_first, w_last, p.window), sc);
    r.template weights<F::KB>(p.c, sc);
    r.template values<F::KB>(vt, sc);
  }
  for (; it < tiles; ++it) advance(it);
  r.l = add_xor32(r.l);
  if (r.spoiled()) r.redo(p, range, w.k, w.v);
  r.store(p);
}

// The same for calls with too few rows to fill the GPU: the waves of a workgroup
// share its 32 rows and take their key tiles in turn, each through tiles of its
// own with no barrier, and join their sums at the end. Bound by the latency of a
// row tile's walk: 777 tokens, 32 heads of 128 on 8: 18 us; 2,048 tokens, 4 heads
// of 64, float32: 39 us, the last rows' 64 key tiles on eight waves.
template <int DT, int D, int NW>
struct Split {
  using L = Tile<DT, D>;
  static constexpr int BN = 32, TILE = BN * L::ROW;
  static constexpr int SUMS = 64 * (L::MB * 16 + 2) * 4;  // a wave's sums
  static constexpr int LDS = NW * 2 * TILE > NW / 2 * SUMS ? NW * 2 * TILE : NW / 2 * SUMS;
};

template <int DT, int D, int NW, int WAVES>
__global__ __launch_bounds__(NW * 64, WAVES) void window_split_kernel(const WindowParams p) {
  using F = Split<DT, D, NW>;
  using L = typename F::L;
  constexpr int BN = F::BN, MB = L::MB;
  using Stage = KeyStage<DT, D, BN, 1, (L::ROW < 512)>;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  PBGDN_POISON_LDS(lds, F::LDS);
  PBGDN_POISON_SYNC();
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const Place w = place_rows<32>(p);
  if (w.empty) return;
  const int w_first = position(w, w.row0, p.group), w_last = position(w, w.row0 + 31, p.group);
  const KeyRange range = key_range(w_first, w_last, p.window, p.sinks);
  const Stage stage(w.k, p.k.token, w.v, p.v.token, range, 0, lane);
  const int tiles = (range.count + BN - 1) / BN;
  unsigned char *const kt = lds + wave * 2 * F::TILE, *const vt = kt + F::TILE;
  WaveRows<DT, D> r;
  r.load(p, w, w.row0, lane);
  if (wave < tiles) {
    stage.keys(wave, kt);
    stage.values(wave, vt);
  }
  // K of the next tile is fetched while this one's weights and values are worked
  // on, V while the next one's scores are.
  for (int it = wave; it < tiles; it += NW) {
    const bool more = it + NW < tiles;
    float16_t sc[1];
    wait_dma<Stage::LOADS>();
    r.template scores<1>(p, range, kt, it * BN, whole_tile(range, it * BN, BN, w_first, w_last, p.window), sc);
    wait_lds();
    if (more) stage.keys(it + NW, kt);
    r.template weights<1>(p.c, sc);
    if (more)
      wait_dma<Stage::LOADS>();
    else
      wait_dma<0>();
    r.template values<1>(vt, sc);
    wait_lds();
    if (more) stage.values(it + NW, vt);
  }
  r.l = add_xor32(r.l);

  // the waves' sums into wave 0, the upper half into the lower
#pragma unroll
  for (int half = NW / 2; half > 0; half >>= 1) {
    __syncthreads();
    float *const at = reinterpret_cast<float *>(lds + (wave % half) * F::SUMS);
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float4_t *>(at + ((4 * i + e) * 64 + lane) * 4) =
              float4_t{r.o[i][4 * e], r.o[i][4 * e + 1], r.o[i][4 * e + 2], r.o[i][4 * e + 3]};
      at[MB * 1024 + lane] = r.m;
      at[MB * 1024 + 64 + lane] = r.l;
    }
    __syncthreads();
    if (wave < half) {
      const float m2 = at[MB * 1024 + lane], top = fmaxf(r.m, m2), base = top == -INFINITY ? 0.0f : top;
      const float f1 = __builtin_amdgcn_exp2f((r.m - base) * p.c), f2 = __builtin_amdgcn_exp2f((m2 - base) * p.c);
      r.m = top;
      r.l = r.l * f1 + at[MB * 1024 + 64 + lane] * f2;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4_t x = *reinterpret_cast<const float4_t *>(at + ((4 * i + e) * 64 + lane) * 4);
#pragma unroll
          for (int c = 0; c < 4; ++c) r.o[i][4 * e + c] = r.o[i][4 * e + c] * f1 + x[c] * f2;
        }
    }
  }
  if (wave != 0) return;
  if (r.spoiled()) r.redo(p, range, w.k, w.v);
  r.store(p);
}

template <typename Kernel>
static int launch_rows(WindowParams &p, int B, Kernel kernel, int bm, int nw, int lds, std::atomic<bool> *flags,
                       hipStream_t stream) {
  if (!smem_configured(reinterpret_cast<const void *>(kernel), lds, flags)) return PBGDN_ERR_LAUNCH;
  const long slots = window_slots(p, bm), blocks = slots * (p.cu_q ? 1 : B) * p.Hk;
  if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  p.slots = static_cast<int>(slots);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(nw * 64), lds, stream, p);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

template <int DT, int D, int NW, int WAVES>
static int launch_split(WindowParams &p, int B, hipStream_t stream) {
  static std::atomic<bool> flags[MAX_DEVICES];
  return launch_rows(p, B, window_split_kernel<DT, D, NW, WAVES>, 32, NW, Split<DT, D, NW>::LDS, flags, stream);
}

// Which of the two, by how far the rows fill the GPU. n workgroups of 32 rows,
// whose waves share the keys, up to five a CU (three with rows of 512 bytes and
// more); of more rows, 128 to a workgroup.
// Waves of a workgroup: two where a row's walk is no longer than five tiles or
// workgroups of four would number more than a CU's LDS and registers hold (or two
// a CU), else four, or eight for narrow heads where the workgroups number no more
// than the CUs. Measured,
// us, window 1,024, one sequence (128 rows to a workgroup / 2 / 4 / 8 waves to 32):
//   32 heads of 128 on 8, bf16      64 tokens   7.8 /  5.7 /  6.8 /  7.9
//                                  500 tokens  16.5 / 12.3 / 10.9 / 17.2
//                                  777 tokens  21.6 / 18.5 / 20.5 / 32.5
//                                1,300 tokens  29.8 / 28.0 / 34.4 / 53.2
//                                1,700 tokens  32.8 / 39.6 / 46.6 / 67.9
//   16 heads of 256 on 2, bf16     500 tokens  27.7 / 18.0 / 14.3
//                                1,300 tokens  48.5 / 36.5 / 44.6
//                                1,700 tokens  49.4 / 52.8 / 61.7
//   4 heads of 64, float32       1,300 tokens  90.1 / 44.0 / 27.2 / 25.5
template <int DT, int D, int BN, int WAVES>
static int launch_fwd(WindowParams &p, int B, hipStream_t stream) {
  static std::atomic<bool> flags[MAX_DEVICES];
  using F = Fwd<DT, D, 4, BN>;
  constexpr int ROW = Tile<DT, D>::ROW;
  DeviceShape shape;
  if (!device_shape(shape)) return PBGDN_ERR_LAUNCH;
  const long n = window_slots(p, 32) * (p.cu_q ? 1 : B) * p.Hk;
  const long keys = p.window < p.Tk ? static_cast<long>(p.window) + p.sinks : p.Tk, walk = (keys + 31) / 32;
  if (n <= (ROW <= 256 ? 5L : 3L) * shape.cus) {
    if constexpr (D == 64) {
      if (n <= shape.cus && walk > 20) return launch_split<DT, D, 8, WAVES>(p, B, stream);
    }
    if constexpr (ROW <= 512) {
      constexpr int RESIDENT = ROW <= 128 ? 4 : 2;
      if (n <= RESIDENT * shape.cus && walk > 5) return launch_split<DT, D, 4, WAVES>(p, B, stream);
    }
    return launch_split<DT, D, 2, WAVES>(p, B, stream);
  }
  return launch_rows(p, B, window_fwd_kernel<DT, D, 4, BN, WAVES>, F::BM, 4, F::LDS, flags, stream);
}

template <int DT>
static int dispatch_fwd(WindowParams &p, int B, int D, hipStream_t stream) {
  constexpr bool wide = DT == PBGDN_F32;
  switch (D) {
    case 64: return launch_fwd<DT, 64, 64, 2>(p, B, stream);
    case 128: return launch_fwd<DT, 128, wide ? 32 : 64, wide ? 1 : 2>(p, B, stream);
    case 256: return launch_fwd<DT, 256, 32, wide ? 1 : 2>(p, B, stream);
    default: return PBGDN_ERR_UNSUPPORTED;
  }
}

int window_params(WindowParams &p, const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                  const int32_t *cu_q, const int32_t *cu_k, int num_seqs, int B, int Tq, int Tk, int Hq, int Hk, int D,
                  float scale, int window, int sinks) {
  if (B < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hk <= 0 || Hq % Hk != 0 || D <= 0 || num_seqs < 0 || sinks < 0 ||
      !attn_dtype(dtype) || !strides || !(scale - scale == 0.0f)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (cu_k && !cu_q) return PBGDN_ERR_INVALID_ARGUMENT;
  if (cu_q ? B != 1 || (!cu_k && Tq != Tk) : num_seqs != B) return PBGDN_ERR_INVALID_ARGUMENT;
  p = WindowParams{};
  if (B == 0 || Tq == 0 || num_seqs == 0) return PBGDN_OK;
  if (!q || (Tk > 0 && (!k || !v))) return PBGDN_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return PBGDN_ERR_INVALID_ARGUMENT;
  if (D != 64 && D != 128 && D != 256) return PBGDN_ERR_UNSUPPORTED;
  if (Tq >= NO_WINDOW || Tk >= NO_WINDOW) return PBGDN_ERR_UNSUPPORTED;
  if (static_cast<long>(Tq) * (Hq / Hk) > 0x7fffffffL - 1024) return PBGDN_ERR_UNSUPPORTED;  // rows of a key head
  const int bytes = attn_bytes(dtype);
  View *views[3] = {&p.q, &p.k, &p.v};
  const void *bases[3] = {q, k, v};
  for (int i = 0; i < 3; ++i) {
    const int64_t *s = strides + 3 * i;
    for (int a = 0; a < 3; ++a)
      if (s[a] < 0 || s[a] * bytes % 16 != 0) return PBGDN_ERR_INVALID_ARGUMENT;
    if (s[1] * bytes >= (1 << 24)) return PBGDN_ERR_UNSUPPORTED;
    *views[i] = View{static_cast<const unsigned char *>(bases[i]), s[0] * bytes, s[1] * bytes, s[2] * bytes};
  }
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.nseq = num_seqs;
  p.Tq = Tq;
  p.Tk = Tk;
  p.Hq = Hq;
  p.Hk = Hk;
  p.group = Hq / Hk;
  p.window = window <= 0 || window > NO_WINDOW ? NO_WINDOW : window;
  p.sinks = sinks < NO_WINDOW ? sinks : NO_WINDOW;
  const float c = __builtin_fabsf(scale) * LOG2E;
  p.c = c > 1.17549435e-38f ? c : 1.17549435e-38f;
  p.negate = scale < 0.0f;
  return PBGDN_OK;
}

}  // namespace pbgdn

extern "C" int pbattn_abi_version(void) { return PBATTN_ABI_VERSION; }

extern "C" int pbattn_window_fwd(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                                 const int32_t *cu_q, const int32_t *cu_k, int num_seqs, void *o, float *lse, int B,
                                 int Tq, int Tk, int Hq, int Hk, int D, float scale, int window, int sinks,
                                 void *stream) {
  using namespace pbgdn;
  WindowParams p;
  const int status = window_params(p, q, k, v, dtype, strides, cu_q, cu_k, num_seqs, B, Tq, Tk, Hq, Hk, D, scale,
                                   window, sinks);
  if (status != PBGDN_OK || p.nseq == 0) return status;
  if (!o || !aligned16(o)) return PBGDN_ERR_INVALID_ARGUMENT;
  p.o = o;
  p.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t rows = static_cast<size_t>(B) * Tq * Hq;
  debug_poison(o, rows * D * attn_bytes(dtype), st);
  if (lse) debug_poison(lse, rows * sizeof(float), st);
  switch (dtype) {
    case PBGDN_F32: return dispatch_fwd<PBGDN_F32>(p, B, D, st);
    case PBGDN_BF16: return dispatch_fwd<PBGDN_BF16>(p, B, D, st);
    default: return dispatch_fwd<PBGDN_F16>(p, B, D, st);
  }
}
