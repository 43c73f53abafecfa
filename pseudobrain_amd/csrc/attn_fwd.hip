// Windowed attention, forward (pbattn_window_fwd).
//
// A workgroup owns BM rows of one (sequence, key head): a row is a (query
// token, head of the key head's group) pair, tokens outermost, so that the
// heads that share keys also share the tile's one pass over them, and a tile
// of BM / G tokens overhangs its window by that little. It walks the union of
// its rows' keys (the sinks, then the window) in tiles of BN, staged by
// direct-to-LDS loads one tile ahead, with the running maximum and sum of an
// online softmax held by the lanes that hold the scores.
#include <atomic>

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

constexpr float LAG = 8.0f;  // weights stay below 2^8

template <int DT, int D, int CB, int NW, int BN>
struct Fwd {
  using L = Tile<DT, D>;
  using E = Elem<DT>;
  static constexpr int BM = 32 * CB * NW, KB = BN / 32, TILE = BN * L::ROW;
  static constexpr int LDS = 4 * TILE;
};

template <int DT, int D, int CB, int NW, int BN, int WAVES>
__global__ __launch_bounds__(NW * 64, WAVES) void window_fwd_kernel(const WindowParams p) {
  using F = Fwd<DT, D, CB, NW, BN>;
  using L = typename F::L;
  using E = typename F::E;
  constexpr int KB = F::KB, S = L::STEPS, MB = L::MB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  PBGDN_POISON_LDS(lds, F::LDS);
  PBGDN_POISON_SYNC();

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = lane & 31, h = lane >> 5, G = p.group;
  const int groups = gridDim.x / p.slots;
  int grp, slot;
  place(blockIdx.x, groups, p.slots, grp, slot);
  const int b = grp / p.Hk, hk = grp % p.Hk;
  int seq = b;
  if (p.cu_q) {
    seq = slot_sequence(p.cu_q, p.nseq, p.Tq, G, F::BM, slot);
    slot -= slot_start(p.cu_q, seq, p.Tq, G, F::BM);
  }
  const Seq sq = sequence<false>(p.cu_q, p.cu_k, seq, p.nseq, p.Tq, p.Tk);
  const long total = static_cast<long>(sq.nq) * G, row0 = static_cast<long>(slot) * F::BM;
  if (slot < 0 || row0 >= total) return;

  // positions of the workgroup's first and last row, and of this wave's
  const int off = sq.nk - sq.nq;
  const auto position = [&](long row) __attribute__((always_inline)) { return static_cast<int>((row < total ? row : total - 1) / G) + off; };
  const KeyRange range = key_range(position(row0), position(row0 + F::BM - 1), p.window, p.sinks);
  const long wrow = row0 + wave * 32 * CB;
  const int w_first = position(wrow), w_last = position(wrow + 32 * CB - 1);

  const unsigned char *kb_ = p.k.base + b * p.k.batch + hk * p.k.head + sq.k0 * p.k.token;
  const unsigned char *vb_ = p.v.base + b * p.v.batch + hk * p.v.head + sq.k0 * p.v.token;
  const KeyStage<DT, D, BN, NW> stage(kb_, p.k.token, vb_, p.v.token, range, wave, lane);
  const int tiles = (range.count + BN - 1) / BN;
  if (tiles > 0) stage.tile(0, lds, wave);

  // this lane's columns: their query rows
  v4u32_t qf[CB][S];
  int pos[CB];
  long out[CB];  // (token, head) index of the row, or -1
  float m[CB], l[CB];
  float16_t o[CB][MB];
#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const long row = wrow + 32 * cb + n;
    const long r = row < total ? row : total - 1;
    const int t = static_cast<int>(r / G), head = hk * G + static_cast<int>(r % G);
    pos[cb] = t + off;
    out[cb] = row < total ? (static_cast<long>(b) * p.Tq + sq.q0 + t) * p.Hq + head : -1;
    const unsigned char *src = p.q.base + b * p.q.batch + (sq.q0 + t) * p.q.token + head * p.q.head;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      qf[cb][s] = *reinterpret_cast<const v4u32_t *>(src + (2 * s + h) * 16);
      if (p.negate) qf[cb][s] ^= E::BYTES == 2 ? 0x80008000u : 0x80000000u;
    }
    m[cb] = -INFINITY;
    l[cb] = 0.0f;
#pragma unroll
    for (int i = 0; i < MB; ++i) o[cb][i] = zero16();
  }

  const uint32_t rbase = L::rows_base(n, h), cbase = L::cols_base(lane);
  const auto advance = [&](int it) __attribute__((always_inline)) {
    wait_dma();
    block_sync();
    if (it + 1 < tiles) stage.tile(it + 1, lds + ((it + 1) & 1) * F::TILE, wave);
  };
  const int mine = wave_tiles(range, tiles, w_last, BN);
  int it = 0;
  for (; it < mine; ++it) {
    advance(it);
    const unsigned char *kt = lds + (it & 1) * F::TILE, *vt = kt + 2 * F::TILE;
    const int u0 = it * BN;
    const bool whole = whole_tile(range, u0, BN, w_first, w_last, p.window);

    float16_t sc[KB][CB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) sc[kb][cb] = zero16();
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const v4u32_t a = L::rows(kt, rbase, 32 * kb, s);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) sc[kb][cb] = E::mma(a, qf[cb][s], sc[kb][cb]);
      }
    }
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int u = u0 + 32 * kb + acc_row(i, h);
          const int j = u < range.sinks ? u : u + range.delta;
#pragma unroll
          for (int cb = 0; cb < CB; ++cb)
            sc[kb][cb][i] = sees(pos[cb], j, p.window, p.sinks) ? sc[kb][cb][i] : -INFINITY;
        }
    }
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float mx = sc[0][cb][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][cb][i]);
      // The reference the weights are taken against moves only when a score
      // passes it by more than LAG powers of two, so most tiles leave the sums
      // as they are.
      mx = max_xor32(mx);
      if (__any((mx - m[cb]) * p.c > LAG)) {
        const float top = fmaxf(m[cb], mx);
        const float alpha = __builtin_amdgcn_exp2f((m[cb] - (top == -INFINITY ? 0.0f : top)) * p.c);
        m[cb] = top;
        l[cb] *= alpha;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[cb][i][e] *= alpha;
      }
      const float base = m[cb] == -INFINITY ? 0.0f : m[cb], at = base * p.c;
      float sum = 0.0f;
      if (__any(fabsf(at) > EXACT_SCORES)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[kb][cb][i] = __builtin_amdgcn_exp2f((sc[kb][cb][i] - base) * p.c);
      } else {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[kb][cb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][cb][i], p.c, -at));
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += sc[kb][cb][i];
      l[cb] += sum;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) L::cols_product(vt, cbase, 32 * kb, L::operand(sc[kb][cb]), o[cb]);
    }
  }
  for (; it < tiles; ++it) advance(it);

#pragma unroll
  for (int cb = 0; cb < CB; ++cb) {
    const float sum = add_xor32(l[cb]);
    const float inv = sum > 0.0f ? 1.0f / sum : sum;  // no key seen: zeros (a NaN stays)
    if (out[cb] < 0) continue;
    if (p.lse && h == 0) p.lse[out[cb]] = sum > 0.0f ? (m[cb] * p.c + __builtin_amdgcn_logf(sum)) * LN2 : sum == 0.0f ? -INFINITY : sum;
    unsigned char *dst = static_cast<unsigned char *>(p.o) + out[cb] * L::ROW;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float4_t x;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = o[cb][i][4 * e + c] * inv;
        const int d = 32 * i + 8 * e + 4 * h;
        if constexpr (E::BYTES == 2) {
          *reinterpret_cast<v2u32_t *>(dst + 2 * d) = v2u32_t{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
        } else {
          *reinterpret_cast<float4_t *>(dst + 4 * d) = x;
        }
      }
  }
}

template <int DT, int D, int CB, int NW, int BN, int WAVES>
static int launch_fwd(WindowParams &p, int B, hipStream_t stream) {
  using F = Fwd<DT, D, CB, NW, BN>;
  static std::atomic<bool> flags[MAX_DEVICES];
  const auto kernel = window_fwd_kernel<DT, D, CB, NW, BN, WAVES>;
  if (!smem_configured(reinterpret_cast<const void *>(kernel), F::LDS, flags)) return PBGDN_ERR_LAUNCH;
  const long slots = window_slots(p, F::BM), blocks = slots * (p.cu_q ? 1 : B) * p.Hk;
  if (blocks > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  p.slots = static_cast<int>(slots);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(NW * 64), F::LDS, stream, p);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

template <int DT>
static int dispatch_fwd(WindowParams &p, int B, int D, hipStream_t stream) {
  constexpr bool wide = DT == PBGDN_F32;
  switch (D) {
    case 64: return launch_fwd<DT, 64, 1, 4, 64, 2>(p, B, stream);
    case 128: return launch_fwd<DT, 128, 1, 4, wide ? 32 : 64, wide ? 1 : 2>(p, B, stream);
    case 256: return launch_fwd<DT, 256, 1, 4, 32, wide ? 1 : 2>(p, B, stream);
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
