// Norms of queries and keys for each head and the rotation by their positions, in one
// pass (pbattn_qk_norm_rope), and its gradients (pbattn_qk_norm_rope_bwd).
//
//   y = x r w,  r = (mean x^2 + eps)^(-1/2)            over a head's D values
//   (a, b) -> (a cos - b sin, b cos + a sin)           over pairs of y's first R values
//   h = the same turned back of the gradient,  dw = sum over rows of h x r,
//   u = h w,  dx = r (u - x r^2 mean(u x))
//
// Bound by bytes: x is read once and y written once (the backward reads x and the
// gradient, writes dx), so the kernels are built around 16-byte accesses. A lane owns two
// units of 16 bytes of a row, such that both values of every pair are its own: units u
// and u + half of the rotated ones (or neighbours, where neighbouring values are paired
// or nothing is rotated). A row takes D / 16 lanes (float32: D / 8), the sums over it
// DPP moves. A wave takes a token's heads one group of rows after the other and keeps
// the token's angles and the weights in registers.
//
// 19,001 tokens of 32 heads of 128 on 8, bf16: forward 76 us, 5.2 TB/s; 8,192 tokens:
// forward 29 us, backward 50 (5.1 TB/s), its sums joined in 4; what a large copy reaches
// is 5.1. 64 tokens: 4.2 us, the launch.
#include <initializer_list>
#include <type_traits>

#include "attn.hpp"
#include "attn_tile.hpp"
#include "device.hpp"

namespace pbgdn {

constexpr int ROPE_WAVES = 4;
constexpr int ROPE_MAX_D = 256;
constexpr long ROPE_MOST = 1 << 20;  // workgroups of a launch; waves take piece after piece where there are more

struct RopeParams {
  const unsigned char *x[2];       // q, k
  long batch[2], token[2], head[2];  // their strides, bytes
  const unsigned char *g[2];       // dense gradients of the outputs (backward)
  unsigned char *out[2];           // dense: the outputs, or the gradients of q and k
  const void *w[2];
  const float *cos, *sin;
  const void *pos;
  long pos_batch, pos_token;       // elements
  float *part;                     // [workgroups][D] sums for the weights' gradients
  long tokens;                     // of all batch rows
  int T, H[2], D, R, rows;         // rows: of the angles' tables
  int split[2];                    // waves a token's heads of q, or k, are divided over
  int blocks_q;                    // workgroups of q; the others are k's
  int wdt, pos64, interleaved;
  float eps, offset;
};

// The token's row of the angles' tables, -1 where there is none.
__device__ __forceinline__ long angle_row(const RopeParams &p, int b, int t) {
  const long i = b * p.pos_batch + t * p.pos_token;
  const long at = p.pos64 ? static_cast<const int64_t *>(p.pos)[i] : static_cast<const int32_t *>(p.pos)[i];
  return at >= 0 && at < p.rows ? at : -1;
}

// Unit `u` of E weights as float32.
template <int E>
__device__ __forceinline__ void load_weights(const void *w, int wdt, int u, float offset, float *out) {
  if (wdt == PBGDN_F32) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4_t x = *reinterpret_cast<const float4_t *>(static_cast<const float *>(w) + u * E + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) out[e + i] = x[i] + offset;
    }
  } else {
    uint32_t x[E / 2];
    const uint32_t *src = reinterpret_cast<const uint32_t *>(static_cast<const u16 *>(w) + u * E);
    if constexpr (E == 8) {
      const v4u32_t y = *reinterpret_cast<const v4u32_t *>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = y[i];
    } else {
      const v2u32_t y = *reinterpret_cast<const v2u32_t *>(src);
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = y[i];
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const bool bf = wdt == PBGDN_BF16;
      out[2 * i] = (bf ? Elem<PBGDN_BF16>::low(x[i]) : Elem<PBGDN_F16>::low(x[i])) + offset;
      out[2 * i + 1] = (bf ? Elem<PBGDN_BF16>::high(x[i]) : Elem<PBGDN_F16>::high(x[i])) + offset;
    }
  }
}

template <int DT>
struct Unit {  // 16 bytes of a row
  static constexpr int E = DT == PBGDN_F32 ? 4 : 8;
  __device__ static __forceinline__ void unpack(v4u32_t w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == PBGDN_F32) {
        x[i] = __uint_as_float(w[i]);
      } else {
        x[2 * i] = Elem<DT>::low(w[i]);
        x[2 * i + 1] = Elem<DT>::high(w[i]);
      }
    }
  }
  __device__ static __forceinline__ v4u32_t pack(const float *x) {
    v4u32_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == PBGDN_F32)
        w[i] = __float_as_uint(x[i]);
      else
        w[i] = Elem<DT>::pack(x[2 * i], x[2 * i + 1]);
    }
    return w;
  }
};

// Sum over the G lanes of a row.
template <int G>
__device__ __forceinline__ float row_sum(float x) {
  x = group_sum(x, G < 16 ? G : 16);
  if constexpr (G == 32) x = add_xor16(x);
  return x;
}

// What a row is multiplied by before its squares are summed, given their mean (and eps):
// a power of two that brings squares past float32's range back into it; nearly always 1. With
// x and eps^(1/2) both multiplied by it y and the weights' gradients stay as they are, dx has to
// be multiplied by it once more. (No time at any size; the float16 backward 56.3 -> 54.6 us at
// 8,192 tokens, as it no longer spills.)
__device__ __forceinline__ bool squares_lost(float mean) { return !(mean > 0x1p-90f) | (mean > 0x1p100f); }
__device__ __forceinline__ float row_scale(float mean) { return mean > 0x1p100f ? 0x1p-70f : mean <= 0x1p-90f ? 0x1p100f : 1.0f; }

// Pairs of a lane's 2 E values turned by +-angle (INVERSE: back); where the lane's
// values are not rotated they stay as they are, infinities too.
template <int E, bool PAIRS, bool INVERSE>
__device__ __forceinline__ void turn(float *v, const float *c, const float *s, bool turns) {
#pragma unroll
  for (int i = 0; i < E; ++i) {
    float &a = v[PAIRS ? 2 * i : i], &b = v[PAIRS ? 2 * i + 1 : E + i];
    const float si = INVERSE ? -s[i] : s[i], x = a * c[i] - b * si, y = b * c[i] + a * si;
    a = turns ? x : a;
    b = turns ? y : b;
  }
}

// The workgroup's sums over its waves to its place.
__device__ __forceinline__ void store_sums(const RopeParams &p, const float (&sums)[ROPE_WAVES][ROPE_MAX_D]) {
  __syncthreads();
  for (int i = threadIdx.x; i < p.D; i += ROPE_WAVES * 64) {
    float y = 0.0f;
#pragma unroll
    for (int wave = 0; wave < ROPE_WAVES; ++wave) y += sums[wave][i];
    p.part[static_cast<long>(blockIdx.x) * p.D + i] = y;
  }
}

// Workgroups are q's or k's, so that one set of weights, and in the backward of their
// sums, is in registers: six waves a SIMD in the forward, four in the backward.
template <int DT, int G, bool PAIRS, bool BWD>
__global__ __launch_bounds__(ROPE_WAVES * 64, 4) void rope_kernel(const RopeParams p) {
  using U = Unit<DT>;
  constexpr int E = U::E, ROWS = 64 / G;  // rows of a wave at a time
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), j = lane % G, group = lane / G;
  const int lanes = p.D / (2 * E), half = p.R / (2 * E);  // lanes of a row; those that rotate
  const bool mine = j < lanes, turns = j < half;
  const int u0 = PAIRS ? 2 * j : turns ? j : 2 * j, u1 = PAIRS || !turns ? u0 + 1 : j + half;
  const bool key = static_cast<int>(blockIdx.x) >= p.blocks_q;
  const int block = key ? blockIdx.x - p.blocks_q : blockIdx.x, blocks = key ? gridDim.x - p.blocks_q : p.blocks_q;
  const int heads = key ? p.H[1] : p.H[0], groups = (heads + ROWS - 1) / ROWS, split = key ? p.split[1] : p.split[0];
  const unsigned char *const x_base = key ? p.x[1] : p.x[0], *const g_base = key ? p.g[1] : p.g[0];
  unsigned char *const out_base = key ? p.out[1] : p.out[0];
  const long batch_step = key ? p.batch[1] : p.batch[0], token_step = key ? p.token[1] : p.token[0],
             head_step = key ? p.head[1] : p.head[0];
  float w[2 * E];
  load_weights<E>(key ? p.w[1] : p.w[0], p.wdt, mine ? u0 : 0, p.offset, w);
  load_weights<E>(key ? p.w[1] : p.w[0], p.wdt, mine ? u1 : 0, p.offset, w + E);
  float dw[BWD ? 2 * E : 1];
#pragma unroll
  for (int i = 0; i < (BWD ? 2 * E : 1); ++i) dw[i] = 0.0f;

  for (long item = block * static_cast<long>(ROPE_WAVES) + wave; item < p.tokens * split;
       item += static_cast<long>(blocks) * ROPE_WAVES) {
    const long tok = item / split;
    const int first = static_cast<int>(item - tok * split);
    const int b = static_cast<int>(tok / p.T), t = static_cast<int>(tok - static_cast<long>(b) * p.T);
    const long row = angle_row(p, b, t);
    const bool known = row >= 0;
    float c[E], s[E];
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      float4_t x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
      if (turns & known) {
        x = *reinterpret_cast<const float4_t *>(p.cos + row * (p.R / 2) + j * E + e);
        y = *reinterpret_cast<const float4_t *>(p.sin + row * (p.R / 2) + j * E + e);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[e + i] = x[i];
        s[e + i] = y[i];
      }
    }
    for (int i = first; i < groups; i += split) {
      const int h = i * ROWS + group;
      const bool here = mine & (h < heads);
      const long at = (tok * heads + h) * p.D * (16 / E);  // of a dense row, bytes
      v4u32_t a = {0, 0, 0, 0}, d = {0, 0, 0, 0}, ga = {0, 0, 0, 0}, gd = {0, 0, 0, 0};
      if (here & known) {
        const unsigned char *src = x_base + b * batch_step + t * token_step + h * head_step;
        a = *reinterpret_cast<const v4u32_t *>(src + u0 * 16);
        d = *reinterpret_cast<const v4u32_t *>(src + u1 * 16);
        if constexpr (BWD) {
          ga = *reinterpret_cast<const v4u32_t *>(g_base + at + u0 * 16);
          gd = *reinterpret_cast<const v4u32_t *>(g_base + at + u1 * 16);
        }
      }
      float v[2 * E];
      U::unpack(a, v);
      U::unpack(d, v + E);
      const auto mean_of_squares = [&](float eps) __attribute__((always_inline)) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
        return row_sum<G>(ss) / p.D + eps;
      };
      float mean = mean_of_squares(p.eps), scale = 1.0f;
      if (__any((here & known) && squares_lost(mean))) {
        scale = row_scale(mean);
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) v[e] *= scale;
        mean = mean_of_squares(p.eps * scale * scale);
      }
      const float r = 1.0f / sqrtf(mean);
      if constexpr (!BWD) {
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) v[e] = v[e] * r * w[e];
        turn<E, PAIRS, false>(v, c, s, turns);
      } else {
        float g[2 * E];
        U::unpack(ga, g);
        U::unpack(gd, g + E);
        turn<E, PAIRS, true>(g, c, s, turns);
        float ux = 0.0f;
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) ux = __builtin_fmaf(g[e] * w[e], v[e], ux);
        const float f = r * r * (row_sum<G>(ux) / p.D);
        if (here & known) {
#pragma unroll
          for (int e = 0; e < 2 * E; ++e) dw[e] += g[e] * (v[e] * r);
        }
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) v[e] = r * (g[e] * w[e] - v[e] * f) * scale;
      }
      if (here) {
        unsigned char *dst = out_base + at;
        const v4u32_t zero = {0, 0, 0, 0};  // a row without a position
        *reinterpret_cast<v4u32_t *>(dst + u0 * 16) = known ? U::pack(v) : zero;
        *reinterpret_cast<v4u32_t *>(dst + u1 * 16) = known ? U::pack(v + E) : zero;
      }
    }
  }
  if constexpr (BWD) {
    __shared__ float sums[ROPE_WAVES][ROPE_MAX_D];
    PBGDN_POISON_LDS(sums, sizeof(sums));
    PBGDN_POISON_SYNC();
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      float y = dw[e];
#pragma unroll
      for (int off = G; off < 64; off *= 2) y += __shfl_xor(y, off, 64);
      if (mine & (group == 0)) sums[wave][(e < E ? u0 : u1) * E + e % E] = y;
    }
    store_sums(p, sums);
  }
}

// Any width, alignment and stride: a wave a row, element lane + 64 e of it a lane; the
// other value of a pair is read (and normed) again by the lane that needs it.
template <int DT, bool BWD>
__global__ __launch_bounds__(ROPE_WAVES * 64) void rope_any_kernel(const RopeParams p) {
  constexpr int N = ROPE_MAX_D / 64;
  constexpr int BYTES = DT == PBGDN_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int key = static_cast<int>(blockIdx.x) >= p.blocks_q, heads = p.H[key];
  const int block = key ? blockIdx.x - p.blocks_q : blockIdx.x, blocks = key ? gridDim.x - p.blocks_q : p.blocks_q;
  float dw[N];
#pragma unroll
  for (int e = 0; e < N; ++e) dw[e] = 0.0f;
  for (long item = block * static_cast<long>(ROPE_WAVES) + wave; item < p.tokens * heads;
       item += static_cast<long>(blocks) * ROPE_WAVES) {
    const long tok = item / heads;
    const int h = static_cast<int>(item - tok * heads);
    const int b = static_cast<int>(tok / p.T), t = static_cast<int>(tok - static_cast<long>(b) * p.T);
    const long row = angle_row(p, b, t), at = item * p.D;
    if (row < 0) {
      for (int i = lane; i < p.D; i += 64) store_elem(p.out[key], at + i, DT, 0.0f);
      continue;
    }
    const unsigned char *x = p.x[key] + b * p.batch[key] + t * p.token[key] + h * p.head[key];
    const unsigned char *g = BWD ? p.g[key] + at * BYTES : x;
    const auto weight = [&](int i) { return load_elem(p.w[key], i, p.wdt) + p.offset; };
    float v[N], y[N], mean, ux, scale = 1.0f;
    const auto row_values = [&]() __attribute__((always_inline)) {
      float ss = 0.0f;
      ux = 0.0f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = lane + 64 * e;
        v[e] = y[e] = 0.0f;
        if (i >= p.D) continue;
        v[e] = load_elem(x, i, DT) * scale;
        ss = __builtin_fmaf(v[e], v[e], ss);
        // the forward turns x w, the backward the gradient back; r enters afterwards
        const auto value = [&](int k) { return BWD ? load_elem(g, k, DT) : load_elem(x, k, DT) * scale * weight(k); };
        y[e] = value(i);
        if (i < p.R) {
          const int half = p.R / 2;
          const bool second = p.interleaved ? i & 1 : i >= half;
          const int other = p.interleaved ? i ^ 1 : second ? i - half : i + half;
          const long k = row * half + (p.interleaved ? i / 2 : second ? i - half : i);
          const float c = p.cos[k], s = p.sin[k];
          y[e] = y[e] * c + value(other) * (second != BWD ? s : -s);
        }
        if constexpr (BWD) ux = __builtin_fmaf(y[e] * weight(i), v[e], ux);
      }
      mean = wave_sum(ss) / p.D + p.eps * scale * scale;
    };
    row_values();
    if (squares_lost(mean)) {  // (the whole wave's row)
      scale = row_scale(mean);
      row_values();
    }
    const float r = 1.0f / sqrtf(mean), f = BWD ? r * r * (wave_sum(ux) / p.D) : 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = lane + 64 * e;
      if (i >= p.D) continue;
      if constexpr (BWD) {
        dw[e] += y[e] * (v[e] * r);
        store_elem(p.out[key], at + i, DT, r * (y[e] * weight(i) - v[e] * f) * scale);
      } else {
        store_elem(p.out[key], at + i, DT, y[e] * r);
      }
    }
  }
  if constexpr (BWD) {
    __shared__ float sums[ROPE_WAVES][ROPE_MAX_D];
    PBGDN_POISON_LDS(sums, sizeof(sums));
    PBGDN_POISON_SYNC();
#pragma unroll
    for (int e = 0; e < N; ++e) sums[wave][lane + 64 * e] = dw[e];
    store_sums(p, sums);
  }
}

// The weights' gradients from the workgroups' sums, in a fixed order: 16 columns a
// workgroup, every 64th sum a thread.
constexpr int JOIN_COLS = 16, JOIN_ROWS = 64;
__global__ __launch_bounds__(JOIN_COLS * JOIN_ROWS) void rope_join_kernel(const float *part, int blocks_q, int blocks, int D,
                                                                          void *dq, void *dk, int wdt) {
  __shared__ float sums[JOIN_ROWS][JOIN_COLS];
  PBGDN_POISON_LDS(sums, sizeof(sums));
  PBGDN_POISON_SYNC();
  const int tiles = (D + JOIN_COLS - 1) / JOIN_COLS;
  const bool key = static_cast<int>(blockIdx.x) >= tiles;
  const int c = threadIdx.x % JOIN_COLS, r = threadIdx.x / JOIN_COLS;
  const int col = (key ? blockIdx.x - tiles : blockIdx.x) * JOIN_COLS + c, end = key ? blocks : blocks_q;
  float x = 0.0f;
  if (col < D) {
#pragma unroll 8
    for (int i = (key ? blocks_q : 0) + r; i < end; i += JOIN_ROWS) x += part[static_cast<long>(i) * D + col];
  }
  sums[r][c] = x;
#pragma unroll
  for (int n = JOIN_ROWS / 2; n > 0; n /= 2) {
    __syncthreads();
    if (r < n) sums[r][c] += sums[r + n][c];
  }
  if (r == 0 && col < D) store_elem(key ? dk : dq, col, wdt, sums[0][c]);
}

// Most workgroups of the backward: as many as the GPU holds at once, four a CU.
static long rope_bwd_blocks() {
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  return 4L * shape.cus;
}

static int rope_params(RopeParams &p, const void *q, const void *k, int dtype, const int64_t *strides, const void *qw,
                       const void *kw, int wdt, float offset, const float *cos, const float *sin, int rows,
                       const void *positions, int pos64, const int64_t *pos_strides, int B, int T, int Hq, int Hk, int D,
                       int R, float eps, int interleaved) {
  if (B < 0 || T < 0 || Hq <= 0 || Hk <= 0 || D <= 0 || R < 0 || R % 2 != 0 || R > D || rows < 0 || !attn_dtype(dtype) ||
      !attn_dtype(wdt) || !strides || !pos_strides || !(eps >= 0.0f) || !(eps - eps == 0.0f) || !(offset - offset == 0.0f) ||
      (pos64 & ~1) || (interleaved & ~1)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (D > ROPE_MAX_D) return PBGDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return PBGDN_OK;
  const long size = attn_bytes(dtype), heads = static_cast<long>(Hq) + Hk;
  if (!q || !k || !qw || !kw || !positions || (R > 0 && rows > 0 && (!cos || !sin))) return PBGDN_ERR_INVALID_ARGUMENT;
  const auto off = [](const void *x, long bytes) { return reinterpret_cast<uintptr_t>(x) % bytes != 0; };
  if (off(q, size) || off(k, size) || off(qw, attn_bytes(wdt)) || off(kw, attn_bytes(wdt)) || off(cos, 4) || off(sin, 4) ||
      off(positions, pos64 ? 8 : 4)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  for (int a = 0; a < 6; ++a)
    if (strides[a] < 0) return PBGDN_ERR_INVALID_ARGUMENT;
  if (pos_strides[0] < 0 || pos_strides[1] < 0) return PBGDN_ERR_INVALID_ARGUMENT;
  if (heads > 0x7fffff00L) return PBGDN_ERR_UNSUPPORTED;
  const void *x[2] = {q, k}, *w[2] = {qw, kw};
  for (int a = 0; a < 2; ++a) {
    p.x[a] = static_cast<const unsigned char *>(x[a]);
    p.batch[a] = strides[3 * a] * size;
    p.token[a] = strides[3 * a + 1] * size;
    p.head[a] = strides[3 * a + 2] * size;
    p.w[a] = w[a];
  }
  p.cos = cos;
  p.sin = sin;
  p.pos = positions;
  p.pos_batch = pos_strides[0];
  p.pos_token = pos_strides[1];
  p.tokens = static_cast<long>(B) * T;
  p.T = T;
  p.H[0] = Hq;
  p.H[1] = Hk;
  p.D = D;
  p.R = R;
  p.rows = rows;
  p.wdt = wdt;
  p.pos64 = pos64;
  p.interleaved = interleaved;
  p.eps = eps;
  p.offset = offset;
  return PBGDN_OK;
}

// The rows can be moved in 16-byte units that pairs do not cross.
static bool rope_units(const RopeParams &p, int dtype, std::initializer_list<const void *> bases) {
  const int E = dtype == PBGDN_F32 ? 4 : 8;
  if (p.D % (2 * E) != 0 || p.R % (2 * E) != 0) return false;
  for (int a = 0; a < 2; ++a)
    if (p.batch[a] % 16 != 0 || p.token[a] % 16 != 0 || p.head[a] % 16 != 0) return false;
  for (const void *b : bases)
    if (!aligned16(b)) return false;
  return true;
}

// Workgroups for items of q and of k: one for every four, or, where that is more than
// `most`, as many of them as their share of the work; at least one each.
static unsigned rope_blocks(RopeParams &p, long items_q, long items_k, long most) {
  long nq = (items_q + ROPE_WAVES - 1) / ROPE_WAVES, nk = (items_k + ROPE_WAVES - 1) / ROPE_WAVES;
  if (nq + nk > most) {
    nq = most * p.H[0] / (p.H[0] + p.H[1]);
    nq = nq < 1 ? 1 : nq < most ? nq : most - 1;
    nk = most - nq;
  }
  p.blocks_q = static_cast<int>(nq);
  return static_cast<unsigned>(nq + nk);
}

template <bool BWD>
static int launch_rope(RopeParams &p, int dtype, bool units, long most, unsigned &blocks, hipStream_t stream) {
  const auto go = [&](auto kernel, long items_q, long items_k) {
    blocks = rope_blocks(p, items_q, items_k, most);
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(ROPE_WAVES * 64), 0, stream, p);
  };
  if (!units) {
    const long nq = p.tokens * p.H[0], nk = p.tokens * p.H[1];
    switch (dtype) {
      case PBGDN_F32: go(rope_any_kernel<PBGDN_F32, BWD>, nq, nk); break;
      case PBGDN_BF16: go(rope_any_kernel<PBGDN_BF16, BWD>, nq, nk); break;
      default: go(rope_any_kernel<PBGDN_F16, BWD>, nq, nk); break;
    }
    return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
  }
  const int lanes = p.D / (dtype == PBGDN_F32 ? 8 : 16);
  const auto by_pairs = [&](auto DT, auto G) {
    constexpr int dt = decltype(DT)::value, g = decltype(G)::value, rows = 64 / g;
    // a token's heads on as many pieces as it takes to have 16 a CU, in the backward, whose
    // workgroups take piece after piece, 64: its last round is then a small part
    DeviceShape shape;
    if (!device_shape(shape)) shape.cus = 256;
    const long want = ((BWD ? 64L : 16L) * shape.cus + p.tokens - 1) / p.tokens;
    for (int a = 0; a < 2; ++a) {
      const int groups = (p.H[a] + rows - 1) / rows;
      p.split[a] = static_cast<int>(want < groups ? want : groups);
    }
    if (p.interleaved)
      go(rope_kernel<dt, g, true, BWD>, p.tokens * p.split[0], p.tokens * p.split[1]);
    else
      go(rope_kernel<dt, g, false, BWD>, p.tokens * p.split[0], p.tokens * p.split[1]);
  };
  const auto by_lanes = [&](auto DT) {
    if (lanes <= 4)
      by_pairs(DT, std::integral_constant<int, 4>{});
    else if (lanes <= 8)
      by_pairs(DT, std::integral_constant<int, 8>{});
    else if (lanes <= 16)
      by_pairs(DT, std::integral_constant<int, 16>{});
    else if constexpr (decltype(DT)::value == PBGDN_F32)  // (16-bit rows end at 16 lanes)
      by_pairs(DT, std::integral_constant<int, 32>{});
  };
  switch (dtype) {
    case PBGDN_F32: by_lanes(std::integral_constant<int, PBGDN_F32>{}); break;
    case PBGDN_BF16: by_lanes(std::integral_constant<int, PBGDN_BF16>{}); break;
    default: by_lanes(std::integral_constant<int, PBGDN_F16>{}); break;
  }
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

}  // namespace pbgdn

extern "C" int pbattn_qk_norm_rope(const void *q, const void *k, int dtype, const int64_t *strides, const void *q_weight,
                                   const void *k_weight, int weight_dtype, float weight_offset, const float *cos,
                                   const float *sin, int rows, const void *positions, int positions64,
                                   const int64_t *pos_strides, void *q_out, void *k_out, int B, int T, int Hq, int Hk, int D,
                                   int R, float eps, int interleaved, void *stream) {
  using namespace pbgdn;
  RopeParams p{};
  const int status = rope_params(p, q, k, dtype, strides, q_weight, k_weight, weight_dtype, weight_offset, cos, sin, rows,
                                 positions, positions64, pos_strides, B, T, Hq, Hk, D, R, eps, interleaved);
  if (status != PBGDN_OK || B == 0 || T == 0) return status;
  if (!q_out || !k_out || !aligned16(q_out) || !aligned16(k_out)) return PBGDN_ERR_INVALID_ARGUMENT;
  p.out[0] = static_cast<unsigned char *>(q_out);
  p.out[1] = static_cast<unsigned char *>(k_out);
  hipStream_t s = static_cast<hipStream_t>(stream);
  debug_poison(q_out, static_cast<size_t>(p.tokens) * Hq * D * attn_bytes(dtype), s);
  debug_poison(k_out, static_cast<size_t>(p.tokens) * Hk * D * attn_bytes(dtype), s);
  unsigned blocks;
  return launch_rope<false>(p, dtype, rope_units(p, dtype, {q, k, q_weight, k_weight, cos, sin}), ROPE_MOST, blocks, s);
}

extern "C" size_t pbattn_qk_norm_rope_bwd_workspace_size(int D) {
  return D > 0 && D <= pbgdn::ROPE_MAX_D ? static_cast<size_t>(pbgdn::rope_bwd_blocks()) * D * sizeof(float) : 0;
}

extern "C" int pbattn_qk_norm_rope_bwd(const void *q, const void *k, int dtype, const int64_t *strides, const void *q_weight,
                                       const void *k_weight, int weight_dtype, float weight_offset, const float *cos,
                                       const float *sin, int rows, const void *positions, int positions64,
                                       const int64_t *pos_strides, const void *grad_q, const void *grad_k, void *dq, void *dk,
                                       void *dq_weight, void *dk_weight, int B, int T, int Hq, int Hk, int D, int R,
                                       float eps, int interleaved, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace pbgdn;
  RopeParams p{};
  const int status = rope_params(p, q, k, dtype, strides, q_weight, k_weight, weight_dtype, weight_offset, cos, sin, rows,
                                 positions, positions64, pos_strides, B, T, Hq, Hk, D, R, eps, interleaved);
  if (status != PBGDN_OK || B == 0 || T == 0) return status;
  if (!grad_q || !grad_k || !dq || !dk || !dq_weight || !dk_weight || !workspace || !aligned16(grad_q) || !aligned16(grad_k) ||
      !aligned16(dq) || !aligned16(dk) || !aligned16(dq_weight) || !aligned16(dk_weight) || !aligned16(workspace) ||
      workspace_bytes < pbattn_qk_norm_rope_bwd_workspace_size(D)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  p.g[0] = static_cast<const unsigned char *>(grad_q);
  p.g[1] = static_cast<const unsigned char *>(grad_k);
  p.out[0] = static_cast<unsigned char *>(dq);
  p.out[1] = static_cast<unsigned char *>(dk);
  p.part = static_cast<float *>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  debug_poison(dq, static_cast<size_t>(p.tokens) * Hq * D * attn_bytes(dtype), s);
  debug_poison(dk, static_cast<size_t>(p.tokens) * Hk * D * attn_bytes(dtype), s);
  debug_poison(workspace, pbattn_qk_norm_rope_bwd_workspace_size(D), s);
  unsigned blocks = 0;
  const int launched = launch_rope<true>(p, dtype, rope_units(p, dtype, {q, k, q_weight, k_weight, cos, sin}),
                                         rope_bwd_blocks(), blocks, s);
  if (launched != PBGDN_OK) return launched;
  hipLaunchKernelGGL(rope_join_kernel, dim3(2 * ((D + JOIN_COLS - 1) / JOIN_COLS)), dim3(JOIN_COLS * JOIN_ROWS), 0, s, p.part,
                     p.blocks_q, static_cast<int>(blocks), D, dq_weight, dk_weight, weight_dtype);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}
