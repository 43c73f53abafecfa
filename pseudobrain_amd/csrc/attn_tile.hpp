// Tiles of the attention kernels (gfx950): rows of D elements in LDS, staged by
// direct-to-LDS loads, and the two matrix products every kernel is made of.
//
// All kernels keep scores transposed or not so that one side of every product
// lives in registers, on the 32x32 matrix instructions (lane l: n = l & 31,
// h = l >> 5; an accumulator holds rows 8 (i / 4) + 4 h + i % 4 of column n in
// its element i):
//
//   rows product   X[r][n] = sum_d M[r][d] Y[n][d]
//                  M a tile in LDS, read 16 bytes of a row at a time; Y held by
//                  the wave, lane (n, h) with units 2 s + h of row n.
//   cols product   Z[d][n] += sum_r M[r][d] X[r][n]
//                  X as the rows product left it: its accumulator is the B
//                  operand as it stands, because the order of the contraction
//                  index is free as long as both operands agree; M's columns
//                  come from LDS by transposing reads (16-bit) or single
//                  elements (float32).
//
// So S = K Q^T then O^T = V^T P needs no exchange between lanes: a query is one
// lane pair's column from the score to the output.
#pragma once

#include "common.hpp"
#include "pbattn.h"

namespace pbgdn {

typedef float float16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Weights are exp2(s c - m c), one fused operation a score: the rounding of m c
// is the same for every score of a row and cancels in its sum. Past this |m c|
// it would no longer stay near 1 (2^-24 of it), and the kernels subtract first.
constexpr float EXACT_SCORES = 65536.0f;

// The reference the weights are taken against moves only when a score passes it
// by more than LAG powers of two: most tiles leave the sums as they are. Weights
// stay below 2^8.
constexpr float LAG = 8.0f;

// Element types: bytes, one matrix step of the rows product (a 16-byte unit per
// lane and side) and the packing of two float32 values.
template <int DT>
struct Elem;

template <>
struct Elem<PBGDN_BF16> {
  static constexpr int BYTES = 2;
  using T = u16;
  __device__ static float16_t mma(v4u32_t a, v4u32_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
  __device__ static float4_t mma16(v4u32_t a, v4u32_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  }
  __device__ static float4_t mma16(v2u32_t a, v2u32_t b, float4_t c) {  // 16 wide in the contraction
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4_t, a), __builtin_bit_cast(i16x4_t, b), c,
                                                     0, 0, 0);
  }
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x), static_cast<__bf16>(y)});
  }
  __device__ static float low(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ static float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};

template <>
struct Elem<PBGDN_F16> {
  static constexpr int BYTES = 2;
  using T = half_t;
  __device__ static float16_t mma(v4u32_t a, v4u32_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  }
  __device__ static float4_t mma16(v4u32_t a, v4u32_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  }
  __device__ static float4_t mma16(v2u32_t a, v2u32_t b, float4_t c) {
    return mfma16(__builtin_bit_cast(half4_t, a), __builtin_bit_cast(half4_t, b), c);
  }
  __device__ static uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, half2_t{static_cast<half_t>(x), static_cast<half_t>(y)});
  }
  __device__ static float low(uint32_t w) { return static_cast<float>(__builtin_bit_cast(half2_t, w)[0]); }
  __device__ static float high(uint32_t w) { return static_cast<float>(__builtin_bit_cast(half2_t, w)[1]); }
};

template <>
struct Elem<PBGDN_F32> {
  static constexpr int BYTES = 4;
  using T = float;
  __device__ static float16_t mma(v4u32_t a, v4u32_t b, float16_t c) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ float16_t zero16() {
  float16_t z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// Row, within 32, of element i of an accumulator in lane half h.
__device__ __forceinline__ constexpr int acc_row(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

// ---------------------------------------------------------------------------
// A tile's place in LDS: row r at r * ROW bytes, its 16-byte unit u at unit
// u ^ swz(r). The permutation spreads both read patterns over all 64 banks: the
// 16 rows of a quarter wave's rows-product read fall on 16 different units of
// 256 bytes, and the 4 rows x 64 bytes of a transposing read on one line.
// ---------------------------------------------------------------------------
template <int DT, int D>
struct Tile {
  using E = Elem<DT>;
  static constexpr int ROW = D * E::BYTES;  // bytes of a row
  static constexpr int UNITS = ROW / 16;
  static constexpr int STEPS = UNITS / 2;   // matrix steps of a rows product
  static constexpr int MB = D / 32;         // 32-row blocks of a cols product's result
  static constexpr int PER_DMA = 64 / UNITS > 0 ? 64 / UNITS : 1;  // rows a wave-wide load fills (UNITS <= 64)
  static_assert(UNITS == 8 || UNITS == 16 || UNITS == 32 || UNITS == 64, "rows of 128 to 1024 bytes");

  __device__ static __forceinline__ int swz(int r) {
    return UNITS == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
  }

  // Rows product's read: lane base, then unit 2 s of rows r0 .. r0 + 31.
  __device__ static __forceinline__ uint32_t rows_base(int n, int h) { return n * ROW + ((h ^ swz(n)) * 16); }
  __device__ static __forceinline__ v4u32_t rows(const unsigned char *tile, uint32_t base, int r0, int s) {
    const uint32_t lo = (2 * s) % 16, hi = (2 * s) / 16;
    return *reinterpret_cast<const v4u32_t *>(tile + ((base ^ (lo * 16)) + hi * 256 + r0 * ROW));
  }

  // Cols product's read, 16-bit: the A operand of matrix step t (16 rows from
  // r0 + 16 t) for columns 32 m .. 32 m + 31.
  __device__ static __forceinline__ uint32_t cols_base(int lane) {
    if constexpr (E::BYTES == 2) {
      const int c = lane & 15, dh = (lane >> 4) & 1, h = lane >> 5;
      const int r = 4 * h + (c >> 2);
      return r * ROW + (((2 * dh + ((c & 3) >> 1)) ^ swz(r)) * 16) + 8 * (c & 1);
    } else {
      const int n = lane & 31, h = lane >> 5;
      return 4 * h * ROW + (((n >> 2) ^ h) * 16) + 4 * (n & 3);
    }
  }
  __device__ static __forceinline__ v2u32_t tr(const unsigned char *tile, uint32_t base, int row, int m, int b) {
    const uint32_t lo = ((4 * m) % UNITS % 16) ^ (2 * b), hi = (4 * m) / 16;
    const uint32_t at = (base ^ (lo * 16)) + hi * 256 + row * ROW;
    return __builtin_bit_cast(v2u32_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) i16x4_t *)(tile + at)));
  }
  __device__ static __forceinline__ v4u32_t cols(const unsigned char *tile, uint32_t base, int r0, int t, int m) {
    const v2u32_t x = tr(tile, base, r0 + 16 * t, m, 0), y = tr(tile, base, r0 + 16 * t + 8, m, 1);
    return v4u32_t{x[0], x[1], y[0], y[1]};
  }
  // The same, float32: element i of the contraction.
  __device__ static __forceinline__ float col1(const unsigned char *tile, uint32_t base, int r0, int i, int m) {
    const uint32_t k = ((8 * m) % 16) ^ ((i % 4) << 2) ^ ((2 * (i / 4)) & 3), hi = (8 * m) / 16;
    return *reinterpret_cast<const float *>(tile + ((base ^ (k * 16)) + hi * 256 + (r0 + 8 * (i / 4) + i % 4) * ROW));
  }

  // The products, KB x 32 rows of a tile at once. Reads run AHEAD steps before
  // the matrix instruction that takes them, and nothing is moved across a step:
  // left to itself the compiler reads one step ahead, and every instruction waits
  // for LDS (three to four of them, 32 cycles each, cover its latency).
  static constexpr int AHEAD = 3;

  // x[kb] = M[32 kb ..] Y^T; y: STEPS units a lane.
  template <int KB>
  __device__ static __forceinline__ void rows_product(const unsigned char *tile, uint32_t base, const v4u32_t *y,
                                                      float16_t *x) {
    v4u32_t a[AHEAD + 1];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) x[kb] = zero16();
#pragma unroll
    for (int j = -AHEAD; j < KB * STEPS; ++j) {
      if (j + AHEAD < KB * STEPS)
        a[(j + AHEAD) % (AHEAD + 1)] = rows(tile, base, 32 * ((j + AHEAD) % KB), (j + AHEAD) / KB);
      __builtin_amdgcn_sched_barrier(0);
      if (j >= 0) x[j % KB] = E::mma(a[j % (AHEAD + 1)], y[j / KB], x[j % KB]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // The same for 32 rows with Y's rows in LDS too (two reads a step, of which two
  // are as much ahead).
  __device__ static __forceinline__ float16_t rows_product_lds(const unsigned char *tile, const unsigned char *other,
                                                               uint32_t base) {
    constexpr int LDS_AHEAD = 2;
    v4u32_t a[LDS_AHEAD + 1], b[LDS_AHEAD + 1];
    float16_t x = zero16();
#pragma unroll
    for (int j = -LDS_AHEAD; j < STEPS; ++j) {
      if (j + LDS_AHEAD < STEPS) {
        a[(j + LDS_AHEAD) % (LDS_AHEAD + 1)] = rows(tile, base, 0, j + LDS_AHEAD);
        b[(j + LDS_AHEAD) % (LDS_AHEAD + 1)] = rows(other, base, 0, j + LDS_AHEAD);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (j >= 0) x = E::mma(a[j % (LDS_AHEAD + 1)], b[j % (LDS_AHEAD + 1)], x);
      __builtin_amdgcn_sched_barrier(0);
    }
    return x;
  }

  // X as the B operand of a cols product.
  struct Operand {
    v4u32_t w[E::BYTES == 2 ? 2 : 4];
  };
  __device__ static __forceinline__ Operand operand(const float16_t &x) {
    Operand o;
    if constexpr (E::BYTES == 2) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) o.w[t][j] = E::pack(x[8 * t + 2 * j], x[8 * t + 2 * j + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) o.w[i / 4][i % 4] = __float_as_uint(x[i]);
    }
    return o;
  }
  // z[m] += columns 32 m .. of M[32 kb ..] times x[kb], every m and kb.
  template <int KB>
  __device__ static __forceinline__ void cols_product(const unsigned char *tile, uint32_t base, const Operand *x,
                                                      float16_t *z) {
    constexpr int PER = (E::BYTES == 2 ? 2 : 16) * MB, N = KB * PER;  // instructions of 32 rows
    v4u32_t a[AHEAD + 1];
#pragma unroll
    for (int j = -AHEAD; j < N; ++j) {
      const int r = j + AHEAD;
      if (r < N) {
        if constexpr (E::BYTES == 2)
          a[r % (AHEAD + 1)] = cols(tile, base, 32 * (r / PER), r % PER / MB, r % MB);
        else
          a[r % (AHEAD + 1)][0] = __float_as_uint(col1(tile, base, 32 * (r / PER), r % PER / MB, r % MB));
      }
      __builtin_amdgcn_sched_barrier(0);
      if (j >= 0) {
        const v4u32_t y = a[j % (AHEAD + 1)];
        const Operand &o = x[j / PER];
        const int t = j % PER / MB, m = j % MB;
        if constexpr (E::BYTES == 2)
          z[m] = E::mma(y, o.w[t], z[m]);
        else
          z[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(y[0]), __uint_as_float(o.w[t / 4][t % 4]), z[m], 0,
                                                      0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// A row of transposed accumulators: column d of z[d / 32], times f, as DT.
template <int DT, int D>
__device__ __forceinline__ void store_row(void *dst, const float16_t *z, int h, float f) {
  using E = Elem<DT>;
#pragma unroll
  for (int m = 0; m < D / 32; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4_t x = {z[m][4 * e] * f, z[m][4 * e + 1] * f, z[m][4 * e + 2] * f, z[m][4 * e + 3] * f};
      const int d = 32 * m + 8 * e + 4 * h;
      if constexpr (E::BYTES == 2) {
        *reinterpret_cast<v2u32_t *>(static_cast<unsigned char *>(dst) + 2 * d) =
            v2u32_t{E::pack(x[0], x[1]), E::pack(x[2], x[3])};
      } else {
        *reinterpret_cast<float4_t *>(static_cast<unsigned char *>(dst) + 4 * d) = x;
      }
    }
}

// Loads of x have returned when the code after this runs. (Registers loaded
// before a loop and first used in it are otherwise waited for inside it, by a
// counter that the loop's own loads share.)
template <typename T>
__device__ __forceinline__ void settle(T &x) {
  asm volatile("" : "+v"(x));
}

// x, of which the compiler knows nothing more: what is computed from it inside a
// loop is computed there instead of being kept in registers across it.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A wave-uniform value in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---------------------------------------------------------------------------
// Direct-to-LDS loads: 16 bytes per lane, lane l to `lds` + 16 l. Assembly, so
// that the compiler does not wait for them before LDS reads it cannot tell
// apart; the waits are the ones written (wait_dma, then a barrier).
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  typedef __attribute__((address_space(3))) const unsigned char lds_byte;
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_byte *)p));
}
// From `off` bytes into a buffer resource; what lies outside it arrives as zeros.
__device__ __forceinline__ void dma(v4u32_t desc, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(desc)
               : "memory");
}
// 4 bytes per lane, lane l to `lds` + 4 l: for sources aligned to no more.
__device__ __forceinline__ void dma4(v4u32_t desc, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(desc)
               : "memory");
}
// From a 64-bit address per lane.
__device__ __forceinline__ void dma(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src)
               : "memory");
}
// (the words in scalar registers whatever unit the compiler worked them out on)
__device__ __forceinline__ v4u32_t dma_desc(const void *base, long bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return v4u32_t{static_cast<uint32_t>(uniform(static_cast<int>(a))),
                 static_cast<uint32_t>(uniform(static_cast<int>(a >> 32))) & 0xffffu,
                 static_cast<uint32_t>(uniform(static_cast<int>(bytes > 0 ? bytes : 0))),
                 static_cast<uint32_t>(RSRC_WORD3)};
}
// All but the last N loads of this wave have arrived.
template <int N>
__device__ __forceinline__ void wait_dma() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// This wave's LDS reads have returned.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// Every wave has reached this point; its LDS reads have returned.
__device__ __forceinline__ void block_sync() {
  wait_lds();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// x and its other lane half's (lane ^ 32).
__device__ __forceinline__ float max_xor32(float x) {
  float a = x, b = x;
  swap32(a, b);
  return fmaxf(a, b);
}

// The logarithm of a row's softmax sum, l against its largest score m. -infinity is
// left to rows that see no key: others end at the type's largest values.
__device__ __forceinline__ float row_lse(float m, float l, float c) {
  if (!(l > 0.0f)) return l == 0.0f ? -INFINITY : l;
  const float powers = m * c;
  const float lse = fabsf(powers) < INFINITY ? (powers + __builtin_amdgcn_logf(l)) * LN2 : m * LN2 * c;
  return fminf(fmaxf(lse, -__FLT_MAX__), __FLT_MAX__);
}

// ---------------------------------------------------------------------------
// Which keys a query sees: position p sees key j when j <= p and
// (j > p - window or j < sinks). Without branches, and used to select, never to
// guard the write of one element of a matrix accumulator: hipcc (ROCm 7.2) has
// dropped such a guarded write.
// ---------------------------------------------------------------------------
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) {
  return (j <= p) & ((j > p - window) | (j < sinks));
}

// One sequence of a call.
struct Seq {
  int q0, nq;  // its first query token and how many
  int k0, nk;  // its first key token and how many
};

// Sequence b's bounds, clamped into the tensors whatever the boundaries hold.
// b == nseq: what a packed call's last boundaries leave over; KEYS says whether
// the caller walks keys (the leftover has no queries) or queries (no keys).
__device__ __forceinline__ int boundary(const int32_t *cu, int i, int total) {
  const int x = cu[i];
  return x < 0 ? 0 : x > total ? total : x;
}
template <bool KEYS>
__device__ __forceinline__ Seq sequence(const int32_t *cu_q, const int32_t *cu_k, int b, int nseq, int Tq, int Tk) {
  if (!cu_q) return Seq{0, Tq, 0, Tk};
  Seq s;
  s.q0 = boundary(cu_q, b, Tq);
  s.nq = (b < nseq ? boundary(cu_q, b + 1, Tq) : KEYS ? s.q0 : Tq) - s.q0;
  const int32_t *cu = cu_k ? cu_k : cu_q;
  s.k0 = boundary(cu, b, Tk);
  s.nk = (b < nseq ? boundary(cu, b + 1, Tk) : KEYS ? Tk : s.k0) - s.k0;
  return s;
}

// Tiles of a packed call without a list of them: sequence b's tiles start at
// slot floor(first[b] rows / TILE) + b, which leaves each of them at least the
// ceil(rows / TILE) slots it needs, whatever the lengths; slots past that are
// empty. What the boundaries leave over counts as sequence n. Returns the
// sequence of `slot` by bisection.
__device__ __forceinline__ int slot_start(const int32_t *cu, int b, int total, int rows, int tile) {
  return static_cast<int>(static_cast<long>(boundary(cu, b, total)) * rows / tile) + b;
}
__device__ __forceinline__ int slot_sequence(const int32_t *cu, int n, int total, int rows, int tile, int slot) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (slot_start(cu, mid, total, rows, tile) <= slot)
      lo = mid;
    else
      hi = mid - 1;
  }
  return uniform(lo);
}

// ---------------------------------------------------------------------------
// The keys a block of rows sees, in order: the sinks [0, sinks), then from
// `lo` on. Index u is key u below `sinks`, key u + delta from there.
struct KeyRange {
  int sinks, delta, count;
};
__device__ __forceinline__ KeyRange key_range(int p_first, int p_last, int window, int sinks) {
  KeyRange r;
  const int low = p_first - window + 1;
  const int lo = low > 0 ? low : 0;
  r.sinks = sinks < lo ? sinks : lo;
  r.delta = lo - r.sinks;
  r.count = p_last < 0 ? 0 : r.sinks + p_last - lo + 1;
  return r;
}

// How many of a workgroup's key tiles a wave whose last row stands at w_last
// looks at: those up to the one that holds the key there. (The rest of the tiles
// are a loop of their own, in which it only keeps step with the staging: around
// a way past the products inside one loop, the compiler moves every accumulator
// between register files.)
__device__ __forceinline__ int wave_tiles(const KeyRange &r, int tiles, int w_last, int bn) {
  const int n = w_last < 0 ? 0 : (w_last - r.delta) / bn + 1;
  return n < tiles ? n : tiles;
}
// Every row of the wave sees every key of the tile from u0 on.
__device__ __forceinline__ bool whole_tile(const KeyRange &r, int u0, int bn, int w_first, int w_last, int window) {
  return u0 >= r.sinks && u0 + bn - 1 + r.delta <= w_first && u0 + r.delta > w_last - window;
}

// Stages rows u0 .. of a key range into tiles of K and V: wave w of NW fills its
// share of the loads, load i STEP rows further on. A lane's offset changes from
// load to load by whole rows and by the permutation of the row's units, which
// repeats every 16 rows: VARS offsets, kept in registers, serve all loads. With
// HELD false they are worked out at each tile, where registers are scarce (a
// spilled one would be read back through the loads' own counter, and so wait for
// all of them).
template <int DT, int D, int BN, int NW, bool HELD = true>
struct KeyStage {
  using L = Tile<DT, D>;
  static constexpr int STEP = NW * L::PER_DMA, LOADS = BN / STEP, TILE = BN * L::ROW;
  static constexpr int VARS = STEP >= 16 || LOADS == 1 ? 1 : 16 / STEP < LOADS ? 16 / STEP : LOADS;
  static_assert(LOADS * STEP == BN, "whole loads");
  const unsigned char *k, *v;
  long k_stride, v_stride;
  KeyRange range;
  int wave;
  uint32_t k_at[VARS], v_at[VARS];

  // this lane's row of the first load, and its unit of load i
  __device__ __forceinline__ static int row_of(int wave, int lane) { return wave * L::PER_DMA + lane / L::UNITS; }
  __device__ __forceinline__ static uint32_t unit_of(int row, int lane, int i) {
    return ((lane % L::UNITS) ^ L::swz(row) ^ L::swz(i * STEP % 16)) * 16;
  }
  __device__ __forceinline__ static void offsets(int wave, int lane, long stride, uint32_t *at) {
    const int row = row_of(wave, lane);
#pragma unroll
    for (int i = 0; i < VARS; ++i)
      at[i] = (row + i * STEP) * static_cast<uint32_t>(stride) + unit_of(row, lane, i);
  }

  __device__ __forceinline__ KeyStage(const unsigned char *k_, long ks, const unsigned char *v_, long vs,
                                      const KeyRange &r, int wave_, int lane)
      : k(k_), v(v_), k_stride(ks), v_stride(vs), range(r), wave(wave_) {
    if constexpr (HELD) {
      offsets(wave, lane, ks, k_at);
      offsets(wave, lane, vs, v_at);
    }
  }

  __device__ __forceinline__ void one(const unsigned char *base, long stride, const uint32_t *held, int u0,
                                      unsigned char *lds) const {
    const uint32_t to = uniform(lds_address(lds) + wave * 1024);
    if (u0 >= range.sinks) {  // one run of keys
      const int left = range.count - u0, rows = left < BN ? left : BN;
      const v4u32_t desc = dma_desc(base + (u0 + range.delta) * stride, (rows - 1) * stride + L::ROW);
      uint32_t at[VARS];
      if constexpr (!HELD) offsets(wave, opaque(threadIdx.x & 63), stride, at);
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        dma(desc, (HELD ? held : at)[i % VARS] + static_cast<uint32_t>(i / VARS * VARS * STEP) * static_cast<uint32_t>(stride),
            to + i * NW * 1024);
    } else {  // sinks and the window's start in one tile; rows past the end repeat the last key
      const int lane = opaque(threadIdx.x & 63), row = row_of(wave, lane);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        int u = u0 + row + i * STEP;
        u = u < range.count ? u : range.count - 1;
        const long j = u < range.sinks ? u : u + range.delta;
        dma(base + j * stride + unit_of(row, lane, i), to + i * NW * 1024);
      }
    }
  }
  __device__ __forceinline__ void keys(int it, unsigned char *tile) const { one(k, k_stride, k_at, it * BN, tile); }
  __device__ __forceinline__ void values(int it, unsigned char *tile) const { one(v, v_stride, v_at, it * BN, tile); }
  // Tile `it` into `buffer`: K, and V two tiles further on.
  __device__ __forceinline__ void tile(int it, unsigned char *buffer) const {
    keys(it, buffer);
    values(it, buffer + 2 * TILE);
  }
};

// Position of a workgroup in the call: the (batch, key head) `group` and its
// tile `slot`. Workgroups go to the XCDs in turn, and each XCD has its own L2:
// the tiles of a group, which share keys, stay on one XCD (or on as few as
// there are groups for), the longest of a causal call first.
__device__ __forceinline__ void place(int id, int groups, int slots, int &group, int &slot) {
  if (groups % 8 == 0) {
    const int x = id & 7, i = id >> 3;
    group = x + 8 * (i / slots);
    slot = i % slots;
  } else {
    group = id % groups;
    slot = id / groups;
  }
  // (divisions are done in vector registers: say that the results are uniform)
  group = uniform(group);
  slot = uniform(slots - 1 - slot);
}

}  // namespace pbgdn
