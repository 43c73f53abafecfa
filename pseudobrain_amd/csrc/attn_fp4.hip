// The cache held in 4 bits (attn_fp4.hpp): decoding over it (pbattn_fp4_decode),
// its writes (pbattn_fp4_write) and its reading back (pbattn_fp4_read).
#include <type_traits>

#include "attn_decode.hpp"
#include "attn_fp4.hpp"
#include "pages.hpp"

namespace pbgdn {

struct Fp4DecodeParams {
  DecodeParams d;                       // k, v, token, head: the codes'
  const unsigned char *k_scale, *v_scale;  // their strides: a sixteenth of the codes'
};

// Q and the weights enter bfloat16 products as one, two or three parts that sum up to
// them: bfloat16 rows as they are, float16 rows in two, float32 rows in three, all of
// them exactly; the weights of bfloat16 rows are rounded once to 2^-9, those of the
// others cut to 16 and 24 bits. So the cache's values, exact in bfloat16, meet every
// type of row in the same kernel.
template <int DT>
struct Parts {
  static constexpr int N = DT == PBGDN_BF16 ? 1 : DT == PBGDN_F16 ? 2 : 3;
};
// The upper halves of two words.
__device__ __forceinline__ uint32_t upper_halves(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
// Two values as N pairs of bfloat16, cut, not rounded (no part passes the type's range).
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t *out) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    out[i] = upper_halves(a, b);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
}

template <int DT, int D>
struct Fp4 {
  static constexpr int N = Parts<DT>::N;
  static constexpr int ROW = D / 2;           // bytes of a key's codes
  static constexpr int SROW = D / FP4_BLOCK;  // and of its scales
  static constexpr int KSTEPS = D / 32;       // matrix steps of a score
  static constexpr int KW = ROW / 16;         // words a lane reads of a key: one a step
  static constexpr int KSCALES = D == 256 ? 2 : 1;  // and of its scales
  static constexpr int OT = D / 16;           // output tiles: values a lane reads of a value row
  static constexpr int VW = D == 64 ? 1 : OT / 8;   // words that hold them
  static constexpr int KG = 2, KEYS = 16 * KG;      // keys at a time
  // Q in LDS where its parts would take more than 64 registers.
  static constexpr bool q_in_lds(int rb) { return KSTEPS * N * rb > 16; }
  // First of the eight columns that lane group g takes in matrix step s.
  __device__ static constexpr int column(int g, int s) {
    return D == 64 ? 16 * g + 8 * s : 128 * (s / 4) + 32 * g + 8 * (s % 4);
  }
};

template <int DT, int D, int RB>
__global__ __launch_bounds__(DEC_WAVES * 64, 2) void fp4_decode_kernel(const Fp4DecodeParams pp) {
  using K = Fp4<DT, D>;
  using E = Elem<PBGDN_BF16>;
  constexpr int KS = K::KSTEPS, OT = K::OT, KG = K::KG, KEYS = K::KEYS, N = K::N;
  constexpr bool Q_LDS = K::q_in_lds(RB);
  constexpr int JOINS = RB * D <= 256 ? 2 : 1;
  constexpr int Q_UNITS = Q_LDS ? RB * N * KS * 64 : 1;  // 16-byte units: [row tile][part][step][lane]
  typedef float Merge[JOINS][RB * DEC_ROWS * (D + 2)];
  __shared__ union {  // Q's place is the joins' afterwards
    Merge merge;
    v4u32_t q[Q_UNITS];
  } lds;
  PBGDN_POISON_LDS(&lds, sizeof(lds));
  PBGDN_POISON_SYNC();
  v4u32_t *const q_lds = lds.q;
  const DecodeParams &p = pp.d;

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

  // this lane's rows of Q (column c of every row tile), in parts; in LDS, each wave brings in a share
  v4u32_t qf[Q_LDS ? 1 : RB][Q_LDS ? 1 : N][Q_LDS ? 1 : KS];
  int pos[RB];
  constexpr int QB = DT == PBGDN_F32 ? 4 : 2;  // bytes of an element of Q
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + r * DEC_ROWS + c;
    const int rr = row < p.rows ? row : p.rows - 1;
    const int t = rr / p.group;
    pos[r] = len - p.T + t;
    const unsigned char *src = p.q + ((static_cast<long>(b) * p.T + t) * p.Hq + hk * p.group + rr - t * p.group) * (D * QB);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (Q_LDS && s % DEC_WAVES != wave) continue;
      v4u32_t part[N];
      if constexpr (DT == PBGDN_BF16) {
        part[0] = *reinterpret_cast<const v4u32_t *>(src + K::column(g, s) * 2);
        if (p.negate) part[0] ^= 0x80008000u;
      } else {
        float x[8];
        if constexpr (DT == PBGDN_F16) {
          const half8_t h = *reinterpret_cast<const half8_t *>(src + K::column(g, s) * 2);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(h[e]);
        } else {
          const float4_t lo = *reinterpret_cast<const float4_t *>(src + K::column(g, s) * 4),
                         hi = *reinterpret_cast<const float4_t *>(src + K::column(g, s) * 4 + 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[e] = lo[e];
            x[4 + e] = hi[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          uint32_t w[N];
          split_pair<N>(p.negate ? -x[e] : x[e], p.negate ? -x[e + 1] : x[e + 1], w);
#pragma unroll
          for (int i = 0; i < N; ++i) part[i][e / 2] = w[i];
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (Q_LDS)
          q_lds[((r * N + i) * KS + s) * 64 + lane] = part[i];
        else
          qf[r][i][s] = part[i];
      }
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
  const unsigned char *ksbase = pp.k_scale + hk * (p.head / 16), *vsbase = pp.v_scale + hk * (p.head / 16);
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
  // A key's row as lane (c, g) takes it: unit g of key 16 kb + c; its scales.
  uint32_t kf[KG][K::KW], ks[KG][K::KSCALES];
  // Values: lane (c, .) takes columns OT c .. of the keys that its weights belong to.
  uint32_t vf[4 * KG][K::VW], vs[4 * KG];
  const auto load_keys = [&](int rows) __attribute__((always_inline)) {
    const int safe = rows >= 0 ? rows : 0;
#pragma unroll
    for (int kb = 0; kb < KG; ++kb) {
      const long row = __shfl(safe, 16 * kb + c, 64);
      const unsigned char *src = kbase + row * p.token, *ss = ksbase + row * (p.token / 16);
      if constexpr (D == 64) {
        const v2u32_t w = __builtin_nontemporal_load(reinterpret_cast<const v2u32_t *>(src + g * 8));
        kf[kb][0] = w[0];
        kf[kb][1] = w[1];
        ks[kb][0] = ss[g / 2];
      } else {
#pragma unroll
        for (int h = 0; h < D / 128; ++h) {
          const v4u32_t w = __builtin_nontemporal_load(reinterpret_cast<const v4u32_t *>(src + h * 64 + g * 16));
#pragma unroll
          for (int e = 0; e < 4; ++e) kf[kb][4 * h + e] = w[e];
          ks[kb][h] = ss[4 * h + g];
        }
      }
    }
  };
  const auto load_values = [&](int rows) __attribute__((always_inline)) {
    const int safe = rows >= 0 ? rows : 0;
#pragma unroll
    for (int i = 0; i < 4 * KG; ++i) {
      const long row = __shfl(safe, i / 4 * 16 + 4 * g + i % 4, 64);
      const unsigned char *src = vbase + row * p.token + c * (OT / 2);
      if constexpr (D == 64) {
        vf[i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t *>(src));
      } else if constexpr (D == 128) {
        vf[i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(src));
      } else {
        const v2u32_t w = __builtin_nontemporal_load(reinterpret_cast<const v2u32_t *>(src));
        vf[i][0] = w[0];
        vf[i][1] = w[1];
      }
      vs[i] = vsbase[row * (p.token / 16) + c * OT / FP4_BLOCK];
    }
  };
  // A block's keys are fetched while the one before is weighed, its values while the
  // scores are formed; the pages of the block after are asked for before those values.
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
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v4u32_t a[KG];
#pragma unroll
      for (int kb = 0; kb < KG; ++kb) a[kb] = fp4_unpack8(kf[kb][s], fp4_scale(ks[kb][D == 256 ? s / 4 : 0]));
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          v4u32_t q;
          if constexpr (Q_LDS)
            q = q_lds[((r * N + i) * KS + s) * 64 + lane];
          else
            q = qf[r][i][s];
#pragma unroll
          for (int kb = 0; kb < KG; ++kb) sc[r][kb] = E::mma16(a[kb], q, sc[r][kb]);
        }
    }
    const int next = more ? cache_row(page, place) : -1;
    if constexpr (more) load_keys(next);
    if (!all) {  // values of absent keys: zeros, whatever the row they were read from holds
#pragma unroll
      for (int i = 0; i < 4 * KG; ++i) {
        const bool in = __shfl(valid, i / 4 * 16 + 4 * g + i % 4, 64) >= 0;
#pragma unroll
        for (int x = 0; x < K::VW; ++x) vf[i][x] = in ? vf[i][x] : 0u;
        vs[i] = in ? vs[i] : 127u;
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
    // O^T += V^T P; element e of the lane's values makes output tile e
    v4u32_t w[RB][KG / 2][N];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int h = 0; h < KG / 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = sc[r][2 * h + i / 2][2 * (i % 2)], y = sc[r][2 * h + i / 2][2 * (i % 2) + 1];
          if constexpr (N == 1) {
            w[r][h][0][i] = E::pack(x, y);
          } else {
            uint32_t part[N];
            split_pair<N>(x, y, part);
#pragma unroll
            for (int n = 0; n < N; ++n) w[r][h][n][i] = part[n];
          }
        }
    const auto pair_of_tiles = [&](auto E0) __attribute__((always_inline)) {  // tiles 2 e and 2 e + 1
      constexpr int e = decltype(E0)::value;
#pragma unroll
      for (int h = 0; h < KG / 2; ++h) {
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fp4_pair<e % 4>(vf[8 * h + i][e / 4], fp4_scale(vs[8 * h + i]));
        v4u32_t lo, hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
          hi[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
        }
#pragma unroll
        for (int n = 0; n < N; ++n)
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
    if constexpr (more) {
      lookup(blk + 2 * DEC_WAVES, page, place);
      load_values(next);
      valid = next;
    }
  };
  int blk = begin + wave;
  for (; blk + DEC_WAVES < end; blk += DEC_WAVES) step(blk, std::false_type{});
  if (blk < end) step(blk, std::true_type{});
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
      const auto value = [&](const unsigned char *codes, const unsigned char *scales, int d) __attribute__((always_inline)) {
        return bf16_bits_to_float(static_cast<u16>(fp4_pair<0>(codes[d / 2] >> (d % 2 * 4), fp4_scale(scales[d / FP4_BLOCK]))));
      };
      for (int at = begin + wave; at < end; at += DEC_WAVES) {
        int pg, place_;
        lookup(at, pg, place_);
        const int rows = cache_row(pg, place_);
        for (int key = 0; key < KEYS; ++key) {
          const int slot_ = __shfl(rows, key, 64), u = at * KEYS + key, j = u < range.sinks ? u : u + range.delta;
          if (slot_ < 0) continue;
          const long cr = static_cast<long>(slot_) * p.token;
          float dot = 0.0f;
          for (int d = g * (D / 4); d < (g + 1) * (D / 4); ++d)
            dot += value(kbase + cr, ksbase + cr / 16, d) * load_elem(qrow, d, DT);
          dot = add_xor32(add_xor16(dot)) * sign;
          if (!sees(pos[r], j, p.window, p.sinks)) continue;
          const float w = __builtin_amdgcn_exp2f((dot - base) * p.c);
#pragma unroll
          for (int e = 0; e < OT; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][e][i] += w * value(vbase + cr, vsbase + cr / 16, (4 * g + i) * OT + e);
        }
      }
    }
  }
  if constexpr (Q_LDS) __syncthreads();
  join_waves<RB, D, JOINS>(lds.merge, m, l, o, wave, lane, p.c);
  if (wave != 0) return;
  store_decoded<DT, D, RB, OT>(p, share, b, hk, row0, slot, lane, m, l, o);
}

// ---------------------------------------------------------------------------
// Writes: eight values of a key and of a value a thread, four threads a scale.
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
// rows of its tokens, and copies them.
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
  constexpr int BYTES = DT == PBGDN_F32 ? 4 : 2;
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
  const int per = p.Hk * p.eighths;
  for (int i = threadIdx.x; i < n * per; i += SCAN_THREADS) {
    const int tok = i / per, x = i - tok * per, hd = x / p.eighths, u = x - hd * p.eighths;
    const long row = rows[tok];
    uint32_t k = 0, v = 0, ks = 127, vs = 127;
    if (row >= 0) {
      const long from = row + hd * p.cache.head, scales = from / 16 + u / 4;
      k = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p.cache.k + from + u * 4));
      v = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p.cache.v + from + u * 4));
      ks = p.cache.k_scale[scales];
      vs = p.cache.v_scale[scales];
    }
    const long to = (static_cast<long>(first + tok) * per + x) * (8 * BYTES);
    store8<DT>(static_cast<unsigned char *>(p.k) + to, k, fp4_scale(ks));
    store8<DT>(static_cast<unsigned char *>(p.v) + to, v, fp4_scale(vs));
  }
}

template <int DT, int D>
static int launch_fp4(Fp4DecodeParams &p, hipStream_t stream) {
  const auto run = [&](auto kernel, int rb) {
    const unsigned blocks = decode_blocks(p.d, rb);
    if (blocks) hipLaunchKernelGGL(kernel, dim3(blocks), dim3(DEC_WAVES * 64), 0, stream, p);
    return blocks != 0;
  };
  const bool ok = p.d.rows <= DEC_ROWS ? run(fp4_decode_kernel<DT, D, 1>, 1) : run(fp4_decode_kernel<DT, D, 2>, 2);
  if (!ok) return PBGDN_ERR_UNSUPPORTED;
  launch_join<DT, D>(p.d, stream);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

template <int DT>
static int dispatch_fp4(Fp4DecodeParams &p, int D, hipStream_t stream) {
  switch (D) {
    case 64: return launch_fp4<DT, 64>(p, stream);
    case 128: return launch_fp4<DT, 128>(p, stream);
    default: return launch_fp4<DT, 256>(p, stream);
  }
}

// Parts wanted over all sequences.
static int fp4_target(int Hk, int rows) {
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  const int tiles = (rows + 2 * DEC_ROWS - 1) / (2 * DEC_ROWS);
  const int t = 8 * shape.cus / (Hk * tiles);
  return t > 1 ? t : 1;
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
  if (!decode_sizes_ok(B, T, Hq, Hk, D)) return 0;
  const int rows = Hq / Hk * T;
  const size_t slots = static_cast<size_t>(fp4_target(Hk, rows)) + B;
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
  const long page_rows = cache.token > 0 ? cache.page_stride / cache.token : 0;
  if (page_rows * (num_pages > 0 ? num_pages - 1 : 0) + page_size > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  if (workspace_bytes < pbattn_fp4_decode_workspace_size(B, T, Hq, Hk, D)) return PBGDN_ERR_INVALID_ARGUMENT;
  Fp4DecodeParams pp{};
  DecodeParams &p = pp.d;
  p.q = static_cast<const unsigned char *>(q);
  p.k = cache.k;
  p.v = cache.v;
  pp.k_scale = cache.k_scale;
  pp.v_scale = cache.v_scale;
  p.token = cache.token;
  p.head = cache.head;
  p.page_rows = static_cast<int>(page_rows);
  p.page = page_size;
  p.num_pages = max_pages > 0 ? num_pages : 0;  // (no table: no keys)
  p.max_pages = max_pages;
  p.table = page_table;
  p.lengths = lengths;
  p.o = o;
  p.lse = lse;
  decode_call(p, B, T, Hq, Hk, scale, window, sinks, fp4_target(Hk, Hq / Hk * T));
  const size_t used = decode_workspace(p, workspace, D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  debug_poison(o, static_cast<size_t>(B) * T * Hq * D * attn_bytes(dtype), s);
  if (lse) debug_poison(lse, static_cast<size_t>(B) * T * Hq * sizeof(float), s);
  debug_poison(workspace, used, s);
  switch (dtype) {
    case PBGDN_F32: return dispatch_fp4<PBGDN_F32>(pp, D, s);
    case PBGDN_BF16: return dispatch_fp4<PBGDN_BF16>(pp, D, s);
    default: return dispatch_fp4<PBGDN_F16>(pp, D, s);
  }
}

extern "C" int pbattn_fp4_write(const void *k, const void *v, int dtype, const int64_t *kv_strides, void *k_cache,
                                void *v_cache, void *k_scale, void *v_scale, const int64_t *strides, int page_size,
                                int num_pages, const int64_t *slots, int N, int Hk, int D, void *stream) {
  using namespace pbgdn;
  if (N < 0 || Hk <= 0 || D <= 0 || !attn_dtype(dtype) || !kv_strides || !strides || page_size <= 0 || num_pages < 0) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  if (!fp4_width(D)) return PBGDN_ERR_UNSUPPORTED;
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
  if (!fp4_width(D) || B > MAX_REQUESTS) return PBGDN_ERR_UNSUPPORTED;
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
  // Tokens of a workgroup: as many as leave the GPU four workgroups a CU, READ_TOKENS at most.
  DeviceShape shape;
  if (!device_shape(shape)) shape.cus = 256;
  const int even = (tokens + 4 * shape.cus - 1) / (4 * shape.cus);
  p.per_block = even < 1 ? 1 : even > READ_TOKENS ? READ_TOKENS : even;
  if (static_cast<long>(p.per_block) * Hk * p.eighths > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  const int blocks = (tokens + p.per_block - 1) / p.per_block;
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
