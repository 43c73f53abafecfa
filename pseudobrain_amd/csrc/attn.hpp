// What the attention kernels' sources share on the host side.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"
#include "pbattn.h"

namespace pbgdn {

constexpr int NO_WINDOW = 1 << 30;  // positions stay below it

// A [batch, token, head, D] tensor by its strides in bytes.
struct View {
  const unsigned char *base;
  long batch, token, head;
};

struct WindowParams {
  View q, k, v;
  void *o;
  float *lse;
  const int32_t *cu_q, *cu_k;
  int nseq, Tq, Tk, Hq, Hk, group;
  int window, sinks;
  float c;     // |scale| log2(e), at least the smallest normal number
  int negate;  // scale < 0: q enters with its sign changed
  int slots;   // tiles of a (batch, key head), the empty ones of a packed call included
};

inline bool attn_dtype(int d) { return d == PBGDN_F32 || d == PBGDN_BF16 || d == PBGDN_F16; }
inline int attn_bytes(int d) { return d == PBGDN_F32 ? 4 : 2; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks and fills what forward and backward have in common. PBGDN_OK with
// p.nseq = 0 when there is nothing to do.
int window_params(WindowParams &p, const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                  const int32_t *cu_q, const int32_t *cu_k, int num_seqs, int B, int Tq, int Tk, int Hq, int Hk, int D,
                  float scale, int window, int sinks);

// Tiles of `tile` rows (query tokens x heads of a group) a (batch, key head) has.
inline long window_slots(const WindowParams &p, int tile) {
  const long rows = static_cast<long>(p.Tq) * p.group;
  return p.cu_q ? rows / tile + p.nseq + 1 : (rows + tile - 1) / tile;
}

}  // namespace pbgdn
