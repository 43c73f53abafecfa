// Packed sequences from their lengths, worked out by every workgroup for itself:
// where each sequence's tokens start, and which sequence a token belongs to.
#pragma once

#include "common.hpp"
#include "pbattn.h"

namespace pbgdn {

constexpr int MAX_REQUESTS = PBATTN_MAX_REQUESTS;  // sequences of one call: their starts are held in LDS
constexpr int SCAN_THREADS = 256;
constexpr int SCAN_WAVES = SCAN_THREADS / 64;

// Sum of x over the threads before this one, in `total` over all of them. (64 bits:
// neither wrong counts nor many large ones may wrap around.)
template <int WAVES>
__device__ __forceinline__ long block_scan(long x, long (&waves)[WAVES], long &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long scan = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const long y = __shfl_up(scan, off, 64);
    if (lane >= off) scan += y;
  }
  __syncthreads();
  if (lane == 63) waves[wave] = scan;
  __syncthreads();
  long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += waves[w];
    total += waves[w];
  }
  return before + scan - x;
}

// The last b in [0, n) with start[b] <= t, 0 where there is none: the sequence of
// token t when start[0] = 0 and a next sequence starts past it.
template <typename T>
__device__ __forceinline__ int sequence_of(const T *start, int n, T t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

}  // namespace pbgdn
