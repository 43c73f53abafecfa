// The pages of a paged cache, given and taken back on the device
// (pbattn_pages_extend, pbattn_pages_release).
//
// Both are sums over the requests and then one independent piece of work for each
// token or page: every workgroup forms the sums for itself (a scan over at most 4,096
// requests in LDS), finds its pieces' requests by bisection and writes them, so that a
// call is one launch and needs nothing kept between workgroups. Bound by latency: the
// launch, the requests' numbers, three scans, the table's entry (64 requests: release 3.6
// us, extend 4.7; 233 with 4,000 tokens 4.1 and 6.1).
#include "attn.hpp"
#include "pages.hpp"
#include "device.hpp"

namespace pbgdn {

struct PoolParams {
  int32_t *table;
  long table_row;           // the table's row stride, entries
  const int32_t *a, *b;     // extend: lengths and counts; release: first and end
  int32_t *free_pages;
  const int32_t *num_free;
  int32_t *num_free_out;
  int64_t *slots;
  int32_t *positions, *cu, *lengths_out;
  int B, max_pages, page, capacity, tokens;
};

__device__ __forceinline__ int pool_height(const PoolParams &p) {
  const int n = *p.num_free;
  return n < 0 ? 0 : n < p.capacity ? n : p.capacity;
}
__device__ __forceinline__ int pages_of(long tokens, int page) { return static_cast<int>((tokens + page - 1) / page); }

// A request's share of an extension.
struct Want {
  long count;      // new tokens
  int held, rows;  // pages before and after
  bool fits;       // its tokens and its row of the table
};
__device__ __forceinline__ Want want(const PoolParams &p, int b, long asked) {
  const int len = p.a[b], count = p.b[b];
  Want w;
  w.count = count > 0 ? count : 0;
  const long after = static_cast<long>(len > 0 ? len : 0) + w.count, room = static_cast<long>(p.max_pages) * p.page;
  w.fits = (len >= 0) & (after <= room) & (asked + w.count <= p.tokens);
  w.held = w.fits ? pages_of(len, p.page) : 0;
  w.rows = w.fits ? pages_of(after, p.page) : 0;
  return w;
}

// Tokens a thread: one, so that a prompt's tokens spread over the GPU.
__global__ __launch_bounds__(SCAN_THREADS) void extend_kernel(const PoolParams p) {
  __shared__ int start[MAX_REQUESTS], source[MAX_REQUESTS];  // first token; pool entry of the request's page 0, were it new
  __shared__ long waves[SCAN_WAVES];
  PBGDN_POISON_LDS(start, sizeof(start));
  PBGDN_POISON_LDS(source, sizeof(source));
  PBGDN_POISON_SYNC();
  const int each = (p.B + SCAN_THREADS - 1) / SCAN_THREADS, b0 = threadIdx.x * each;
  const int b1 = b0 + each < p.B ? b0 + each : p.B, pool = pool_height(p);
  long sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += p.b[b] > 0 ? p.b[b] : 0;
  const long asked0 = block_scan(sum, waves, total);
  sum = 0;
  long asked = asked0;
  for (int b = b0; b < b1; ++b) {
    const Want w = want(p, b, asked);
    asked += w.count;
    sum += w.rows - w.held;
  }
  const long wanted0 = block_scan(sum, waves, total);
  // a request is granted when it wants no page or the pool holds all wanted up to it
  long wanted = wanted0, granted = 0;
  asked = asked0;
  for (int b = b0; b < b1; ++b) {
    const Want w = want(p, b, asked);
    asked += w.count;
    wanted += w.rows - w.held;
    if (w.fits & ((w.rows == w.held) | (wanted <= pool))) granted += w.count;
  }
  long packed = block_scan(granted, waves, total);
  wanted = wanted0;
  asked = asked0;
  long taken = 0;  // pages of this thread's granted requests
  for (int b = b0; b < b1; ++b) {
    const Want w = want(p, b, asked);
    asked += w.count;
    wanted += w.rows - w.held;
    const bool ok = w.fits & ((w.rows == w.held) | (wanted <= pool));
    start[b] = static_cast<int>(packed);
    // page i >= held is entry pool - 1 - (pages wanted before + i - held)
    source[b] = ok ? static_cast<int>(pool - 1 - (wanted - (w.rows - w.held)) + w.held) : 0;
    if (ok) taken += w.rows - w.held;
    if (blockIdx.x == 0) {
      p.cu[b] = static_cast<int>(packed);
      p.lengths_out[b] = p.a[b] + (ok ? static_cast<int>(w.count) : 0);
    }
    if (ok) packed += w.count;
  }
  if (blockIdx.x == 0) {
    long all;
    block_scan(taken, waves, all);
    if (threadIdx.x == 0) {
      p.cu[p.B] = static_cast<int>(total);
      *p.num_free_out = pool - static_cast<int>(all);
    }
  }
  __syncthreads();
  for (long t = blockIdx.x * static_cast<long>(SCAN_THREADS) + threadIdx.x; t < p.tokens;
       t += static_cast<long>(gridDim.x) * SCAN_THREADS) {
    if (t >= total) {
      p.slots[t] = -1;
      p.positions[t] = -1;
      continue;
    }
    const int b = sequence_of(start, p.B, static_cast<int>(t)), len = p.a[b];
    const int pos = len + static_cast<int>(t) - start[b], i = pos / p.page, place = pos - i * p.page;
    int32_t *entry = p.table + b * p.table_row + i;
    const bool fresh = i >= pages_of(len, p.page);
    const int pg = fresh ? p.free_pages[source[b] - i] : *entry;
    if (fresh & (place == 0)) *entry = pg;  // (the first token of a new page is always among these)
    p.slots[t] = pg >= 0 ? static_cast<int64_t>(pg) * p.page + place : -1;
    p.positions[t] = pos;
  }
}

// The entries of all ranges, in the requests' order, are one list, of which each workgroup
// takes a run: it counts the pages before its own and pushes those in it. An entry below 0 is
// no page (the caches' other operators skip it too) and must not come back as one. (64 requests,
// one page each 3.9 us; a request's 16,384 pages 6.6; 256 requests of 1,024 pages 74: a run's
// start costs the reading of all before it, which a serving step, of few pages, does not notice.)
constexpr int RELEASE_THREADS = 512, RELEASE_WAVES = RELEASE_THREADS / 64;
constexpr int RELEASE_BLOCKS = 64;  // most workgroups

__global__ __launch_bounds__(RELEASE_THREADS) void release_kernel(const PoolParams p) {
  constexpr int AT_ONCE = 16;  // entries of a thread in flight
  __shared__ long start[MAX_REQUESTS], table_of[MAX_REQUESTS];  // first entry in the list; entry k is table[table_of + k]
  __shared__ long waves[RELEASE_WAVES], counts[RELEASE_WAVES];
  PBGDN_POISON_LDS(start, sizeof(start));
  PBGDN_POISON_LDS(table_of, sizeof(table_of));
  PBGDN_POISON_SYNC();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int each = (p.B + RELEASE_THREADS - 1) / RELEASE_THREADS, b0 = threadIdx.x * each;
  const int b1 = b0 + each < p.B ? b0 + each : p.B, pool = pool_height(p);
  // pages whose last token lies in [first, end): from first / page up to end / page
  const auto low = [&](int b) { return p.a[b] > 0 ? p.a[b] / p.page : 0; };
  const auto pages = [&](int b) {
    const int hi = p.b[b] > 0 ? p.b[b] / p.page : 0, lo = low(b), top = hi < p.max_pages ? hi : p.max_pages;
    return top > lo ? top - lo : 0;
  };
  long sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += pages(b);
  long at = block_scan(sum, waves, total);
  for (int b = b0; b < b1; ++b) {
    start[b] = at;
    table_of[b] = b * p.table_row + low(b) - at;
    at += pages(b);
  }
  __syncthreads();
  const long even = (total + gridDim.x - 1) / gridDim.x, run = (even + RELEASE_THREADS - 1) / RELEASE_THREADS * RELEASE_THREADS;
  const long k0 = blockIdx.x * run, k1 = k0 + run < total ? k0 + run : total;
  if (blockIdx.x > 0 && k0 >= total) return;
  // Entries k + 64 i of the list below `end` (-1 past it, where the last is read, so that all
  // loads are in flight together). Where a request's have ended it is the next one's, or one that
  // bisection finds.
  int top = 1;
  while (top < p.B) top *= 2;
  int b = -1;  // whose the last entry was, where that request's entries lie and the next one's begin
  long from = 0, next = 0;
  const auto entries = [&](auto &x, long k, long end) __attribute__((always_inline)) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const long at = k + 64 * i < end ? k + 64 * i : end - 1;
      if (at >= next) {
        const auto ends = [&] { return b + 1 < p.B ? start[b + 1] : total; };
        ++b;
        next = ends();
        if (at >= next) {
          b = 0;
          for (int step = top / 2; step > 0; step /= 2)  // the last b with start[b] <= at
            if (b + step < p.B && start[b + step] <= at) b += step;
          next = ends();
        }
        from = table_of[b];
      }
      x[i] = p.table[from + at];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = k + 64 * i < end ? x[i] : -1;
  };
  // pages of the threads before this one, in `all` those of all of them
  const auto ranks = [&](long mine, long &all) __attribute__((always_inline)) {
    __syncthreads();
    if (lane == 0) counts[wave] = mine;
    __syncthreads();
    long before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < RELEASE_WAVES; ++w) {
      if (w < wave) before += counts[w];
      all += counts[w];
    }
    return before;
  };
  long before = 0;
  if (k0 > 0) {
    long mine = 0;
    for (long first = 0; first < k0; first += AT_ONCE * RELEASE_THREADS) {
      int x[AT_ONCE];
      entries(x, first + wave * (64 * AT_ONCE) + lane, k0);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) mine += __popcll(__ballot(x[i] >= 0));
    }
    ranks(mine, before);
  }
  for (long first = k0; first < k1; first += RELEASE_THREADS) {
    int x[1];
    long held;
    entries(x, first + threadIdx.x, k1);
    const uint64_t there = __ballot(x[0] >= 0);
    const long to = pool + before + ranks(__popcll(there), held) + __popcll(there & ((1ull << lane) - 1));
    if (x[0] >= 0 && to < p.capacity) p.free_pages[to] = x[0];  // (past it: more than the pool can have given)
    before += held;
  }
  if (k1 == total && threadIdx.x == 0) *p.num_free_out = static_cast<int>(pool + before < p.capacity ? pool + before : p.capacity);
}

static int pool_params(PoolParams &p, int32_t *table, int64_t table_row, int max_pages, const int32_t *a, const int32_t *b,
                       int B, int page_size, int32_t *free_pages, int capacity, const int32_t *num_free,
                       int32_t *num_free_out) {
  if (B < 0 || max_pages < 0 || page_size <= 0 || capacity < 0 || table_row < 0) return PBGDN_ERR_INVALID_ARGUMENT;
  if (B > MAX_REQUESTS || static_cast<long>(max_pages) * page_size > 0x7fffffffL) return PBGDN_ERR_UNSUPPORTED;
  if (!num_free || !num_free_out || (capacity > 0 && !free_pages) || (B > 0 && (!a || !b)) ||
      (B > 0 && max_pages > 0 && !table)) {
    return PBGDN_ERR_INVALID_ARGUMENT;
  }
  p.table = table;
  p.table_row = table_row;
  p.a = a;
  p.b = b;
  p.free_pages = free_pages;
  p.num_free = num_free;
  p.num_free_out = num_free_out;
  p.B = B;
  p.max_pages = max_pages;
  p.page = page_size;
  p.capacity = capacity;
  return PBGDN_OK;
}

}  // namespace pbgdn

extern "C" int pbattn_pages_extend(int32_t *page_table, int64_t table_row, int max_pages, const int32_t *lengths,
                                   const int32_t *counts, int B, int page_size, const int32_t *free_pages, int capacity,
                                   const int32_t *num_free, int tokens, int64_t *slots, int32_t *positions,
                                   int32_t *cu_seqlens, int32_t *new_lengths, int32_t *new_num_free, void *stream) {
  using namespace pbgdn;
  PoolParams p{};
  const int status = pool_params(p, page_table, table_row, max_pages, lengths, counts, B, page_size,
                                 const_cast<int32_t *>(free_pages), capacity, num_free, new_num_free);
  if (status != PBGDN_OK) return status;
  if (tokens < 0 || !cu_seqlens || (B > 0 && !new_lengths) || (tokens > 0 && (!slots || !positions)))
    return PBGDN_ERR_INVALID_ARGUMENT;
  p.tokens = tokens;
  p.slots = slots;
  p.positions = positions;
  p.cu = cu_seqlens;
  p.lengths_out = new_lengths;
  const int blocks = (tokens + SCAN_THREADS - 1) / SCAN_THREADS;
  hipLaunchKernelGGL(extend_kernel, dim3(blocks < 1 ? 1 : blocks < 1024 ? blocks : 1024), dim3(SCAN_THREADS), 0,
                     static_cast<hipStream_t>(stream), p);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}

extern "C" int pbattn_pages_release(const int32_t *page_table, int64_t table_row, int max_pages, const int32_t *first,
                                    const int32_t *end, int B, int page_size, int32_t *free_pages, int capacity,
                                    const int32_t *num_free, int32_t *new_num_free, void *stream) {
  using namespace pbgdn;
  PoolParams p{};
  const int status = pool_params(p, const_cast<int32_t *>(page_table), table_row, max_pages, first, end, B, page_size,
                                 free_pages, capacity, num_free, new_num_free);
  if (status != PBGDN_OK) return status;
  // as many threads as there are pages to give at most, up to RELEASE_BLOCKS workgroups of them
  const long blocks = (static_cast<long>(B) * max_pages + RELEASE_THREADS - 1) / RELEASE_THREADS;
  hipLaunchKernelGGL(release_kernel, dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks < RELEASE_BLOCKS ? blocks : RELEASE_BLOCKS)),
                     dim3(RELEASE_THREADS), 0, static_cast<hipStream_t>(stream), p);
  return hipGetLastError() == hipSuccess ? PBGDN_OK : PBGDN_ERR_LAUNCH;
}
