// Page tables of the paged KV cache, kept on the device: pages are taken from
// and given back to a stack of free pages, and each new token gets its slot
// (page * page_size + row in page), from the requests' lengths alone, so a
// serving step needs no host copy of any table and can be captured in a graph.
//
// The reference has one contiguous cache per sequence (src/memory/KVCache.hpp:
// 9-45) and a host-side cursor; this is the bookkeeping of the paged layout of
// aila_hip_gqa_decode_paged.
//
// Reserve is three prefix sums: of the new tokens (where a request's tokens
// start), of the pages that the new rows touch (the flat list of table entries
// to look at), and of the holes among those entries (which free page a hole
// takes). A few hundred requests are a few KiB, so one workgroup does it all in
// LDS and the cost is latency: the chain of lengths -> table entries -> free
// pages -> slots, four dependent round trips to memory.
#include "common.hpp"

namespace aila {
namespace {

constexpr int kMaxRequests = 2048;   // their prefix sums live in LDS
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Slots that the planning workgroup fills itself; more are a second launch's.
constexpr int kSlotsInPlan = 8192;

// Inclusive sum over the workgroup's threads; `total` gets the sum of all.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* s_wave, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();   // s_wave of the scan before is read
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    const T v = s_wave[w];
    if (w < wave) before += v;
    all += v;
  }
  *total = all;
  return x + before;
}

// The last b with start[b] <= x, for start[0] = 0 <= x < start[n] (entries of
// equal value are requests without elements: the last of them is taken).
__device__ __forceinline__ int find_request(const int* start, int n, int x) {
  int lo = 0, hi = n;   // start[lo] <= x < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

struct Lens { long c, n; bool fits; };
__device__ __forceinline__ Lens load_lens(const int* cached, const int* fresh, int b, long max_rows) {
  Lens l{cached[b], fresh[b], false};
  if (l.c < 0 || l.n < 0) return Lens{0, 0, false};   // absent
  l.fits = l.c + l.n <= max_rows;
  return l;
}

__device__ __forceinline__ int slot_of(const int* table, int max_pages, int page_size, int num_pages, int b, int row) {
  const int page = table[static_cast<size_t>(b) * max_pages + row / page_size];
  return page >= 0 && page < num_pages ? page * page_size + row % page_size : -1;
}

__global__ __launch_bounds__(kPlanThreads) void kv_pages_reserve_kernel(
    const int* __restrict__ cached, const int* __restrict__ fresh, int* table, const int* __restrict__ free_pages,
    int* free_count, int* __restrict__ query_start, int* __restrict__ seq_lens, int* __restrict__ slots, int B,
    int max_pages, int page_size, int num_pages, int max_tokens, int fill_slots) {
  extern __shared__ int s_dyn[];
  int* s_start = s_dyn;                 // [B + 1] first token of each request
  int* s_flat = s_start + B + 1;        // [B + 1] first entry of each request's pages
  int* s_first = s_flat + B + 1;        // [B] holes before the request's
  int* s_last = s_first + B;            // [B] holes up to its end
  __shared__ long s_wl[kPlanWaves];
  __shared__ int s_wi[kPlanWaves];
  __shared__ int s_taken;
  const int tid = threadIdx.x;
  const long max_rows = static_cast<long>(max_pages) * page_size;
  const int have = min(max(*free_count, 0), num_pages);

  // ---- tokens and table entries of each request ---------------------------
  long tok0 = 0;
  int flat0 = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    Lens l{0, 0, false};
    if (b < B) l = load_lens(cached, fresh, b, max_rows);
    const int np = l.fits ? static_cast<int>((l.c + l.n + page_size - 1) / page_size - l.c / page_size) : 0;
    long all_tok;
    int all_np;
    const long tok = tok0 + block_scan<long>(l.n, s_wl, &all_tok);
    const int flat = flat0 + block_scan<int>(np, s_wi, &all_np);
    if (b < B) {
      s_start[b + 1] = static_cast<int>(min(tok, 0x7fffffffL));
      s_flat[b + 1] = flat;
      s_first[b] = s_last[b] = 0;
    }
    tok0 += all_tok;
    flat0 += all_np;
  }
  if (tid == 0) {
    s_start[0] = s_flat[0] = 0;
    s_taken = 0;
  }
  __syncthreads();
  const int total = s_start[B];
  for (int b = tid; b <= B; b += kPlanThreads) query_start[b] = s_start[b];

  // ---- holes among the entries, in order of request and page --------------
  int holes0 = 0;
  for (int f0 = 0; f0 < flat0; f0 += kPlanThreads) {
    const int f = f0 + tid;
    int b = 0, hole = 0;
    if (f < flat0) {
      b = find_request(s_flat, B, f);
      const int p = cached[b] / page_size + f - s_flat[b];
      hole = table[static_cast<size_t>(b) * max_pages + p] < 0;
    }
    int all;
    const int incl = holes0 + block_scan<int>(hole, s_wi, &all);
    if (f < flat0) {
      if (f == s_flat[b]) s_first[b] = incl - hole;
      if (f + 1 == s_flat[b + 1]) s_last[b] = incl;
    }
    holes0 += all;
  }
  __syncthreads();

  // Admitted: its rows fit the table, its tokens the batch, its holes the pool.
  // Both sums only grow, so the admitted requests that take pages come first
  // among those that need any, and the k-th hole takes the k-th page from the top.
  auto admitted = [&](int b, bool fits) __attribute__((always_inline)) {
    return fits && s_start[b + 1] <= max_tokens && (s_last[b] == s_first[b] || s_last[b] <= have);
  };
  int carry = 0;
  for (int f0 = 0; f0 < flat0; f0 += kPlanThreads) {
    const int f = f0 + tid;
    int b = 0, hole = 0, *entry = nullptr;
    if (f < flat0) {
      b = find_request(s_flat, B, f);
      entry = table + static_cast<size_t>(b) * max_pages + cached[b] / page_size + f - s_flat[b];
      hole = *entry < 0;
    }
    int all;
    const int k = carry + block_scan<int>(hole, s_wi, &all) - 1;
    if (hole && admitted(b, true)) {   // only requests that fit have entries here
      *entry = free_pages[have - 1 - k];
      if (k + 1 == s_last[b]) atomicMax(&s_taken, k + 1);
    }
    carry += all;
  }
  for (int b = tid; b < B; b += kPlanThreads) {
    const Lens l = load_lens(cached, fresh, b, max_rows);
    const bool ok = admitted(b, l.fits);
    seq_lens[b] = ok ? static_cast<int>(l.c + l.n) : 0;
  }
  __syncthreads();   // the table's new entries, for this workgroup
  if (tid == 0) *free_count = have - s_taken;

  // ---- slots ---------------------------------------------------------------
  if (!fill_slots) return;
  for (int t = tid; t < max_tokens; t += kPlanThreads) {
    int slot = -1;
    if (t < total) {
      const int b = find_request(s_start, B, t);
      const Lens l = load_lens(cached, fresh, b, max_rows);
      if (admitted(b, l.fits))
        slot = slot_of(table, max_pages, page_size, num_pages, b, static_cast<int>(l.c) + t - s_start[b]);
    }
    slots[t] = slot;
  }
}

// Slots of one request's tokens (grid.x = B), or of the batch's tail (the last one).
__global__ __launch_bounds__(256) void kv_pages_slots_kernel(const int* __restrict__ cached, const int* __restrict__ table,
                                                             const int* __restrict__ query_start,
                                                             const int* __restrict__ seq_lens, int* __restrict__ slots,
                                                             int B, int max_pages, int page_size, int num_pages,
                                                             int max_tokens) {
  const int b = blockIdx.x;
  const int step = 256 * static_cast<int>(gridDim.y), t0 = blockIdx.y * 256 + threadIdx.x;
  if (b == B) {
    for (long t = static_cast<long>(query_start[B]) + t0; t < max_tokens; t += step) slots[t] = -1;
    return;
  }
  const int q0 = query_start[b], q1 = min(query_start[b + 1], max_tokens);
  const int c = cached[b];
  // an admitted request of new tokens has rows; a refused one's length is 0
  const bool ok = seq_lens[b] > 0;
  for (long t = static_cast<long>(q0) + t0; t < q1; t += step)
    slots[t] = ok ? slot_of(table, max_pages, page_size, num_pages, b, c + static_cast<int>(t - q0)) : -1;
}

// Entries of flagged rows go onto the stack in order of request and page. A
// wave counts a row's entries; the rows' counts are summed; a wave then writes
// its row's entries behind those of the rows before.
__global__ __launch_bounds__(kPlanThreads) void kv_pages_release_kernel(const int* __restrict__ release, int* table,
                                                                        int* free_pages, int* free_count, int B,
                                                                        int max_pages, int num_pages) {
  extern __shared__ int s_dyn[];
  int* s_at = s_dyn;   // [B + 1]
  __shared__ int s_wi[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int have = min(max(*free_count, 0), num_pages);
  for (int b = wave; b < B; b += kPlanWaves) {
    int n = 0;
    if (release[b] != 0)
      for (int p = lane; p < max_pages; p += 64) n += table[static_cast<size_t>(b) * max_pages + p] >= 0;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) n += __shfl_xor(n, off);
    if (lane == 0) s_at[b + 1] = n;
  }
  if (tid == 0) s_at[0] = 0;
  __syncthreads();
  int sum = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int n = b < B ? s_at[b + 1] : 0;
    int all;
    const int incl = sum + block_scan<int>(n, s_wi, &all);
    if (b < B) s_at[b + 1] = incl;
    sum += all;
  }
  __syncthreads();
  for (int b = wave; b < B; b += kPlanWaves) {
    if (s_at[b + 1] == s_at[b]) continue;
    int at = have + s_at[b];
    for (int p0 = 0; p0 < max_pages; p0 += 64) {
      const int p = p0 + lane;
      int* entry = table + static_cast<size_t>(b) * max_pages + p;
      const int page = p < max_pages ? *entry : -1;
      const unsigned long long held = __ballot(page >= 0);
      if (page >= 0) {
        const int k = at + __popcll(held & ((1ull << lane) - 1));
        if (k < num_pages) free_pages[k] = page;
        *entry = -1;
      }
      at += __popcll(held);
    }
  }
  if (tid == 0) *free_count = min(have + sum, num_pages);
}

}  // namespace
}  // namespace aila

extern "C" int aila_hip_kv_pages_reserve(const int* cached_lens, const int* new_lens, int* block_table,
                                         const int* free_pages, int* free_count, int* query_start, int* seq_lens,
                                         int* slots, int B, int max_pages, int page_size, int num_pages,
                                         int max_tokens, void* stream) {
  using namespace aila;
  AILA_REQUIRE(cached_lens && new_lens && block_table && free_pages && free_count && query_start && seq_lens && slots,
               "kv_pages_reserve: null pointer");
  AILA_REQUIRE(seq_lens != cached_lens && seq_lens != new_lens && query_start != cached_lens && query_start != new_lens,
               "kv_pages_reserve: the lengths going out may not overwrite those coming in");
  AILA_REQUIRE(B > 0 && B <= kMaxRequests, "kv_pages_reserve: B=%d outside [1, %d]", B, kMaxRequests);
  AILA_REQUIRE(page_size > 0 && page_size % 16 == 0, "kv_pages_reserve: page_size=%d must be a positive multiple of 16",
               page_size);
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30),
               "kv_pages_reserve: bad max_pages=%d", max_pages);
  AILA_REQUIRE(static_cast<long>(max_pages) * B < (1L << 31), "kv_pages_reserve: B * max_pages exceeds 2^31");
  AILA_REQUIRE(num_pages > 0 && static_cast<long>(num_pages) * page_size < (1L << 31),
               "kv_pages_reserve: num_pages=%d pages of %d rows: slots must fit 31 bits", num_pages, page_size);
  AILA_REQUIRE(max_tokens > 0, "kv_pages_reserve: max_tokens=%d must be positive", max_tokens);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool in_plan = max_tokens <= kSlotsInPlan;
  const size_t lds = static_cast<size_t>(4 * B + 2) * sizeof(int);
  hipLaunchKernelGGL(kv_pages_reserve_kernel, dim3(1), dim3(kPlanThreads), lds, st, cached_lens, new_lens, block_table,
                     free_pages, free_count, query_start, seq_lens, slots, B, max_pages, page_size, num_pages,
                     max_tokens, in_plan ? 1 : 0);
  if (!in_plan)
    hipLaunchKernelGGL(kv_pages_slots_kernel, dim3(B + 1, 4), dim3(256), 0, st, cached_lens, block_table, query_start,
                       seq_lens, slots, B, max_pages, page_size, num_pages, max_tokens);
  return check_launch("kv_pages_reserve");
}

extern "C" int aila_hip_kv_pages_release(const int* release, int* block_table, int* free_pages, int* free_count, int B,
                                         int max_pages, int num_pages, void* stream) {
  using namespace aila;
  AILA_REQUIRE(release && block_table && free_pages && free_count, "kv_pages_release: null pointer");
  AILA_REQUIRE(B > 0 && B <= kMaxRequests, "kv_pages_release: B=%d outside [1, %d]", B, kMaxRequests);
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * B < (1L << 31), "kv_pages_release: bad max_pages=%d",
               max_pages);
  AILA_REQUIRE(num_pages > 0, "kv_pages_release: num_pages=%d must be positive", num_pages);
  hipLaunchKernelGGL(kv_pages_release_kernel, dim3(1), dim3(kPlanThreads), static_cast<size_t>(B + 1) * sizeof(int),
                     static_cast<hipStream_t>(stream), release, block_table, free_pages, free_count, B, max_pages,
                     num_pages);
  return check_launch("kv_pages_release");
}
