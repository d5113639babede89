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
// LDS and the cost is latency: the chain of lengths -> table entries -> slots,
// three dependent round trips to memory (the free pages nearest the top of the
// stack are fetched beside the lengths), and four sums over the workgroup.
// 32 requests of 4096 rows and 245 new tokens: 6.1 us, of which a launch is 2;
// 256 requests, 16-row pages, 9000 new tokens in a pool too small for them:
// 11.8 us, and 3.9 us for a second launch that fills the slots. Release: 3.9 and
// 5.8 us.
#include "common.hpp"

namespace aila {
namespace {

constexpr int kMaxRequests = 2048;   // their prefix sums live in LDS
constexpr int kPlanThreads = 1024;   // of a large batch
constexpr int kPlanWaves = kPlanThreads / 64;
// Slots that the planning workgroup fills itself; more are a second launch's (us,
// 32 requests, itself / second launch: 1024 slots 7.9 / 9.0, 4096 10.5 / 9.1, 16384
// 20.8 / 9.3).
constexpr int kSlotsInPlan = 2048;

// Inclusive sum over the workgroup's threads; `total` gets the sum of all.
template <int NT, typename T>
__device__ __forceinline__ T block_scan(T x, T* s_wave, T* total) {
  constexpr int kWaves = NT / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();   // s_wave of the scan before is read
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  // every wave adds up the waves' sums for itself, lane w those up to wave w
  T y = lane < kWaves ? s_wave[lane] : 0;
#pragma unroll
  for (int off = 1; off < kWaves; off <<= 1) {
    const T z = __shfl_up(y, off);
    if (lane >= off) y += z;
  }
  *total = __shfl(y, kWaves - 1);
  const T before = __shfl(y, max(wave - 1, 0));
  return wave > 0 ? x + before : x;
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

struct Lens { int c, n; bool fits; };
__device__ __forceinline__ Lens load_lens(const int* cached, const int* fresh, int b, long max_rows) {
  Lens l{cached[b], fresh[b], false};
  if (l.c < 0 || l.n < 0) return Lens{0, 0, false};   // absent
  l.fits = static_cast<long>(l.c) + l.n <= max_rows;
  return l;
}

// Entries of the flat list whose pages are kept in LDS, and free pages that are
// fetched before it is known how many are needed.
constexpr int kFlatPages = 4096;

template <int NT>
__global__ __launch_bounds__(NT) void kv_pages_reserve_kernel(
    const int* __restrict__ cached, const int* __restrict__ fresh, int* table, const int* __restrict__ free_pages,
    int* free_count, int* __restrict__ query_start, int* __restrict__ seq_lens, int* __restrict__ slots, int B,
    int max_pages, int page_size, int num_pages, int max_tokens, int fill_slots) {
  extern __shared__ int s_dyn[];
  int* s_start = s_dyn;                 // [B + 1] first token of each request
  int* s_flat = s_start + B + 1;        // [B + 1] first entry of each request's pages
  int* s_first = s_flat + B + 1;        // [B] holes before the request's
  int* s_last = s_first + B;            // [B] holes up to its end
  int* s_rows = s_last + B;             // [B] rows it holds
  int* s_ok = s_rows + B;               // [B] its rows fit the table; then: it is admitted
  __shared__ long s_wl[NT / 64];
  __shared__ int s_wi[NT / 64];
  __shared__ int s_taken;
  __shared__ int s_top[NT];   // the free pages nearest the top
  __shared__ int s_page[kFlatPages];    // page of each entry of the flat list
  const int tid = threadIdx.x;
  const long max_rows = static_cast<long>(max_pages) * page_size;
  const int have = min(max(*free_count, 0), num_pages);
  s_top[tid] = tid < have ? free_pages[have - 1 - tid] : -1;

  // ---- tokens and table entries of each request ---------------------------
  long tok0 = 0;
  int flat0 = 0;
  for (int b0 = 0; b0 < B; b0 += NT) {
    const int b = b0 + tid;
    Lens l{0, 0, false};
    if (b < B) l = load_lens(cached, fresh, b, max_rows);
    const int np = l.fits ? static_cast<int>((static_cast<long>(l.c) + l.n + page_size - 1) / page_size) - l.c / page_size : 0;
    long all_tok;
    int all_np;
    const long tok = tok0 + block_scan<NT, long>(l.n, s_wl, &all_tok);
    const int flat = flat0 + block_scan<NT, int>(np, s_wi, &all_np);
    if (b < B) {
      s_start[b + 1] = static_cast<int>(min(tok, 0x7fffffffL));
      s_flat[b + 1] = flat;
      s_first[b] = s_last[b] = 0;
      s_rows[b] = l.c;
      s_ok[b] = l.fits;
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
  for (int b = tid; b <= B; b += NT) query_start[b] = s_start[b];

  // ---- holes among the entries, in order of request and page --------------
  auto entry_of = [&](int f, int* b) __attribute__((always_inline)) {
    *b = find_request(s_flat, B, f);
    return table + static_cast<size_t>(*b) * max_pages + s_rows[*b] / page_size + f - s_flat[*b];
  };
  const bool in_lds = flat0 <= kFlatPages;
  int holes0 = 0;
  for (int f0 = 0; f0 < flat0; f0 += NT) {
    const int f = f0 + tid;
    int b = 0, page = 0;
    if (f < flat0) {
      page = *entry_of(f, &b);
      if (in_lds) s_page[f] = page;
    }
    const int hole = page < 0;
    int all;
    const int incl = holes0 + block_scan<NT, int>(hole, s_wi, &all);
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
  for (int b = tid; b < B; b += NT) {
    const int ok = s_ok[b] && s_start[b + 1] <= max_tokens && (s_last[b] == s_first[b] || s_last[b] <= have);
    s_ok[b] = ok;
    seq_lens[b] = ok ? s_rows[b] + (s_start[b + 1] - s_start[b]) : 0;
    if (ok && s_last[b] != s_first[b]) atomicMax(&s_taken, s_last[b]);
  }
  __syncthreads();
  int carry = 0;
  for (int f0 = 0; f0 < flat0; f0 += NT) {
    const int f = f0 + tid;
    int b = 0, hole = 0, *entry = nullptr;
    if (f < flat0) {
      entry = entry_of(f, &b);
      hole = (in_lds ? s_page[f] : *entry) < 0;
    }
    int all;
    const int k = carry + block_scan<NT, int>(hole, s_wi, &all) - 1;
    if (hole && s_ok[b]) {
      const int page = k < NT ? s_top[k] : free_pages[have - 1 - k];
      *entry = page;
      if (in_lds) s_page[f] = page;
    }
    carry += all;
  }
  __syncthreads();   // the new pages, for this workgroup
  if (tid == 0) *free_count = have - s_taken;

  // ---- slots ---------------------------------------------------------------
  if (!fill_slots) return;
  for (int t = tid; t < max_tokens; t += NT) {
    int slot = -1;
    if (t < total) {
      const int b = find_request(s_start, B, t);
      if (s_ok[b]) {
        const int row = s_rows[b] + t - s_start[b], p = row / page_size;
        const int page = in_lds ? s_page[s_flat[b] + p - s_rows[b] / page_size] : table[static_cast<size_t>(b) * max_pages + p];
        if (page >= 0 && page < num_pages) slot = page * page_size + row - p * page_size;
      }
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
  for (long t = static_cast<long>(q0) + t0; t < q1; t += step) {
    int slot = -1;
    if (ok) {
      const int row = c + static_cast<int>(t - q0), p = row / page_size;
      const int page = table[static_cast<size_t>(b) * max_pages + p];
      if (page >= 0 && page < num_pages) slot = page * page_size + row - p * page_size;
    }
    slots[t] = slot;
  }
}

// Entries of flagged rows go onto the stack in order of request and page. The
// flagged rows are listed; a wave counts a row's entries, 512 at a time, the
// counts are summed, and a wave then writes its row's entries behind those of
// the rows before. Up to 16 rows of up to 512 entries are read once.
constexpr int kRowChunk = 8;    // entries of a lane

__global__ __launch_bounds__(kPlanThreads) void kv_pages_release_kernel(const int* __restrict__ release, int* table,
                                                                        int* free_pages, int* free_count, int B,
                                                                        int max_pages, int num_pages) {
  extern __shared__ int s_dyn[];
  int* s_row = s_dyn;          // [B] the flagged rows
  int* s_at = s_row + B;       // [B + 1] entries of those before
  __shared__ int s_wi[kPlanWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int have = min(max(*free_count, 0), num_pages);
  int rows = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    const int flag = b < B && release[b] != 0;
    int all;
    const int incl = rows + block_scan<kPlanThreads, int>(flag, s_wi, &all);
    if (flag) s_row[incl - 1] = b;
    rows += all;
  }
  if (tid == 0) s_at[0] = 0;
  __syncthreads();
  int v[kRowChunk];
  auto read = [&](const int* row, int p0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kRowChunk; ++i) {
      const int p = p0 + 64 * i + lane;
      v[i] = p < max_pages ? row[p] : -1;
    }
  };
  auto row_of = [&](int k) __attribute__((always_inline)) { return table + static_cast<size_t>(s_row[k]) * max_pages; };
  for (int k = wave; k < rows; k += kPlanWaves) {
    int n = 0;
    for (int p0 = 0; p0 < max_pages; p0 += 64 * kRowChunk) {
      read(row_of(k), p0);
#pragma unroll
      for (int i = 0; i < kRowChunk; ++i) n += __popcll(__ballot(v[i] >= 0));
    }
    if (lane == 0) s_at[k + 1] = n;
  }
  __syncthreads();
  int sum = 0;
  for (int k0 = 0; k0 < rows; k0 += kPlanThreads) {
    const int k = k0 + tid;
    const int n = k < rows ? s_at[k + 1] : 0;
    int all;
    const int incl = sum + block_scan<kPlanThreads, int>(n, s_wi, &all);
    if (k < rows) s_at[k + 1] = incl;
    sum += all;
  }
  __syncthreads();
  const bool once = rows <= kPlanWaves && max_pages <= 64 * kRowChunk;
  for (int k = wave; k < rows; k += kPlanWaves) {
    if (s_at[k + 1] == s_at[k]) continue;
    int at = have + s_at[k];
    int* row = row_of(k);
    for (int p0 = 0; p0 < max_pages; p0 += 64 * kRowChunk) {
      if (!once) read(row, p0);
#pragma unroll
      for (int i = 0; i < kRowChunk; ++i) {
        const unsigned long long held = __ballot(v[i] >= 0);
        if (v[i] >= 0) {
          const int j = at + __popcll(held & ((1ull << lane) - 1));
          if (j < num_pages) free_pages[j] = v[i];
          row[p0 + 64 * i + lane] = -1;
        }
        at += __popcll(held);
      }
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
  const size_t lds = static_cast<size_t>(6 * B + 2) * sizeof(int);
  auto plan = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(1), dim3(threads), lds, st, cached_lens, new_lens, block_table, free_pages, free_count,
                       query_start, seq_lens, slots, B, max_pages, page_size, num_pages, max_tokens, in_plan ? 1 : 0);
  };
  // Few requests and slots: 4 waves, whose sums and barriers are shorter (us, 256 /
  // 1024 threads: 32 requests, 32 slots 6.3 / 7.8, 512 6.9 / 7.8, 2048 10.6 / 8.8; 256
  // requests, 512 slots 7.8 / 8.6, 1024 9.4 / 8.7; 512 of one 12.0 / 9.1).
  if (B <= 256 && max_tokens <= 512) plan(kv_pages_reserve_kernel<256>, 256);
  else plan(kv_pages_reserve_kernel<kPlanThreads>, kPlanThreads);
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
  hipLaunchKernelGGL(kv_pages_release_kernel, dim3(1), dim3(kPlanThreads), static_cast<size_t>(2 * B + 1) * sizeof(int),
                     static_cast<hipStream_t>(stream), release, block_table, free_pages, free_count, B, max_pages,
                     num_pages);
  return check_launch("kv_pages_release");
}
