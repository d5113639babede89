// Rows of the 8-bit paged KV cache moved inside it, in all layers at once: the
// accepted rows of a draft to its front, and a request's rows to the pages of its
// forks. Codes are moved as they are, or times a power of two where the block
// that they come to has a larger scale (exact but for underflow): nothing is
// quantised again from a rounded value.
#include "paged_fp8.hpp"

#include <algorithm>
#include <type_traits>

namespace aila {
namespace {

constexpr int kMaxLayers = 64;    // of a launch: their pointers are kernel arguments
struct Layers {
  uint8_t* pages[2 * kMaxLayers];   // K and V of layer 0, of layer 1, ...
  float* scale[2 * kMaxLayers];
};

__device__ __forceinline__ uint32_t scale_codes(uint32_t w, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  const int x = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, x, true));
}

struct KeepArgs {
  const int* table;
  const int* cached;
  const int* kept;        // [B, most]
  const int* kept_lens;
  int* lens;              // null: written by another launch
  int B, most, max_pages, num_pages, Hkv, page_size;
};

// A wave: K or V of kHeads heads of one request and layer, their loads in flight
// together; the request's lengths and places are looked up once. Blocks from the one
// of the first row that moves, in order: a row comes from behind its place (kept
// indices rise), so a block that has been written holds no later block's source.
//
// A few requests are bound by the chain lengths -> kept -> table -> scales and codes -> rows:
// 8 requests, 8 layers of 4 heads, D = 256, 19 moved rows, 4.8 us. Of many, 64 requests, 32
// layers of 8 heads, D = 128, 160 moved rows a layer (21 MB read and written, in runs of 128
// bytes; 4.3 us at a copy's rate), every wave of K or V of a layer goes through that chain
// for itself, and has nothing in flight behind its one batch: 19.6 us in a graph, 26 with the
// cache's rows not in the L2s; waves wait for 71% of their time, the vector ALU (places and
// scales) is busy for 39%.
constexpr int kKeepThreads = 256;
// Workgroups with one head a wave above which a wave takes four. us in a graph, one / four, drafts of
// 26 tokens (60: in parentheses). D = 64, 8 heads: 512 workgroups 5.7/6.7, 1024 6.9/6.7 (7.1/6.7), 2048
// 8.7/7.3 (8.8/7.3), 4096 12.0/9.0, 8192 19.0/12.3. D = 128, 8 heads: 512 5.8/8.4, 1024 7.1/8.5
// (7.2/8.4), 2048 9.3/9.3 (9.4/9.2), 4096 12.5/11.5, 8192 21.0/18.8 (22.4/19.6). D = 256 takes one:
// 4 heads, 1024 7.9/8.3, 2048 10.7/10.4, 4096 15.6/17.2 (16.6/18.9); 16 heads, 2048 10.6/10.8, 4096
// 14.4/14.3 (15.2/14.3), 8192 23.4/25.3, 16384 40.7/38.4 (42.6/42.8).
template <int D> constexpr long kKeepGroups = D == 64 ? 1000 : 2000;
constexpr int kNone = kMinScaleExp - 1;
template <int D, int kHeads>
__global__ __launch_bounds__(kKeepThreads) void kv_keep_paged_fp8_kernel(Layers ly, KeepArgs a) {
  constexpr int LR = D / 16;                // lanes of a row, 16 codes each
  constexpr int RI = 64 / LR;               // rows of an instruction
  constexpr int NI = kScaleRows / RI;       // instructions of a block
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.y;
  const int step = static_cast<int>(gridDim.x) * (kKeepThreads / 64 / 2);            // heads from a wave's to its next
  const int head0 = static_cast<int>(blockIdx.x) * (kKeepThreads / 64 / 2) + (wave >> 1);      // kHeads * step reach the last
  const int cached = a.cached[b];
  const long max_rows = static_cast<long>(a.max_pages) * a.page_size;
  int n = min(max(a.kept_lens[b], 0), a.most);
  const int* kept = a.kept + static_cast<size_t>(b) * a.most;
  const int mine = lane < a.most ? kept[lane] : lane;
  if (cached < 0) n = 0;
  else n = static_cast<int>(min(static_cast<long>(n), max(max_rows - cached, 0L)));
  if (a.lens != nullptr && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) a.lens[b] = cached + n;
  int first = n;      // rows before it stay where they are
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane;
    const unsigned long long off = __ballot(i < n && (i0 == 0 ? mine : kept[i]) != i);
    if (off) {
      first = i0 + __builtin_ctzll(off);
      break;
    }
  }
  if (first == n || head0 >= a.Hkv) return;
  const int arr = 2 * blockIdx.z + (wave & 1);
  uint8_t* pages = ly.pages[arr];
  float* scale = ly.scale[arr];
  const int* row_table = a.table + static_cast<size_t>(b) * a.max_pages;
  const int page_blocks = a.page_size / kScaleRows;
  // block of a row in the pool for head 0, -1: none
  auto block_of = [&](long row) __attribute__((always_inline)) -> int {
    if (row < 0 || row >= max_rows) return -1;
    const int r = static_cast<int>(row), p = r / a.page_size;
    const int page = row_table[p];
    return page >= 0 && page < a.num_pages ? page * a.Hkv * page_blocks + (r - p * a.page_size) / kScaleRows : -1;
  };
  const int rr = lane / LR, c16 = lane % LR * 16;
  const int end = cached + n;
  for (int at = (cached + first) / kScaleRows * kScaleRows; at < end; at += kScaleRows) {
    const int bid0 = block_of(at);
    if (bid0 < 0) continue;
    // where this lane's rows come from: head 0's block, byte in it
    int from[NI], byte[NI];
    bool moves[NI], stays[NI], any = false;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const int j = k * RI + rr, i = at + j - cached;
      stays[k] = i < first;
      moves[k] = !stays[k] && i < n;
      from[k] = bid0;
      byte[k] = j * D + c16;
      if (moves[k]) {
        const int src = kept[i];
        const int sb = src < 0 ? -1 : block_of(static_cast<long>(cached) + src);
        moves[k] = sb >= 0;
        if (sb >= 0) {
          from[k] = sb;
          byte[k] = static_cast<int>((static_cast<long>(cached) + src) % kScaleRows) * D + c16;
        }
      }
      any |= moves[k] || stays[k];
    }
    if (__ballot(any) == 0) continue;     // no row of it is in range
    u32x4 w[kHeads][NI];
    float s_from[kHeads][NI], s_held[kHeads];
#pragma unroll
    for (int x = 0; x < kHeads; ++x) {
      const int off = min(head0 + x * step, a.Hkv - 1) * page_blocks;     // past the last: the last again, not stored
      s_held[x] = scale[bid0 + off];
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        s_from[x][k] = 0.f;
        w[x][k] = u32x4{0u, 0u, 0u, 0u};
        if (moves[k]) {
          s_from[x][k] = scale[from[k] + off];
          w[x][k] = ld16(pages + static_cast<size_t>(from[k] + off) * (kScaleRows * D) + byte[k]);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kHeads; ++x) {
      if (head0 + x * step >= a.Hkv) break;
      const int bid = bid0 + (head0 + x * step) * page_blocks;
      const int held = held_exp(s_held[x]);
      int top = kNone;
#pragma unroll
      for (int k = 0; k < NI; ++k)
        if (moves[k] || stays[k]) top = max(top, stays[k] ? held : held_exp(s_from[x][k]));
      const int e = wave_max(top);
      uint8_t* block = pages + static_cast<size_t>(bid) * (kScaleRows * D);
      if (e != held) {      // the rows that stay change scale too
#pragma unroll
        for (int k = 0; k < NI; ++k)
          if (stays[k]) w[x][k] = ld16(block + byte[k]);
      }
#pragma unroll
      for (int k = 0; k < NI; ++k) {
        if (moves[k] || (stays[k] && e != held)) {
          const int e_from = stays[k] ? held : held_exp(s_from[x][k]);
          if (e != e_from) {
            const float f = pow2f(e_from - e);
#pragma unroll
            for (int y = 0; y < 4; ++y) w[x][k][y] = scale_codes(w[x][k][y], f);
          }
          *reinterpret_cast<u32x4*>(block + (k * RI + rr) * D + c16) = w[x][k];
        }
      }
      if (lane == 0) scale[bid] = pow2f(e);
    }
  }
}

struct CopyArgs {
  const int* table;
  const int* src;
  const int* dst;
  const int* lens;
  int B, max_pages, num_pages, Hkv, page_size, max_len;
  int parts;              // workgroups of a page
};

// One workgroup: a part of a page of one pair, K or V of one layer. A page of all
// heads is contiguous; of the last one the blocks behind the rows are left out.
// Bound by the bytes: 3 copies each of 4001 and 3236 rows, 8 layers, 4 heads of D = 256
// (475 MB with each source read once) 108 us = 4.4 TB/s, where a large copy reaches 4.77;
// 3 of 213 rows, one layer, 4.8 us, which is launch and the chain lengths -> table.
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 32768;     // of a workgroup
template <int D>
__global__ __launch_bounds__(kCopyThreads) void kv_copy_paged_fp8_kernel(Layers ly, CopyArgs a) {
  const int p = static_cast<int>(blockIdx.x) / a.parts, part = static_cast<int>(blockIdx.x) % a.parts;
  const int len = min(a.lens[blockIdx.y], a.max_len);
  const int rows = min(len - p * a.page_size, a.page_size);
  if (rows <= 0) return;
  const int from = a.src[blockIdx.y], to = a.dst[blockIdx.y];
  if (from < 0 || from >= a.B || to < 0 || to >= a.B) return;
  const int sp = a.table[static_cast<size_t>(from) * a.max_pages + p], dp = a.table[static_cast<size_t>(to) * a.max_pages + p];
  if (sp < 0 || sp >= a.num_pages || dp < 0 || dp >= a.num_pages || sp == dp) return;
  const int page_blocks = a.page_size / kScaleRows, blocks = (rows + kScaleRows - 1) / kScaleRows;
  const size_t bytes = static_cast<size_t>(a.Hkv) * a.page_size * D;
  const uint8_t* s = ly.pages[blockIdx.z] + sp * bytes;
  uint8_t* d = ly.pages[blockIdx.z] + dp * bytes;
  const int pieces = static_cast<int>(bytes / 16);      // D of a block
  const int end = min(pieces, (part + 1) * (kCopyBytes / 16));
  for (int i = part * (kCopyBytes / 16) + threadIdx.x; i < end; i += kCopyThreads)
    if (i / D % page_blocks < blocks) *reinterpret_cast<u32x4*>(d + static_cast<size_t>(i) * 16) = ld16(s + static_cast<size_t>(i) * 16);
  if (part == 0) {
    const float* ss = ly.scale[blockIdx.z] + static_cast<size_t>(sp) * a.Hkv * page_blocks;
    float* ds = ly.scale[blockIdx.z] + static_cast<size_t>(dp) * a.Hkv * page_blocks;
    for (int i = threadIdx.x; i < a.Hkv * page_blocks; i += kCopyThreads)
      if (i % page_blocks < blocks) ds[i] = ss[i];
  }
}

// The host's arrays of the layers' pointers, checked; layers [l0, l0 + n) of them.
int check_layers(const char* what, const void* const* k_pages, const void* const* v_pages, const float* const* k_scale,
                 const float* const* v_scale, int layers, int Hkv, int D, int page_size, int num_pages) {
  AILA_REQUIRE(k_pages && v_pages && k_scale && v_scale, "%s: null pointer", what);
  AILA_REQUIRE(layers > 0, "%s: layers=%d must be positive", what, layers);
  for (int l = 0; l < layers; ++l)
    if (int rc = check_paged_fp8(what, k_pages[l], v_pages[l], k_scale[l], v_scale[l], Hkv, D, page_size, num_pages)) return rc;
  return AILA_HIP_OK;
}
Layers some_layers(void* const* k_pages, void* const* v_pages, float* const* k_scale, float* const* v_scale, int l0, int n) {
  Layers ly{};
  for (int l = 0; l < n; ++l) {
    ly.pages[2 * l] = static_cast<uint8_t*>(k_pages[l0 + l]);
    ly.pages[2 * l + 1] = static_cast<uint8_t*>(v_pages[l0 + l]);
    ly.scale[2 * l] = k_scale[l0 + l];
    ly.scale[2 * l + 1] = v_scale[l0 + l];
  }
  return ly;
}

}  // namespace
}  // namespace aila

extern "C" int aila_hip_kv_keep_paged_fp8(void* const* k_pages, void* const* v_pages, float* const* k_scale,
                                          float* const* v_scale, int layers, const int* block_table,
                                          const int* cached_lens, const int* kept, const int* kept_lens, int* lens, int B,
                                          int max_kept, int Hkv, int D, int page_size, int num_pages, int max_pages,
                                          void* stream) {
  using namespace aila;
  AILA_REQUIRE(block_table && cached_lens && kept && kept_lens && lens, "kv_keep_paged_fp8: null pointer");
  if (int rc = check_layers("kv_keep_paged_fp8", k_pages, v_pages, k_scale, v_scale, layers, Hkv, D, page_size, num_pages)) return rc;
  AILA_REQUIRE(B > 0 && B <= 65535, "kv_keep_paged_fp8: B=%d outside [1, 65535]", B);
  AILA_REQUIRE(max_kept > 0 && max_kept <= 65536, "kv_keep_paged_fp8: max_kept=%d outside [1, 65536]", max_kept);
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30), "kv_keep_paged_fp8: bad max_pages=%d",
               max_pages);
  const auto over_lens = [&](const int* x, long count) { return lens < x + count && x < lens + B; };
  AILA_REQUIRE(!over_lens(cached_lens, B) && !over_lens(kept_lens, B) && !over_lens(kept, static_cast<long>(B) * max_kept) &&
                   !over_lens(block_table, static_cast<long>(B) * max_pages),
               "kv_keep_paged_fp8: the lengths going out may not overwrite what comes in");
  bool twice = false;      // rows moved in place, by two waves
  for (int l = 0; l < layers; ++l) {
    twice |= k_pages[l] == v_pages[l];
    for (int m = 0; m < l; ++m)
      twice |= k_pages[l] == k_pages[m] || v_pages[l] == v_pages[m] || k_pages[l] == v_pages[m] || v_pages[l] == k_pages[m];
  }
  AILA_REQUIRE(!twice, "kv_keep_paged_fp8: the same pages twice");
  KeepArgs a{block_table, cached_lens, kept, kept_lens, lens, B, max_kept, max_pages, num_pages, Hkv, page_size};
  const unsigned most_gx = (Hkv + 1) / 2;      // a head a wave
  // fewer than 2^32 threads, the most of a launch
  const long fit = ((1L << 32) - 1) / kKeepThreads / most_gx / B;
  AILA_REQUIRE(fit > 0, "kv_keep_paged_fp8: B=%d requests of %d heads are too many", B, Hkv);
  const int step = static_cast<int>(std::min<long>(kMaxLayers, fit));
  for (int l0 = 0; l0 < layers; l0 += step) {
    const int n = std::min(step, layers - l0);
    const Layers ly = some_layers(k_pages, v_pages, k_scale, v_scale, l0, n);
    auto go = [&](auto kernel, unsigned gx) {
      hipLaunchKernelGGL(kernel, dim3(gx, B, n), dim3(kKeepThreads), 0, static_cast<hipStream_t>(stream), ly, a);
    };
    auto launch = [&](auto d) {
      constexpr int kD = decltype(d)::value;
      if constexpr (kD != 256) {
        if (static_cast<long>(B) * n * most_gx > kKeepGroups<kD>) return go(kv_keep_paged_fp8_kernel<kD, 4>, (most_gx + 3) / 4);
      }
      go(kv_keep_paged_fp8_kernel<kD, 1>, most_gx);
    };
    if (D == 64) launch(std::integral_constant<int, 64>{});
    else if (D == 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 256>{});
    a.lens = nullptr;
  }
  return check_launch("kv_keep_paged_fp8");
}

extern "C" int aila_hip_kv_copy_paged_fp8(void* const* k_pages, void* const* v_pages, float* const* k_scale,
                                          float* const* v_scale, int layers, const int* block_table, const int* src,
                                          const int* dst, const int* lens, int n, int max_len, int B, int Hkv, int D,
                                          int page_size, int num_pages, int max_pages, void* stream) {
  using namespace aila;
  AILA_REQUIRE(block_table && src && dst && lens, "kv_copy_paged_fp8: null pointer");
  if (int rc = check_layers("kv_copy_paged_fp8", k_pages, v_pages, k_scale, v_scale, layers, Hkv, D, page_size, num_pages)) return rc;
  AILA_REQUIRE(B > 0 && n > 0 && n <= 65535, "kv_copy_paged_fp8: bad B=%d or n=%d pairs (at most 65535)", B, n);
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30), "kv_copy_paged_fp8: bad max_pages=%d",
               max_pages);
  AILA_REQUIRE(max_len >= 0 && max_len <= max_pages * page_size, "kv_copy_paged_fp8: max_len=%d outside [0, %d]", max_len,
               max_pages * page_size);
  const long bytes = static_cast<long>(Hkv) * page_size * D;
  AILA_REQUIRE(bytes < (1L << 31), "kv_copy_paged_fp8: a page of %ld bytes is too large", bytes);
  if (max_len == 0) return AILA_HIP_OK;
  CopyArgs a{block_table, src, dst, lens, B, max_pages, num_pages, Hkv, page_size, max_len,
             static_cast<int>((bytes + kCopyBytes - 1) / kCopyBytes)};
  const long gx = static_cast<long>((max_len + page_size - 1) / page_size) * a.parts;
  const long fit = ((1L << 32) - 1) / kCopyThreads / gx / n / 2;
  AILA_REQUIRE(fit > 0, "kv_copy_paged_fp8: %d pairs of up to %d rows are too many", n, max_len);
  const int step = static_cast<int>(std::min<long>(kMaxLayers, fit));
  for (int l0 = 0; l0 < layers; l0 += step) {
    const int m = std::min(step, layers - l0);
    const Layers ly = some_layers(k_pages, v_pages, k_scale, v_scale, l0, m);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(gx), n, 2 * m), dim3(kCopyThreads), 0,
                         static_cast<hipStream_t>(stream), ly, a);
    };
    if (D == 64) go(kv_copy_paged_fp8_kernel<64>);
    else if (D == 128) go(kv_copy_paged_fp8_kernel<128>);
    else go(kv_copy_paged_fp8_kernel<256>);
  }
  return check_launch("kv_copy_paged_fp8");
}
