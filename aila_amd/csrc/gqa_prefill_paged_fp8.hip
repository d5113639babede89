// Causal GQA attention of a ragged batch over the 8-bit paged cache (gfx950).
//
//   o_i = sum_j softmax_j(q_i . K_j / sqrt(D)) V_j over the rows j <= L - n + i
//
// for the n tokens of each request. The query rows of a KV head are (token,
// head) pairs, token-major: all query heads that read a KV head share its rows,
// and a tile of 16 rows holds several tokens of a group.
//
// A wave owns 16 query rows (the columns of the matrix instructions) and walks
// the rows of the cache that the last of them attends, in strips of 32, as the
// decode kernel does.
#include "paged_fp8.hpp"

#include <algorithm>

namespace aila {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxSequences = 4096;

struct Fp8PrefillArgs {
  const bf16* q;
  long q_stride;
  bf16* out;
  const int* query_start;
  const int* seq_lens;
  int T, B, Hq, group;
  int max_len;
  float scale_log2;
};

// Tile x of 16 query rows: request b's tiles begin at floor(query_start[b] *
// group / 16) + b, a number that every request's tiles fit below the next's.
template <int D>
__global__ __launch_bounds__(kThreads, 2) void gqa_prefill_paged_fp8_kernel(PagedFp8 c, Fp8PrefillArgs a, int tiles) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;
  const int x = tiles - 1 - (static_cast<int>(blockIdx.x) * kWaves + wave);   // late tiles, with more rows, first
  if (x < 0) return;
  const int kvh = blockIdx.y;
  auto first_tile = [&](int b) {
    return static_cast<int>(static_cast<long>(min(max(a.query_start[b], 0), a.T)) * a.group / 16) + b;
  };
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile(mid) <= x) lo = mid; else hi = mid;
  }
  const int b = __builtin_amdgcn_readfirstlane(lo);
  const int q0 = min(max(a.query_start[b], 0), a.T), n = min(max(a.query_start[b + 1], 0), a.T) - q0;
  const int r0 = (x - first_tile(b)) * 16;     // first query row of the tile
  if (r0 < 0 || r0 >= n * a.group) return;
  const int len = min(max(a.seq_lens[b], 0), a.max_len);
  const int row = r0 + m16;
  const int tok = row / a.group, h = kvh * a.group + row % a.group;
  const bool there = tok < n;
  // this column attends rows < lim; the tile's last column the most
  const int lim = there ? max(len - n + tok + 1, 0) : 0;
  const int end = max(len - n + min(n - 1, (r0 + 15) / a.group) + 1, 0);

  bf16x8_t q[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (there)
      w = ld16(a.q + static_cast<size_t>(q0 + tok) * a.q_stride + static_cast<size_t>(h) * D + 64 * (ks >> 1) + 16 * g4 +
               8 * (ks & 1));
    q[ks] = as_bf16x8(w);
  }
  Column<D> col;
  clear_column(col);
  // rows below `full` are attended by every column
  const int full = max(len - n + r0 / a.group + 1, 0);
  const int blk_end = (end + kScaleRows - 1) / kScaleRows;
  const int ns = (end + 31) / 32;
  for (int n0 = 0; n0 < ns; n0 += 32) {
    const BlockRef mine = block_ref(c, b, kvh, 2 * n0 + lane, blk_end);
    const int n1 = min(ns - n0, 32);
    for (int i = 0; i < n1; ++i) {
      const int ba = __builtin_amdgcn_readlane(mine.bid, 2 * i), bb = __builtin_amdgcn_readlane(mine.bid, 2 * i + 1);
      const float ka = readlane_f(mine.ks, 2 * i) * a.scale_log2, kb = readlane_f(mine.ks, 2 * i + 1) * a.scale_log2;
      const float va = readlane_f(mine.vs, 2 * i), vb = readlane_f(mine.vs, 2 * i + 1);
      Strip<D> s;
      load_strip<D, false>(s, c, ba, bb, m16, g4);
      const int at = 32 * (n0 + i);
      strip_step<D>(col, s, q, ka, kb, va, vb, at + 32 > full || r0 + 16 > n * a.group || (ba | bb) < 0, at, lim, ba >= 0,
                    bb >= 0, g4);
    }
  }
  const float l = xrow4_sum(col.l);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (there) {
    bf16* o = a.out + (static_cast<size_t>(q0 + tok) * a.Hq + h) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < D / 16; t += 2)
        *reinterpret_cast<uint32_t*>(o + (D / 16) * (4 * g4 + i) + t) = pack_bf16x2(col.acc[t][i] * inv, col.acc[t + 1][i] * inv);
    }
  }
}

template <int D>
int launch(const PagedFp8& c, const Fp8PrefillArgs& a, hipStream_t st) {
  const int tiles = static_cast<int>(static_cast<long>(a.T) * a.group / 16) + a.B;
  hipLaunchKernelGGL((gqa_prefill_paged_fp8_kernel<D>), dim3((tiles + kWaves - 1) / kWaves, c.Hkv), dim3(kThreads), 0, st,
                     c, a, tiles);
  return check_launch("gqa_prefill_paged_fp8");
}

}  // namespace
}  // namespace aila

extern "C" size_t aila_hip_gqa_prefill_paged_fp8_workspace_size(int T, int B, int Hq, int Hkv, int D, int max_len) {
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || max_len < 0) return 0;
  return 0;
}

extern "C" int aila_hip_gqa_prefill_paged_fp8(const void* q, long q_stride, const void* k_pages, const void* v_pages,
                                              const float* k_scale, const float* v_scale, void* out, void* workspace,
                                              size_t workspace_bytes, int T, int B, int Hq, int Hkv, int D,
                                              int page_size, int num_pages, const int* block_table, int max_pages,
                                              int max_len, const int* query_start, const int* seq_lens, void* stream) {
  using namespace aila;
  (void)workspace;
  (void)workspace_bytes;
  AILA_REQUIRE(q && out && block_table && query_start && seq_lens, "gqa_prefill_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("gqa_prefill_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  AILA_REQUIRE(B > 0 && B <= kMaxSequences, "gqa_prefill_paged_fp8: B=%d outside [1, %d]", B, kMaxSequences);
  AILA_REQUIRE(Hq > 0 && Hq % Hkv == 0 && Hq <= 65535, "gqa_prefill_paged_fp8: bad heads (Hq=%d Hkv=%d)", Hq, Hkv);
  AILA_REQUIRE(T > 0 && static_cast<long>(T) * (Hq / Hkv) <= (1L << 30), "gqa_prefill_paged_fp8: T=%d tokens are too many", T);
  AILA_REQUIRE(q_stride >= static_cast<long>(Hq) * D && q_stride % 8 == 0,
               "gqa_prefill_paged_fp8: query stride %ld must be a multiple of 8 and hold Hq * D = %ld values", q_stride,
               static_cast<long>(Hq) * D);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
               "gqa_prefill_paged_fp8: q and out must be 16-byte aligned");
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30),
               "gqa_prefill_paged_fp8: bad max_pages=%d", max_pages);
  AILA_REQUIRE(max_len >= 0 && max_len <= max_pages * page_size, "gqa_prefill_paged_fp8: max_len=%d outside [0, %d]",
               max_len, max_pages * page_size);
  PagedFp8 c{static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), k_scale, v_scale,
             block_table, max_pages, num_pages, Hkv, page_size / kScaleRows};
  Fp8PrefillArgs a{};
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<bf16*>(out);
  a.query_start = query_start;
  a.seq_lens = seq_lens;
  a.T = T; a.B = B; a.Hq = Hq; a.group = Hq / Hkv;
  a.max_len = max_len;
  a.scale_log2 = kLog2e / sqrtf(static_cast<float>(D));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (D) {
    case 64: return launch<64>(c, a, st);
    case 128: return launch<128>(c, a, st);
    default: return launch<256>(c, a, st);
  }
}
