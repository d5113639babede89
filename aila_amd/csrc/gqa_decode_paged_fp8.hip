// Single-token GQA attention over the 8-bit paged cache (gfx950).
//
//   o = sum_j softmax_j(q . K_j / sqrt(D)) V_j  over the rows j < len.
//
// One pass with a running maximum and sum; a workgroup serves all query heads
// of a KV head (up to 16: the columns of the matrix instructions), so each code
// is read from HBM once. Codes go from memory to registers, are converted to
// bf16 there (exact) and feed the matrix cores; nothing passes through LDS but
// the waves' results. Bound by the bytes of K and V: 8 ragged sequences of up to
// 32768 rows (4 KV heads, D = 256) 68 us = 6.1 TB/s and 4.6 us of merge, 64 of up
// to 4001 (8 KV heads of 5 query heads, D = 128) 76 us = 5.3 TB/s; a large copy
// reaches 4.7, a pure read 7.1. One sequence of 32768 rows is 17 us (4.0 TB/s):
// a workgroup's share is 4 units there, and start-up and the end of the waves are
// half of it.
//
// Split: the rows of all sequences and KV heads form one line, in units of 128
// rows (a strip of 32 for each of the 4 waves), and every workgroup takes an
// equal piece of it, whatever the lengths are: a ragged batch keeps every CU
// busy until the end. Whether to split is the host's choice, which knows the
// bound of the lengths alone. A piece that covers a (sequence, head) whole writes its
// output; the others write records {acc[D], m, l}, at most two a workgroup, and
// the merge kernel joins those of each (sequence, head).
#include "paged_fp8.hpp"

#include <algorithm>

namespace aila {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kUnit = 32 * kWaves;     // rows of a unit
constexpr int kMaxTile = 16;           // query heads of a workgroup
constexpr int kMaxSequences = 4096;    // their unit counts live in LDS
constexpr int kRecTail = 4;

struct Fp8DecodeArgs {
  const bf16* q;
  long q_stride;                       // elements between sequences' queries
  bf16* out;
  float* part;                         // records; null: one workgroup per (sequence, head)
  int* units;                          // [B + 1] for the merge: units of the sequences before
  const int* seq_lens;
  int B, Hq, group, tile, chunks;      // query heads per KV head; per workgroup; workgroups per KV head
  int max_len;
  float scale_log2;
};

__device__ __forceinline__ int units_of(const Fp8DecodeArgs& a, int b, int* len) {
  *len = min(max(a.seq_lens[b], 0), a.max_len);
  return max(1, (*len + kUnit - 1) / kUnit);    // an empty sequence's output is written too
}

// s_pre[b] = units of the sequences before b, for b <= B.
__device__ __forceinline__ void scan_units(const Fp8DecodeArgs& a, int* s_pre) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int b = b0 + lane;
      int len, n = b < a.B ? units_of(a, b, &len) : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(n, off);
        if (lane >= off) n += y;
      }
      if (b < a.B) s_pre[b + 1] = sum + n;
      sum += __shfl(n, 63);
    }
    if (lane == 0) s_pre[0] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ int find_sequence(const int* pre, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Workgroup w of W <= U holds units [w U / W, (w + 1) U / W), one at least.
__device__ __forceinline__ int share_begin(int w, int units, int groups) {
  return __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<long>(w) * units / groups));
}

template <int D>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void gqa_decode_paged_fp8_kernel(PagedFp8 c, Fp8DecodeArgs a) {
  // Strips of a wave in registers: one is worked on while the next arrives. (us a
  // call, merge included, in a graph that changes its inputs. Three: 8 ragged
  // sequences of up to 32768, 16/4, D = 256, 75.6 against 73.3; 8 of 8000, 32/8, D =
  // 128, 32.0 against 31.0. Two workgroups a CU at D = 256 instead spill: 109.8.)
  constexpr int kDepth = 2;
  extern __shared__ __attribute__((aligned(16))) unsigned char s_dyn[];
  float* s_acc = reinterpret_cast<float*>(s_dyn);             // [kWaves][tile][D]
  float* s_ml = s_acc + kWaves * a.tile * D;                  // [kWaves][tile][2]
  int* s_pre = reinterpret_cast<int*>(s_ml + kWaves * a.tile * 2);   // [B + 1]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;
  const int heads = c.Hkv * a.chunks;

  int u, u1;
  if (a.part == nullptr) {
    u = blockIdx.x;       // (sequence, head) here
    u1 = u + 1;
  } else {
    scan_units(a, s_pre);
    const int units = s_pre[a.B] * heads, groups = min(static_cast<int>(gridDim.x), units);
    const int w = blockIdx.x;
    if (w == 0)
      for (int i = threadIdx.x; i <= a.B; i += kThreads) a.units[i] = s_pre[i];
    if (w >= groups) return;
    u = share_begin(w, units, groups);
    u1 = share_begin(w + 1, units, groups);
  }
  while (u < u1) {
    int b, hc, i0, i1, nu, len;
    if (a.part == nullptr) {
      b = u / heads;
      hc = u % heads;
      nu = units_of(a, b, &len);
      i0 = 0;
      i1 = nu;
      u = u1;
    } else {
      b = __builtin_amdgcn_readfirstlane(find_sequence(s_pre, a.B, u / heads));
      const int at = __builtin_amdgcn_readfirstlane(u - s_pre[b] * heads);
      nu = units_of(a, b, &len);
      hc = at / nu;
      i0 = at % nu;
      i1 = min(nu, i0 + (u1 - u));
      u += i1 - i0;
    }
    const int kvh = hc / a.chunks, chunk = hc % a.chunks;
    const int h0 = kvh * a.group + chunk * a.tile;
    const int gv = min(a.tile, a.group - chunk * a.tile);

    bf16x8_t q[D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if (m16 < gv)
        w = ld16(a.q + b * a.q_stride + static_cast<size_t>(h0 + m16) * D + 64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1));
      q[ks] = as_bf16x8(w);
    }
    Column<D> col;
    clear_column(col);

    // strips of this wave: row i0 * kUnit + 32 wave + kUnit n, n < ns
    const int row0 = i0 * kUnit + 32 * wave;
    const int end = min(i1 * kUnit, len);
    const int ns = row0 < end ? (end - row0 + kUnit - 1) / kUnit : 0;
    const int blk_end = (end + kScaleRows - 1) / kScaleRows;
    for (int n0 = 0; n0 < ns; n0 += 32) {
      // lane l holds block l % 2 of strip n0 + l / 2
      const BlockRef mine = block_ref(c, b, kvh, row0 / kScaleRows + (n0 + (lane >> 1)) * (kUnit / kScaleRows) + (lane & 1),
                                      blk_end);
      const int n1 = min(ns - n0, 32);
      auto load = [&](Strip<D>& s, int n) __attribute__((always_inline)) {
        const bool in = n < n1;
        const int ba = __builtin_amdgcn_readlane(mine.bid, 2 * n & 63), bb = __builtin_amdgcn_readlane(mine.bid, (2 * n + 1) & 63);
        load_strip<D, true>(s, c, in ? ba : -1, in ? bb : -1, m16, g4);
      };
      auto step = [&](Strip<D>& s, int n) __attribute__((always_inline)) {
        const int ba = __builtin_amdgcn_readlane(mine.bid, 2 * n), bb = __builtin_amdgcn_readlane(mine.bid, 2 * n + 1);
        const float ka = readlane_f(mine.ks, 2 * n) * a.scale_log2, kb = readlane_f(mine.ks, 2 * n + 1) * a.scale_log2;
        const float va = readlane_f(mine.vs, 2 * n), vb = readlane_f(mine.vs, 2 * n + 1);
        const int row = row0 + (n0 + n) * kUnit;
        strip_step<D>(col, s, q, ka, kb, va, vb, row + 32 > end || (ba | bb) < 0, row, end, ba >= 0, bb >= 0, g4);
      };
      Strip<D> s[kDepth];
#pragma unroll
      for (int i = 0; i < kDepth - 1; ++i) load(s[i], i);
      for (int n = 0; n < n1; n += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
          if (n + i < n1) {
            load(s[(i + kDepth - 1) % kDepth], n + i + kDepth - 1);
            step(s[i], n + i);
          }
        }
      }
    }

    // ---- the waves' results meet ------------------------------------------
    const float l = xrow4_sum(col.l);
    __syncthreads();   // the segment before has been read
    if (m16 < gv) {
      float* row = s_acc + (wave * a.tile + m16) * D;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) row[(D / 16) * (4 * g4 + i) + t] = col.acc[t][i];
      }
      if (g4 == 0) {
        s_ml[(wave * a.tile + m16) * 2] = col.m;
        s_ml[(wave * a.tile + m16) * 2 + 1] = l;
      }
    }
    __syncthreads();
    const bool whole = i0 == 0 && i1 == nu;
    float* rec = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (i0 == 0 ? 1 : 0)) * a.tile * (D + kRecTail);
    for (int idx = threadIdx.x; idx < gv * D; idx += kThreads) {
      const int h = idx / D, d = idx % D;
      float M = -INFINITY, A = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_ml[(w * a.tile + h) * 2]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float mw = s_ml[(w * a.tile + h) * 2];
        const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
        A += f * s_acc[(w * a.tile + h) * D + d];
        L += f * s_ml[(w * a.tile + h) * 2 + 1];
      }
      if (whole) {
        a.out[(static_cast<size_t>(b) * a.Hq + h0 + h) * D + d] = f2bf(L == 0.f ? 0.f : A / L);
      } else {
        rec[h * (D + kRecTail) + d] = A;
        if (d == 0) {
          rec[h * (D + kRecTail) + D] = M;
          rec[h * (D + kRecTail) + D + 1] = L;
        }
      }
    }
  }
}

// The workgroups [w0, w1] that walked a (sequence, head).
__device__ __forceinline__ void holders(const PagedFp8& c, const Fp8DecodeArgs& a, int b, int hc, int launched, int* w0, int* w1) {
  const int heads = c.Hkv * a.chunks, before = a.units[b], nu = a.units[b + 1] - before;
  const int units = a.units[a.B] * heads, groups = min(launched, units);
  const int first = before * heads + hc * nu;
  // workgroup w holds unit x: the largest w with w U / W < x + 1
  *w0 = static_cast<int>((static_cast<long>(first + 1) * groups - 1) / units);
  *w1 = static_cast<int>((static_cast<long>(first + nu) * groups - 1) / units);
}

// Joins the records of a (sequence, head) that several workgroups walked:
// o = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i. Few sequences, many
// records each: a workgroup takes a query head's 64 dims, 16 columns of 4 dims
// and 16 record phases.
template <int D>
__global__ __launch_bounds__(256) void gqa_decode_paged_fp8_merge_kernel(PagedFp8 c, Fp8DecodeArgs a, int launched) {
  __shared__ f32x4 s_a[16][16];
  __shared__ float s_m[16], s_l[16];
  const int b = blockIdx.y, hq = blockIdx.x;
  const int kvh = hq / a.group, in = hq % a.group;
  const int hc = kvh * a.chunks + in / a.tile, h = in % a.tile;
  int w0, w1;
  holders(c, a, b, hc, launched, &w0, &w1);
  if (w0 == w1) return;   // one workgroup wrote the output
  const int col = threadIdx.x & 15, ph = threadIdx.x >> 4;
  const int d = blockIdx.z * 64 + 4 * col;
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  for (int w = w0 + ph; w <= w1; w += 16) {
    const float* r = a.part + ((static_cast<size_t>(w) * 2 + (w == w0 ? 1 : 0)) * a.tile + h) * (D + kRecTail);
    const f32x4 x = *reinterpret_cast<const f32x4*>(r + d);
    const float m = r[D], l = r[D + 1];
    const float mn = fmaxf(M, m);
    const float fo = M == -INFINITY ? 0.f : fast_exp2(M - mn), fn = m == -INFINITY ? 0.f : fast_exp2(m - mn);
    A = A * fo + x * fn;
    L = L * fo + l * fn;
    M = mn;
  }
  s_a[ph][col] = A;
  if (col == 0) {
    s_m[ph] = M;
    s_l[ph] = L;
  }
  __syncthreads();
  if (threadIdx.x < 16) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, s_m[i]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float f = s_m[i] == -INFINITY ? 0.f : fast_exp2(s_m[i] - top);
      o += f * s_a[i][threadIdx.x];
      sum += f * s_l[i];
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    o *= inv;
    *reinterpret_cast<u32x2*>(a.out + (static_cast<size_t>(b) * a.Hq + hq) * D + blockIdx.z * 64 + 4 * threadIdx.x) =
        u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
  }
}

// The same for many sequences, few records each: a workgroup takes a
// (sequence, head), a thread 4 dims of a query head.
template <int D>
__global__ __launch_bounds__(256) void gqa_decode_paged_fp8_merge_few_kernel(PagedFp8 c, Fp8DecodeArgs a, int launched) {
  const int b = blockIdx.y, hc = blockIdx.x;
  int w0, w1;
  holders(c, a, b, hc, launched, &w0, &w1);
  if (w0 == w1) return;
  const int kvh = hc / a.chunks, chunk = hc % a.chunks;
  const int gv = min(a.tile, a.group - chunk * a.tile);
  for (int i = threadIdx.x; i < gv * (D / 4); i += 256) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    f32x4 A = {0.f, 0.f, 0.f, 0.f};
    float M = -INFINITY, L = 0.f;
    for (int w = w0; w <= w1; ++w) {
      const float* r = a.part + ((static_cast<size_t>(w) * 2 + (w == w0 ? 1 : 0)) * a.tile + h) * (D + kRecTail);
      const f32x4 x = *reinterpret_cast<const f32x4*>(r + d);
      const float m = r[D], l = r[D + 1];
      const float mn = fmaxf(M, m);
      const float fo = M == -INFINITY ? 0.f : fast_exp2(M - mn), fn = m == -INFINITY ? 0.f : fast_exp2(m - mn);
      A = A * fo + x * fn;
      L = L * fo + l * fn;
      M = mn;
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    *reinterpret_cast<u32x2*>(a.out + (static_cast<size_t>(b) * a.Hq + kvh * a.group + chunk * a.tile + h) * D + d) =
        u32x2{pack_bf16x2(A[0] * inv, A[1] * inv), pack_bf16x2(A[2] * inv, A[3] * inv)};
  }
}

// Query heads of a workgroup and workgroups per KV head.
void head_tiles(int group, int* tile, int* chunks) {
  *chunks = (group + kMaxTile - 1) / kMaxTile;
  *tile = (group + *chunks - 1) / *chunks;
}

size_t record_bytes(int tile, int D) { return static_cast<size_t>(2) * tile * (D + kRecTail) * sizeof(float); }
// The unit counts stand before the records.
size_t units_bytes(int B) { return (static_cast<size_t>(B + 1) * sizeof(int) + 255) / 256 * 256; }

template <int D>
int launch(const PagedFp8& c, const Fp8DecodeArgs& a, int groups, hipStream_t st) {
  const size_t lds = (static_cast<size_t>(kWaves) * a.tile * (D + 2)) * sizeof(float) +
                     (a.part ? static_cast<size_t>(a.B + 1) * sizeof(int) : 0);
  hipLaunchKernelGGL((gqa_decode_paged_fp8_kernel<D>), dim3(groups), dim3(kThreads), lds, st, c, a);
  const int heads = c.Hkv * a.chunks;
  // us of decode and merge, the kernel for few records / the other: 64 (sequence,
  // head)s 27.9 / 24.7, 128 36.1 / 35.0, 256 107.1 / 108.0
  if (a.part && a.B * heads >= 256)
    hipLaunchKernelGGL((gqa_decode_paged_fp8_merge_few_kernel<D>), dim3(heads, a.B), dim3(256), 0, st, c, a, groups);
  else if (a.part)
    hipLaunchKernelGGL((gqa_decode_paged_fp8_merge_kernel<D>), dim3(a.Hq, a.B, D / 64), dim3(256), 0, st, c, a, groups);
  return check_launch("gqa_decode_paged_fp8");
}

// Workgroups a split may use: one a unit, and as many as the 256 CUs hold at
// most (the kernel's registers: 1, 2 or 3 a CU), so that all run at once.
long split_groups(int B, int heads, int max_len, int D) {
  const long units = std::max(1L, (static_cast<long>(max_len) + kUnit - 1) / kUnit);
  const long resident = 256 * (D == 256 ? 1 : D == 128 ? 2 : 3);
  return std::min<long>(resident, static_cast<long>(B) * heads * units);
}

}  // namespace
}  // namespace aila

extern "C" size_t aila_hip_gqa_decode_paged_fp8_workspace_size(int B, int Hq, int Hkv, int D, int max_len) {
  using namespace aila;
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || max_len < 0) return 0;
  int tile, chunks;
  head_tiles(Hq / Hkv, &tile, &chunks);
  return units_bytes(B) + std::max(2L, split_groups(B, Hkv * chunks, max_len, D)) * record_bytes(tile, D);
}

extern "C" int aila_hip_gqa_decode_paged_fp8(const void* q, long q_stride, const void* k_pages, const void* v_pages,
                                             const float* k_scale, const float* v_scale, void* out, void* workspace,
                                             size_t workspace_bytes, int B, int Hq, int Hkv, int D, int page_size,
                                             int num_pages, const int* block_table, int max_pages, int max_len,
                                             const int* seq_lens, void* stream) {
  using namespace aila;
  AILA_REQUIRE(q && out && block_table && seq_lens, "gqa_decode_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("gqa_decode_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  AILA_REQUIRE(B > 0 && B <= kMaxSequences, "gqa_decode_paged_fp8: B=%d outside [1, %d]", B, kMaxSequences);
  AILA_REQUIRE(Hq > 0 && Hq % Hkv == 0 && Hq <= 65535, "gqa_decode_paged_fp8: bad heads (Hq=%d Hkv=%d)", Hq, Hkv);
  AILA_REQUIRE(q_stride >= static_cast<long>(Hq) * D && q_stride % 8 == 0,
               "gqa_decode_paged_fp8: query stride %ld must be a multiple of 8 and hold Hq * D = %ld values", q_stride,
               static_cast<long>(Hq) * D);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
               "gqa_decode_paged_fp8: q and out must be 16-byte aligned");
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30),
               "gqa_decode_paged_fp8: bad max_pages=%d", max_pages);
  AILA_REQUIRE(max_len >= 0 && max_len <= max_pages * page_size, "gqa_decode_paged_fp8: max_len=%d outside [0, %d]",
               max_len, max_pages * page_size);
  PagedFp8 c{static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), k_scale, v_scale,
             block_table, max_pages, num_pages, Hkv, page_size / kScaleRows};
  Fp8DecodeArgs a{};
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<bf16*>(out);
  a.seq_lens = seq_lens;
  a.B = B; a.Hq = Hq; a.group = Hq / Hkv;
  head_tiles(a.group, &a.tile, &a.chunks);
  a.max_len = max_len;
  a.scale_log2 = kLog2e / sqrtf(static_cast<float>(D));
  const int heads = Hkv * a.chunks;
  AILA_REQUIRE(static_cast<long>(B) * heads * ((max_len + kUnit - 1) / kUnit + 1) < (1L << 31),
               "gqa_decode_paged_fp8: B=%d sequences of up to %d rows and %d heads are too many", B, max_len, heads);
  // one workgroup each without a split: fewer than 2^32 threads, the most of a launch
  AILA_REQUIRE(static_cast<long>(B) * heads * kThreads < (1L << 32), "gqa_decode_paged_fp8: B=%d sequences of %d heads are too many",
               B, heads);
  long groups = static_cast<long>(B) * heads;
  // One workgroup per (sequence, head) where that is faster than a split and its
  // merge: up to 6 units a sequence (D = 64: 8, D = 256: 4), and the longer the more
  // of the CUs they fill, up to 4096 rows (D = 256: 2048) where they fill all. us in
  // a graph, whole / split, lengths between 5 and 100% of the bound. D = 128, 8 heads:
  // 1 sequence of 768 rows 7.9 / 8.7, 900 9.2 / 8.7; 8 of 1024 11.2 / 11.4, 1300 13.7 /
  // 11.8; 16 of 1024 11.6 / 16.0, 2000 19.0 / 18.8, 3000 25.8 / 20.4; 64 of 2000 30.2 /
  // 41.2, 4000 57.2 / 56.7, 8000 108 / 101. D = 64, 8 heads: 1 of 1024 7.4 / 7.7, 1300
  // 9.0 / 7.8; 16 of 2000 12.4 / 13.8, 3000 16.6 / 14.8; 64 of 4000 29.9 / 35.3. D = 256,
  // 4 heads: 1 of 512 10.9 / 11.1, 612 13.0 / 11.2; 32 of 1024 19.6 / 26.6, 2000 32.8 /
  // 32.6; 64 of 2000 35.4 / 44.0, 4000 65.7 / 61.7. The bound is all that the rule sees:
  // one long sequence among short ones pays for it (32 / 8, D = 128, one of 4096 rows
  // and 31 of 100, 32.5 / 22.2; 16 / 4, D = 256, one of 2048 and 63 of 100, 33.1 / 23.1),
  // and so do short sequences under a loose bound (32 of up to 1024, 14.6 / 22.8).
  const long few = (D == 64 ? 8 : D == 128 ? 6 : 4) * kUnit, many = D == 256 ? 2048 : 4096;
  const bool whole = max_len <= std::max(few, many * std::min(groups, 256L) / 256);
  if (workspace != nullptr) {
    AILA_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "gqa_decode_paged_fp8: workspace must be 16-byte aligned");
    const size_t rec = record_bytes(a.tile, D);
    if (workspace_bytes < units_bytes(B) + 2 * rec)
      return set_error(AILA_HIP_EWORKSPACE, "gqa_decode_paged_fp8: workspace %zu bytes, %zu are the least", workspace_bytes,
                       units_bytes(B) + 2 * rec);
    if (!whole) {
      groups = std::min<long>(split_groups(B, heads, max_len, D), static_cast<long>((workspace_bytes - units_bytes(B)) / rec));
      a.units = static_cast<int*>(workspace);
      a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + units_bytes(B));
    }
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (D) {
    case 64: return launch<64>(c, a, static_cast<int>(groups), st);
    case 128: return launch<128>(c, a, static_cast<int>(groups), st);
    default: return launch<256>(c, a, static_cast<int>(groups), st);
  }
}
