// GQA attention of drafted token trees over the 8-bit paged cache (gfx950).
//
//   o_i = sum_j softmax_j(q_i . K_j / sqrt(D)) V_j
//
// over the rows j < L - n before a request's n drafted tokens, and the drafted
// rows whose bit is set in token i's mask. The query rows of a KV head are its
// columns: (token, head) pairs, token-major, in tiles of 16, the columns of the
// matrix instructions (v_mfma_f32_16x16x32_bf16, products and lane layout as
// Strip in paged_fp8.hpp). Codes go from memory to registers, are converted to
// bf16 there (exact, unscaled: the scales are powers of two and go into the
// softmax's exponents) and serve every tile of the wave.
#include "paged_fp8.hpp"

#include <algorithm>

namespace aila {
namespace {

constexpr int kTiles = 2;              // column tiles of a wave
constexpr int kMaxSequences = 4096;    // their unit counts live in LDS
constexpr int kRecTail = 4;
constexpr int kCus = 256;
// D = 256: a wave's columns and strips take more than half of a SIMD's registers.
template <int D> constexpr int kWavesOf = D == 256 ? 4 : 8;
template <int D> constexpr int kCap = kWavesOf<D> * kTiles;   // column tiles of a workgroup
template <int D> constexpr int kAccStride = D + 4;            // of a column in LDS, padded

struct TreeArgs {
  const bf16* q;
  long q_stride;
  bf16* out;
  const uint32_t* mask;                // [T, 2 words]
  int words32;
  float* part;                         // records; null: one workgroup per item
  int* units;                          // [B + 1] for the merge: units of a KV head before each request
  const int* query_start;
  const int* seq_lens;
  int T, B, Hq, group;
  int max_len;
  int chunks;                          // most items of a request and KV head
  int rec_cols;                        // columns of a record
  float scale_log2;
};

// What a request's columns are cut into. An item is up to kCap column tiles of a
// KV head and all keys; its tiles are spread over `lanes` waves (a power of two),
// and the workgroup's other waves take other keys, so that a unit - a strip of 32
// keys for each wave - costs the same whatever the number of columns.
struct Shape {
  int q0, n, len;      // first token, tokens that are computed, rows
  int base;            // first drafted row
  int tiles;           // column tiles of an item
  int items;           // of a KV head
  int lanes_log2;
  int units;           // of an item
};

template <int D>
__device__ __forceinline__ int unit_rows(const Shape& s) { return (32 * kWavesOf<D>) >> s.lanes_log2; }

template <int D>
__device__ __forceinline__ Shape shape_of(const TreeArgs& a, int b) {
  Shape s;
  s.q0 = min(max(a.query_start[b], 0), a.T);
  s.n = max(min(max(a.query_start[b + 1], 0), a.T) - s.q0, 0);
  s.len = min(max(a.seq_lens[b], 0), a.max_len);
  s.base = s.len - s.n;
  s.n = min(s.n, 32 * a.words32);   // those behind have no mask
  const int all = (s.n * a.group + 15) / 16;
  s.items = (all + kCap<D> - 1) / kCap<D>;
  s.tiles = s.items > 0 ? (all + s.items - 1) / s.items : 0;
  const int lanes = (s.tiles + kTiles - 1) / kTiles;
  s.lanes_log2 = lanes <= 1 ? 0 : 32 - __builtin_clz(lanes - 1);
  s.units = max(1, (s.len + unit_rows<D>(s) - 1) / unit_rows<D>(s));   // an output without keys is written too
  return s;
}

// s_pre[b] = units of a KV head of the requests before b, for b <= B.
template <int D>
__device__ __forceinline__ void scan_units(const TreeArgs& a, int* s_pre) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int b = b0 + lane;
      int n = 0;
      if (b < a.B) {
        const Shape s = shape_of<D>(a, b);
        n = s.items * s.units;
      }
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

// The last request whose units begin at or before x.
__device__ __forceinline__ int find_request(const int* pre, int n, int x) {
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

// acc + the two bf16 of x.
__device__ __forceinline__ float add_pair(uint32_t x, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc, false);
}

// The rows [row, row + 32) that a token attends, as bits: those before the draft
// (row < base), the drafted ones by its mask words, none from len on.
__device__ __forceinline__ uint32_t attended(const TreeArgs& a, size_t words_at, int row, int base, int len) {
  const int o = row - base, i = o >> 5, sh = o & 31;
  auto word = [&](int w) __attribute__((always_inline)) -> uint32_t {
    return w < 0 ? ~0u : w < a.words32 ? a.mask[words_at + w] : 0u;
  };
  const uint64_t both = static_cast<uint64_t>(word(i + 1)) << 32 | word(i);
  const uint32_t keep = static_cast<uint32_t>(both >> sh);
  const int left = len - row;
  return left >= 32 ? keep : left > 0 ? keep & ((1u << left) - 1) : 0u;
}

// One strip of 32 keys into N column tiles. ka, kb: the K scales times log2(e) /
// sqrt(D); ea, eb: the exponents of the V scales. masked: keep[t] holds the rows
// that tile t's column of this lane attends.
template <int D, int N>
__device__ __forceinline__ void tree_step(Column<D>* c, Strip<D>& s, const bf16x8_t (*q)[D / 32], float ka, float kb, int ea,
                                          int eb, bool masked, const uint32_t* keep, int g4) {
  f32x4 sa[N], sb[N];
#pragma unroll
  for (int t = 0; t < N; ++t) sa[t] = sb[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int kk = 0; kk < D / 64; ++kk) {
    bf16x8_t alo, ahi, blo, bhi;
    fp8x16_to_bf16(s.k[0][kk], alo, ahi);
    fp8x16_to_bf16(s.k[1][kk], blo, bhi);
#pragma unroll
    for (int t = 0; t < N; ++t) {
      sa[t] = mfma16x16x32(alo, q[t][2 * kk], sa[t]);
      sb[t] = mfma16x16x32(blo, q[t][2 * kk], sb[t]);
      sa[t] = mfma16x16x32(ahi, q[t][2 * kk + 1], sa[t]);
      sb[t] = mfma16x16x32(bhi, q[t][2 * kk + 1], sb[t]);
    }
  }
  // A masked row's weight is 0, but 0 times NaN is NaN, and a masked row may hold
  // anything: a masked strip's NaN codes are taken out of V, and where there are any
  // a second product counts those that each column attends, and puts the NaN back.
  if (masked) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(keep[t] >> (4 * g4 + j) & 1)) sa[t][j] = -INFINITY;
        if (!(keep[t] >> (16 + 4 * g4 + j) & 1)) sb[t][j] = -INFINITY;
      }
    }
    uint32_t seen = 0;
#pragma unroll
    for (int w = 0; w < D / 64; ++w) {
#pragma unroll
      for (int j = 0; j < 8; ++j) seen |= nan_codes(s.v[j][w]);
    }
    if (__ballot(seen != 0)) {
#pragma unroll
      for (int w = 0; w < D / 64; ++w) {
        uint32_t one[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t n = nan_codes(s.v[j][w]) >> 7;
          one[j] = n * 0x38u;      // the code of 1
          s.v[j][w] &= ~(n * 0xffu);
        }
        bf16x8_t vt[4];
        v_tiles(one, vt);
#pragma unroll
        for (int t = 0; t < N; ++t) {
          u32x4 pa;   // 1 where the column attends the row
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t k = keep[t] >> ((e < 2 ? 0 : 16) + 4 * g4 + 2 * (e & 1));
            pa[e] = (k & 1 ? 0x3f80u : 0u) | (k & 2 ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 n = mfma16x16x32(vt[i], as_bf16x8(pa), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int j = 0; j < 4; ++j)   // n[j] is 0 or at least 1
              c[t].acc[4 * w + i][j] = __uint_as_float(__float_as_uint(c[t].acc[4 * w + i][j]) |
                                                       ((0u - min(__float_as_uint(n[j]), 1u)) & 0x7fc00000u));
          }
        }
      }
    }
  }
  // The V scales go into the exponents, and out of the weights' sums again. A weight
  // is rounded to bf16 once (half a step, 2^-8 of it, at random); the sums are taken
  // of the rounded ones, in fp32, so that they add up to 1.
  u32x4 p[N];
#pragma unroll
  for (int t = 0; t < N; ++t) {
    const float ta = fmaxf(fmaxf(sa[t][0], sa[t][1]), fmaxf(sa[t][2], sa[t][3]));
    const float tb = fmaxf(fmaxf(sb[t][0], sb[t][1]), fmaxf(sb[t][2], sb[t][3]));
    const float top = xrow4_max(fmaxf(ta * ka, tb * kb));
    // the reference maximum moves only when a row exceeds it by 2^8
    if (__ballot(top > c[t].m + kLazyLog2)) {
      const float mn = fmaxf(c[t].m, top);
      const float alpha = c[t].m == -INFINITY ? 0.f : fast_exp2(c[t].m - mn);
      c[t].m = mn;
      c[t].l *= alpha;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) c[t].acc[i] *= alpha;
    }
    const float ref = c[t].m == -INFINITY ? 0.f : c[t].m;
    const float ra = static_cast<float>(ea) - ref, rb = static_cast<float>(eb) - ref;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      p[t][e] = pack_bf16x2(fast_exp2(fmaf(sa[t][2 * e], ka, ra)), fast_exp2(fmaf(sa[t][2 * e + 1], ka, ra)));
      p[t][2 + e] = pack_bf16x2(fast_exp2(fmaf(sb[t][2 * e], kb, rb)), fast_exp2(fmaf(sb[t][2 * e + 1], kb, rb)));
    }
    c[t].l = fmaf(add_pair(p[t][1], add_pair(p[t][0], 0.f)), pow2f(-ea), c[t].l);
    c[t].l = fmaf(add_pair(p[t][3], add_pair(p[t][2], 0.f)), pow2f(-eb), c[t].l);
  }
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s.v[j][w];
    bf16x8_t vt[4];
    v_tiles(v, vt);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < N; ++t) c[t].acc[4 * w + i] = mfma16x16x32(vt[i], as_bf16x8(p[t]), c[t].acc[4 * w + i]);
    }
  }
}

template <int D>
__global__ __launch_bounds__(64 * kWavesOf<D>, 1) void gqa_tree_paged_fp8_kernel(PagedFp8 c, TreeArgs a) {
  constexpr int kWaves = kWavesOf<D>, kThreads = 64 * kWaves, kStride = kAccStride<D>;
  extern __shared__ __attribute__((aligned(16))) unsigned char s_dyn[];
  float* s_acc = reinterpret_cast<float*>(s_dyn);             // [kWaves][16 kTiles][kStride]
  float* s_ml = s_acc + kWaves * 16 * kTiles * kStride;       // [kWaves][16 kTiles][2]
  int* s_pre = reinterpret_cast<int*>(s_ml + kWaves * 16 * kTiles * 2);   // [B + 1]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m16 = lane & 15, g4 = lane >> 4;

  int u, u1;
  if (a.part == nullptr) {
    u = blockIdx.x;       // (request, KV head, item) here
    u1 = u + 1;
  } else {
    scan_units<D>(a, s_pre);
    const int units = s_pre[a.B] * c.Hkv, groups = min(static_cast<int>(gridDim.x), units);
    const int w = blockIdx.x;
    if (w == 0)
      for (int i = threadIdx.x; i <= a.B; i += kThreads) a.units[i] = s_pre[i];
    if (w >= groups) return;
    u = share_begin(w, units, groups);
    u1 = share_begin(w + 1, units, groups);
  }
  while (u < u1) {
    int b, kvh, item, i0, i1;
    Shape s;
    if (a.part == nullptr) {
      b = u / (c.Hkv * a.chunks);
      const int hi = u % (c.Hkv * a.chunks);
      kvh = hi / a.chunks;
      item = hi % a.chunks;
      s = shape_of<D>(a, b);
      if (item >= s.items) return;
      i0 = 0;
      i1 = s.units;
      u = u1;
    } else {
      b = __builtin_amdgcn_readfirstlane(find_request(s_pre, a.B, u / c.Hkv));
      s = shape_of<D>(a, b);
      const int at = __builtin_amdgcn_readfirstlane(u - s_pre[b] * c.Hkv);
      const int hi = at / s.units;
      i0 = at % s.units;
      i1 = min(s.units, i0 + (u1 - u));
      u += i1 - i0;
      kvh = hi / s.items;
      item = hi % s.items;
    }
    const int lanes = 1 << s.lanes_log2;
    const int rows = unit_rows<D>(s);
    const int tile0 = item * s.tiles;                                       // of the request's
    const int cols = s.n * a.group;
    const int tiles = min(s.tiles, (cols + 15) / 16 - tile0);
    const int per = (s.tiles + lanes - 1) >> s.lanes_log2;                  // of a wave
    const int mine = min(max(tiles - (wave & (lanes - 1)) * per, 0), per);

    bf16x8_t q[kTiles][D / 32];
    size_t words_at[kTiles];
    Column<D> col[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int x = min(16 * (tile0 + (wave & (lanes - 1)) * per + t) + m16, cols - 1);   // past the last: its copies, not stored
      const int tok = x / a.group;
      const bf16* src = a.q + static_cast<size_t>(s.q0 + tok) * a.q_stride + static_cast<size_t>(kvh * a.group + x - tok * a.group) * D;
      words_at[t] = static_cast<size_t>(s.q0 + tok) * a.words32;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) q[t][ks] = as_bf16x8(ld16(src + 64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1)));
      clear_column(col[t]);
    }

    // strips of this wave: row0 + rows * n, n < ns
    const int row0 = i0 * rows + 32 * (wave >> s.lanes_log2);
    const int end = min(i1 * rows, s.len);
    const int ns = mine > 0 && row0 < end ? (end - row0 + rows - 1) / rows : 0;
    const int blk_end = (end + kScaleRows - 1) / kScaleRows;
    for (int n0 = 0; n0 < ns; n0 += 32) {
      // lane l holds block l % 2 of strip n0 + l / 2
      const BlockRef ref = block_ref(c, b, kvh, (row0 + (n0 + (lane >> 1)) * rows) / kScaleRows + (lane & 1), blk_end);
      const int n1 = min(ns - n0, 32);
      auto load = [&](Strip<D>& x, int n) __attribute__((always_inline)) {
        const bool in = n < n1;
        const int ba = __builtin_amdgcn_readlane(ref.bid, 2 * n & 63), bb = __builtin_amdgcn_readlane(ref.bid, (2 * n + 1) & 63);
        load_strip<D, false>(x, c, in ? ba : -1, in ? bb : -1, m16, g4);
      };
      auto step = [&](Strip<D>& x, int n) __attribute__((always_inline)) {
        const int ba = __builtin_amdgcn_readlane(ref.bid, 2 * n), bb = __builtin_amdgcn_readlane(ref.bid, 2 * n + 1);
        // no page: all rows masked, and -inf times a scale of 0 would be NaN
        const float ka = (ba >= 0 ? readlane_f(ref.ks, 2 * n) : 1.0f) * a.scale_log2;
        const float kb = (bb >= 0 ? readlane_f(ref.ks, 2 * n + 1) : 1.0f) * a.scale_log2;
        const int ea = held_exp(readlane_f(ref.vs, 2 * n)), eb = held_exp(readlane_f(ref.vs, 2 * n + 1));
        const int row = row0 + (n0 + n) * rows;
        const bool masked = row + 32 > min(end, s.base) || (ba | bb) < 0;
        uint32_t keep[kTiles] = {};
        if (masked) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            keep[t] = attended(a, words_at[t], row, s.base, end) & ((ba >= 0 ? 0xffffu : 0u) | (bb >= 0 ? 0xffff0000u : 0u));
        }
        if (mine == kTiles) tree_step<D, kTiles>(col, x, q, ka, kb, ea, eb, masked, keep, g4);
        else tree_step<D, 1>(col, x, q, ka, kb, ea, eb, masked, keep, g4);
      };
      Strip<D> x[2];
      load(x[0], 0);
      for (int n = 0; n < n1; n += 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (n + i < n1) {
            load(x[1 - i], n + i + 1);
            step(x[i], n + i);
          }
        }
      }
    }

    // ---- the waves' results meet ------------------------------------------
    __syncthreads();   // the item before has been read
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const float l = xrow4_sum(col[t].l);
      const int slot = (wave * kTiles + t) * 16 + m16;
      float* row = s_acc + slot * kStride;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) row[(D / 16) * (4 * g4 + i) + d] = col[t].acc[d][i];
      }
      if (g4 == 0) {
        s_ml[slot * 2] = col[t].m;
        s_ml[slot * 2 + 1] = l;
      }
    }
    __syncthreads();
    const bool whole = i0 == 0 && i1 == s.units;
    float* rec = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (i0 == 0 ? 1 : 0)) * a.rec_cols * (D + kRecTail);
    const int here = min(16 * tiles, cols - 16 * tile0);      // columns of the item
    const int parts = kWaves >> s.lanes_log2;
    for (int idx = threadIdx.x; idx < here * (D / 4); idx += kThreads) {
      const int x = idx / (D / 4), d = idx % (D / 4) * 4;
      const int tile = x >> 4, w0 = tile / per;
      const int slot0 = (w0 * kTiles + tile - w0 * per) * 16 + (x & 15);
      const int step = lanes * kTiles * 16;     // the same column, other keys
      float M = -INFINITY, L = 0.f;
      for (int i = 0; i < parts; ++i) M = fmaxf(M, s_ml[(slot0 + i * step) * 2]);
      f32x4 A = {0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < parts; ++i) {
        const int slot = slot0 + i * step;
        const float mw = s_ml[slot * 2];
        const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
        A += f * *reinterpret_cast<const f32x4*>(s_acc + slot * kStride + d);
        L += f * s_ml[slot * 2 + 1];
      }
      if (whole) {
        const int y = 16 * tile0 + x, tok = y / a.group;
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        *reinterpret_cast<u32x2*>(a.out + (static_cast<size_t>(s.q0 + tok) * a.Hq + kvh * a.group + y - tok * a.group) * D + d) =
            u32x2{pack_bf16x2(A[0] * inv, A[1] * inv), pack_bf16x2(A[2] * inv, A[3] * inv)};
      } else {
        float* r = rec + x * (D + kRecTail);
        *reinterpret_cast<f32x4*>(r + d) = A;
        if (d == 0) {
          r[D] = M;
          r[D + 1] = L;
        }
      }
    }
  }
}

// Joins the records of an item that several workgroups walked: o = sum_i 2^(m_i -
// M) acc_i / sum_i 2^(m_i - M) l_i. A workgroup takes kMergeCols columns of a
// request and KV head; its other threads take other records.
constexpr int kMergeCols = 4, kMergeThreads = 256;
template <int D>
__global__ __launch_bounds__(kMergeThreads) void gqa_tree_paged_fp8_merge_kernel(PagedFp8 c, TreeArgs a, int launched) {
  constexpr int kQuads = D / 4, kPhases = kMergeThreads / (kMergeCols * kQuads);
  __shared__ f32x4 s_a[kMergeThreads];
  __shared__ float s_m[kMergeThreads], s_l[kMergeThreads];
  const int b = blockIdx.y, kvh = blockIdx.x;
  const Shape s = shape_of<D>(a, b);
  const int cols = s.n * a.group, x0 = static_cast<int>(blockIdx.z) * kMergeCols;
  if (x0 >= cols) return;
  const int item = x0 / (16 * s.tiles);
  const int before = a.units[b], units = a.units[a.B] * c.Hkv, groups = min(launched, units);
  const int first = before * c.Hkv + (kvh * s.items + item) * s.units;
  // workgroup w holds unit x: the largest w with w U / W < x + 1
  const int w0 = static_cast<int>((static_cast<long>(first + 1) * groups - 1) / units);
  const int w1 = static_cast<int>((static_cast<long>(first + s.units) * groups - 1) / units);
  if (w0 == w1) return;   // one workgroup wrote the output
  const int d = static_cast<int>(threadIdx.x) % kQuads * 4, x = static_cast<int>(threadIdx.x) / kQuads % kMergeCols;
  const int ph = static_cast<int>(threadIdx.x) / (kQuads * kMergeCols);
  const int y = min(x0 + x, cols - 1);
  const float* at = a.part + static_cast<size_t>(y - 16 * s.tiles * item) * (D + kRecTail);
  const size_t step = static_cast<size_t>(a.rec_cols) * (D + kRecTail);
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  for (int w = w0 + ph; w <= w1; w += kPhases) {
    const float* r = at + (static_cast<size_t>(w) * 2 + (w == w0 ? 1 : 0)) * step;
    const f32x4 v = *reinterpret_cast<const f32x4*>(r + d);
    const float m = r[D], l = r[D + 1];
    const float mn = fmaxf(M, m);
    const float fo = M == -INFINITY ? 0.f : fast_exp2(M - mn), fn = m == -INFINITY ? 0.f : fast_exp2(m - mn);
    A = A * fo + v * fn;
    L = L * fo + l * fn;
    M = mn;
  }
  if constexpr (kPhases > 1) {
    s_a[threadIdx.x] = A;
    s_m[threadIdx.x] = M;
    s_l[threadIdx.x] = L;
    __syncthreads();
    if (ph > 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPhases; ++i) top = fmaxf(top, s_m[threadIdx.x + i * kQuads * kMergeCols]);
    A = f32x4{0.f, 0.f, 0.f, 0.f};
    L = 0.f;
#pragma unroll
    for (int i = 0; i < kPhases; ++i) {
      const int j = threadIdx.x + i * kQuads * kMergeCols;
      const float f = s_m[j] == -INFINITY ? 0.f : fast_exp2(s_m[j] - top);
      A += f * s_a[j];
      L += f * s_l[j];
    }
  }
  if (x0 + x >= cols) return;
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  const int tok = y / a.group;
  *reinterpret_cast<u32x2*>(a.out + (static_cast<size_t>(s.q0 + tok) * a.Hq + kvh * a.group + y - tok * a.group) * D + d) =
      u32x2{pack_bf16x2(A[0] * inv, A[1] * inv), pack_bf16x2(A[2] * inv, A[3] * inv)};
}

// The most that a request may have: columns, column tiles, items of a KV head.
struct Most { long cols; int items, rec_cols; };
template <int D>
Most most_of(int T, int words, int group) {
  Most m;
  m.cols = static_cast<long>(std::min<long>(T, 64L * words)) * group;
  const long tiles = (m.cols + 15) / 16;
  m.items = static_cast<int>((tiles + kCap<D> - 1) / kCap<D>);
  m.rec_cols = static_cast<int>(16 * std::min<long>(tiles, kCap<D>));
  return m;
}

size_t units_bytes(int B) { return (static_cast<size_t>(B + 1) * sizeof(int) + 255) / 256 * 256; }
template <int D>
size_t record_bytes(const Most& m) { return static_cast<size_t>(2) * m.rec_cols * (D + kRecTail) * sizeof(float); }

// Units of an item at most: one lane of waves walks all keys.
long most_units(int max_len) { return std::max(1L, (static_cast<long>(max_len) + 31) / 32); }

template <int D>
long split_groups(int B, int Hkv, const Most& m, int max_len) {
  return std::min<long>(kCus, static_cast<long>(B) * Hkv * m.items * most_units(max_len));
}

template <int D>
size_t workspace_need(int T, int B, int Hkv, int group, int words, int max_len) {
  const Most m = most_of<D>(T, words, group);
  return units_bytes(B) + std::max(2L, split_groups<D>(B, Hkv, m, max_len)) * record_bytes<D>(m);
}

template <int D>
int launch(const PagedFp8& c, TreeArgs a, int words, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Most m = most_of<D>(a.T, words, a.group);
  a.chunks = m.items;
  a.rec_cols = m.rec_cols;
  constexpr int kThreads = 64 * kWavesOf<D>;
  const long items = static_cast<long>(a.B) * c.Hkv * m.items;
  AILA_REQUIRE(items * most_units(a.max_len) < (1L << 31) && items * kThreads < (1L << 32),
               "gqa_tree_paged_fp8: B=%d requests of up to %ld query rows and %d keys are too many", a.B, m.cols, a.max_len);
  const long merges = (m.cols + kMergeCols - 1) / kMergeCols;
  AILA_REQUIRE(merges <= 65535, "gqa_tree_paged_fp8: %ld query rows of a KV head are too many", m.cols);
  long groups = items;
  if (workspace != nullptr) {
    const size_t rec = record_bytes<D>(m);
    if (workspace_bytes < units_bytes(a.B) + 2 * rec)
      return set_error(AILA_HIP_EWORKSPACE, "gqa_tree_paged_fp8: workspace %zu bytes, %zu are the least", workspace_bytes,
                       units_bytes(a.B) + 2 * rec);
    groups = std::min<long>(split_groups<D>(a.B, c.Hkv, m, a.max_len), static_cast<long>((workspace_bytes - units_bytes(a.B)) / rec));
    a.units = static_cast<int*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + units_bytes(a.B));
  }
  const size_t lds = static_cast<size_t>(kWavesOf<D>) * 16 * kTiles * (kAccStride<D> + 2) * sizeof(float) +
                     (a.part ? static_cast<size_t>(a.B + 1) * sizeof(int) : 0);
  hipLaunchKernelGGL((gqa_tree_paged_fp8_kernel<D>), dim3(groups), dim3(kThreads), lds, st, c, a);
  if (a.part)
    hipLaunchKernelGGL((gqa_tree_paged_fp8_merge_kernel<D>), dim3(c.Hkv, a.B, merges), dim3(kMergeThreads), 0, st, c, a,
                       static_cast<int>(groups));
  return check_launch("gqa_tree_paged_fp8");
}

}  // namespace
}  // namespace aila

extern "C" size_t aila_hip_gqa_tree_paged_fp8_workspace_size(int T, int B, int Hq, int Hkv, int D, int max_len,
                                                             int mask_words) {
  using namespace aila;
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_len < 0 || mask_words <= 0) return 0;
  switch (D) {
    case 64: return workspace_need<64>(T, B, Hkv, Hq / Hkv, mask_words, max_len);
    case 128: return workspace_need<128>(T, B, Hkv, Hq / Hkv, mask_words, max_len);
    case 256: return workspace_need<256>(T, B, Hkv, Hq / Hkv, mask_words, max_len);
    default: return 0;
  }
}

extern "C" int aila_hip_gqa_tree_paged_fp8(const void* q, long q_stride, const void* k_pages, const void* v_pages,
                                           const float* k_scale, const float* v_scale, void* out, void* workspace,
                                           size_t workspace_bytes, int T, int B, int Hq, int Hkv, int D, int page_size,
                                           int num_pages, const int* block_table, int max_pages, int max_len,
                                           const int* query_start, const int* seq_lens, const void* tree_mask,
                                           int mask_words, void* stream) {
  using namespace aila;
  AILA_REQUIRE(q && out && block_table && query_start && seq_lens && tree_mask, "gqa_tree_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("gqa_tree_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  AILA_REQUIRE(B > 0 && B <= kMaxSequences, "gqa_tree_paged_fp8: B=%d outside [1, %d]", B, kMaxSequences);
  AILA_REQUIRE(Hq > 0 && Hq % Hkv == 0 && Hq <= 65535, "gqa_tree_paged_fp8: bad heads (Hq=%d Hkv=%d)", Hq, Hkv);
  AILA_REQUIRE(mask_words > 0 && mask_words <= 64, "gqa_tree_paged_fp8: mask_words=%d outside [1, 64]", mask_words);
  AILA_REQUIRE(T > 0 && static_cast<long>(T) * (Hq / Hkv) <= (1L << 30), "gqa_tree_paged_fp8: T=%d tokens are too many", T);
  AILA_REQUIRE(q_stride >= static_cast<long>(Hq) * D && q_stride % 8 == 0,
               "gqa_tree_paged_fp8: query stride %ld must be a multiple of 8 and hold Hq * D = %ld values", q_stride,
               static_cast<long>(Hq) * D);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "gqa_tree_paged_fp8: q, out and workspace must be 16-byte aligned");
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(tree_mask) % 8 == 0, "gqa_tree_paged_fp8: tree_mask must be 8-byte aligned");
  AILA_REQUIRE(max_pages > 0 && static_cast<long>(max_pages) * page_size <= (1L << 30),
               "gqa_tree_paged_fp8: bad max_pages=%d", max_pages);
  AILA_REQUIRE(max_len >= 0 && max_len <= max_pages * page_size, "gqa_tree_paged_fp8: max_len=%d outside [0, %d]",
               max_len, max_pages * page_size);
  PagedFp8 c{static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages), k_scale, v_scale,
             block_table, max_pages, num_pages, Hkv, page_size / kScaleRows};
  TreeArgs a{};
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.out = static_cast<bf16*>(out);
  a.mask = static_cast<const uint32_t*>(tree_mask);
  a.words32 = 2 * mask_words;
  a.query_start = query_start;
  a.seq_lens = seq_lens;
  a.T = T; a.B = B; a.Hq = Hq; a.group = Hq / Hkv;
  a.max_len = max_len;
  a.scale_log2 = kLog2e / sqrtf(static_cast<float>(D));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (D) {
    case 64: return launch<64>(c, a, mask_words, workspace, workspace_bytes, st);
    case 128: return launch<128>(c, a, mask_words, workspace, workspace_bytes, st);
    default: return launch<256>(c, a, mask_words, workspace, workspace_bytes, st);
  }
}
