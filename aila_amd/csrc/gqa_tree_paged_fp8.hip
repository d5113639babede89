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

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxSequences = 4096;    // their unit counts live in LDS
constexpr int kRecTail = 4;
constexpr int kCus = 256;
template <int D> constexpr int kTiles = D == 256 ? 1 : 2;     // column tiles of a wave
template <int D> constexpr int kCap = kWaves * kTiles<D>;     // column tiles of a workgroup
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
// KV head and all keys; its tiles are spread over 1, 2, 4 or 8 lanes of waves, the
// workgroup's other waves take other keys, so that a unit - a strip of 32 keys for
// each wave - costs the same whatever the number of columns. Full items first; of
// the rest, more than 3/4 of an item is one, else it is half an item and what is
// left over, or less than that: of 9 tiles in 16 places 7 would idle.
struct Shape {
  int q0, n, len;      // first token, tokens that are computed, rows
  int base;            // first drafted row
  int full;            // items of kCap tiles (the last may be short of them)
  int half, rest;      // tiles of the others, 0: there is none
};

template <int D>
__device__ __forceinline__ int lanes_log2(int tiles) {
  const int lanes = (tiles + kTiles<D> - 1) / kTiles<D>;
  return lanes <= 1 ? 0 : 32 - __builtin_clz(lanes - 1);
}
template <int D>
__device__ __forceinline__ int item_units(int tiles, int len) {
  const int rows = (32 * kWaves) >> lanes_log2<D>(tiles);
  return max(1, (len + rows - 1) / rows);      // an output without keys is written too
}

template <int D>
__device__ __forceinline__ Shape shape_of(const TreeArgs& a, int b) {
  Shape s;
  s.q0 = min(max(a.query_start[b], 0), a.T);
  s.n = max(min(max(a.query_start[b + 1], 0), a.T) - s.q0, 0);
  s.len = min(max(a.seq_lens[b], 0), a.max_len);
  s.base = s.len - s.n;
  s.n = min(s.n, 32 * a.words32);   // those behind have no mask
  const int all = (s.n * a.group + 15) / 16;
  s.full = all / kCap<D>;
  s.rest = all % kCap<D>;
  s.half = 0;
  if (4 * s.rest > 3 * kCap<D>) {
    ++s.full;
    s.rest = 0;
  } else if (2 * s.rest > kCap<D>) {
    s.half = kCap<D> / 2;
    s.rest -= s.half;
  }
  return s;
}
// Units of a KV head.
template <int D>
__device__ __forceinline__ int head_units(const Shape& s) {
  int n = s.full > 0 ? s.full * item_units<D>(kCap<D>, s.len) : 0;
  if (s.half > 0) n += item_units<D>(s.half, s.len);
  if (s.rest > 0) n += item_units<D>(s.rest, s.len);
  return n;
}

// An item: its first tile, its tiles, its units and its KV head's units before it.
struct Item { int tile0, tiles, units, before; };
template <int D>
__device__ __forceinline__ Item item_at(const Shape& s, int index) {
  Item it;
  const int u = item_units<D>(kCap<D>, s.len);
  it.tile0 = min(index, s.full) * kCap<D>;
  it.before = min(index, s.full) * u;
  it.tiles = kCap<D>;
  it.units = u;
  if (index >= s.full) {
    const bool second = s.half > 0 && index > s.full;
    it.tiles = s.half > 0 && !second ? s.half : s.rest;
    it.units = item_units<D>(it.tiles, s.len);
    if (second) {
      it.tile0 += s.half;
      it.before += item_units<D>(s.half, s.len);
    }
  }
  return it;
}
// The item that holds unit `at` of a KV head.
template <int D>
__device__ __forceinline__ Item item_of_unit(const Shape& s, int at) {
  const int u = item_units<D>(kCap<D>, s.len);
  int index = at / u;
  if (index >= s.full) index = s.full + (s.half > 0 && at - s.full * u >= item_units<D>(s.half, s.len) ? 1 : 0);
  return item_at<D>(s, index);
}
__device__ __forceinline__ int item_count(const Shape& s) { return s.full + (s.half > 0) + (s.rest > 0); }

// s_pre[b] = units of a KV head of the requests before b, for b <= B.
template <int D>
__device__ __forceinline__ void scan_units(const TreeArgs& a, int* s_pre) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int b = b0 + lane;
      int n = 0;
      if (b < a.B) n = head_units<D>(shape_of<D>(a, b));
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

// Codes of a strip of 32 keys, as Strip. K and V have registers of one strip each:
// the next strip's K goes out when this one's scores are made, its V when this one's
// products are.
template <int D, bool V>
__device__ __forceinline__ void load_codes(Strip<D>& s, const uint8_t* pages, int bid_a, int bid_b, int m16, int g4) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int bid = x ? bid_b : bid_a;
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(pages) + static_cast<size_t>(max(bid, 0)) * (kScaleRows * D), 0, bid >= 0 ? kScaleRows * D : 0, kBufferRsrcWord3);
    if constexpr (!V) {
#pragma unroll
      for (int kk = 0; kk < D / 64; ++kk) s.k[x][kk] = __builtin_amdgcn_raw_buffer_load_b128(r, m16 * D + 16 * g4 + 64 * kk, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = (4 * g4 + j) * D + m16 * (D / 16);
        if constexpr (D == 256) {
          const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) s.v[4 * x + j][i] = w[i];
        } else if constexpr (D == 128) {
          const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0);
          s.v[4 * x + j][0] = w[0];
          s.v[4 * x + j][1] = w[1];
        } else {
          s.v[4 * x + j][0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
        }
      }
    }
  }
}

// What a strip's blocks contribute: K scales times log2(e) / sqrt(D), exponents of
// the V scales.
struct Scales { float ka, kb; int ea, eb; };

template <int D>
__device__ __forceinline__ void make_scores(f32x4* sa, f32x4* sb, const Strip<D>& s, const bf16x8_t (*q)[D / 32]) {
  constexpr int N = kTiles<D>;
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
    }
#pragma unroll
    for (int t = 0; t < N; ++t) {
      sa[t] = mfma16x16x32(ahi, q[t][2 * kk + 1], sa[t]);
      sb[t] = mfma16x16x32(bhi, q[t][2 * kk + 1], sb[t]);
    }
  }
}

// keep[t]: the rows that tile t's column of this lane attends.
template <int D>
__device__ __forceinline__ void mask_scores(f32x4* sa, f32x4* sb, const uint32_t* keep, int g4) {
#pragma unroll
  for (int t = 0; t < kTiles<D>; ++t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!(keep[t] >> (4 * g4 + j) & 1)) sa[t][j] = -INFINITY;
      if (!(keep[t] >> (16 + 4 * g4 + j) & 1)) sb[t][j] = -INFINITY;
    }
  }
}

// A masked row's weight is 0, but 0 times NaN is NaN, and a masked row may hold
// anything: a masked strip's NaN codes are taken out of V, and where there are any
// a second product counts those that each column attends, and puts the NaN back.
template <int D>
__device__ __forceinline__ void mend_values(Column<D>* c, Strip<D>& s, const uint32_t* keep, int g4) {
  uint32_t seen = 0;
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) seen |= nan_codes(s.v[j][w]);
  }
  if (__ballot(seen != 0) == 0) return;
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
    for (int t = 0; t < kTiles<D>; ++t) {
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

// Scores to weights p. The V scales go into the exponents, and out of the weights'
// sums again. A weight is rounded to bf16 once (half a step, 2^-8 of it, at random);
// the sums are taken of the rounded ones, in fp32, so that they add up to 1.
template <int D>
__device__ __forceinline__ void make_weights(u32x4* p, Column<D>* c, const f32x4* sa, const f32x4* sb, const Scales& x) {
#pragma unroll
  for (int t = 0; t < kTiles<D>; ++t) {
    const float ta = fmaxf(fmaxf(sa[t][0], sa[t][1]), fmaxf(sa[t][2], sa[t][3]));
    const float tb = fmaxf(fmaxf(sb[t][0], sb[t][1]), fmaxf(sb[t][2], sb[t][3]));
    const float top = xrow4_max(fmaxf(ta * x.ka, tb * x.kb));
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
    const float ra = static_cast<float>(x.ea) - ref, rb = static_cast<float>(x.eb) - ref;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      p[t][e] = pack_bf16x2(fast_exp2(fmaf(sa[t][2 * e], x.ka, ra)), fast_exp2(fmaf(sa[t][2 * e + 1], x.ka, ra)));
      p[t][2 + e] = pack_bf16x2(fast_exp2(fmaf(sb[t][2 * e], x.kb, rb)), fast_exp2(fmaf(sb[t][2 * e + 1], x.kb, rb)));
    }
    c[t].l = fmaf(add_pair(p[t][1], add_pair(p[t][0], 0.f)), pow2f(-x.ea), c[t].l);
    c[t].l = fmaf(add_pair(p[t][3], add_pair(p[t][2], 0.f)), pow2f(-x.eb), c[t].l);
  }
}

template <int D>
__device__ __forceinline__ void add_values(Column<D>* c, const Strip<D>& s, const u32x4* p) {
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
      for (int t = 0; t < kTiles<D>; ++t) c[t].acc[4 * w + i] = mfma16x16x32(vt[i], as_bf16x8(p[t]), c[t].acc[4 * w + i]);
    }
  }
}

template <int D>
__global__ __launch_bounds__(kThreads, 1) void gqa_tree_paged_fp8_kernel(PagedFp8 c, TreeArgs a) {
  constexpr int kStride = kAccStride<D>, kT = kTiles<D>;
  extern __shared__ __attribute__((aligned(16))) unsigned char s_dyn[];
  float* s_acc = reinterpret_cast<float*>(s_dyn);             // [kWaves][16 kT][kStride]
  float* s_ml = s_acc + kWaves * 16 * kT * kStride;           // [kWaves][16 kT][2]
  int* s_pre = reinterpret_cast<int*>(s_ml + kWaves * 16 * kT * 2);   // [B + 1]
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
    int b, kvh, i0, i1;
    Shape s;
    Item it;
    if (a.part == nullptr) {
      b = u / (c.Hkv * a.chunks);
      const int hi = u % (c.Hkv * a.chunks);
      kvh = hi / a.chunks;
      s = shape_of<D>(a, b);
      if (hi % a.chunks >= item_count(s)) return;
      it = item_at<D>(s, hi % a.chunks);
      i0 = 0;
      i1 = it.units;
      u = u1;
    } else {
      b = __builtin_amdgcn_readfirstlane(find_request(s_pre, a.B, u / c.Hkv));
      s = shape_of<D>(a, b);
      const int before = __builtin_amdgcn_readfirstlane(s_pre[b]), per = __builtin_amdgcn_readfirstlane(s_pre[b + 1]) - before;
      const int at = u - before * c.Hkv;
      kvh = at / per;
      it = item_of_unit<D>(s, at - kvh * per);
      i0 = at - kvh * per - it.before;
      i1 = min(it.units, i0 + (u1 - u));
      u += i1 - i0;
    }
    const int lg = lanes_log2<D>(it.tiles);
    const int lanes = 1 << lg, rows = (32 * kWaves) >> lg;                  // keys of a unit
    const int cols = s.n * a.group;                                         // the request's
    const int tiles = min(it.tiles, (cols + 15) / 16 - it.tile0);
    const int per = (it.tiles + lanes - 1) >> lg;                           // of a wave
    const int mine = min(max(tiles - (wave & (lanes - 1)) * per, 0), per);

    bf16x8_t q[kT][D / 32];
    size_t words_at[kT];
    Column<D> col[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int x = min(16 * (it.tile0 + (wave & (lanes - 1)) * per + t) + m16, cols - 1);   // past the last: its copies, not stored
      const int tok = x / a.group;
      const bf16* src = a.q + static_cast<size_t>(s.q0 + tok) * a.q_stride + static_cast<size_t>(kvh * a.group + x - tok * a.group) * D;
      words_at[t] = static_cast<size_t>(s.q0 + tok) * a.words32;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) q[t][ks] = as_bf16x8(ld16(src + 64 * (ks >> 1) + 16 * g4 + 8 * (ks & 1)));
      clear_column(col[t]);
    }

    // strips of this wave: row0 + rows * n, n < ns
    const int row0 = i0 * rows + 32 * (wave >> lg);
    const int end = min(i1 * rows, s.len);
    const int ns = mine > 0 && row0 < end ? (end - row0 + rows - 1) / rows : 0;
    const int blk_end = (end + kScaleRows - 1) / kScaleRows;
    const int open = min(end, s.base);        // rows that every column attends
    for (int n0 = 0; n0 < ns; n0 += 32) {
      // lane l holds block l % 2 of strip n0 + l / 2
      const int blk = (row0 + (n0 + (lane >> 1)) * rows) / kScaleRows + (lane & 1);
      const BlockRef ref = block_ref(c, b, kvh, blk, blk_end);
      const int n1 = min(ns - n0, 32);
      Strip<D> x;
      auto bid = [&](int n, int i) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(ref.bid, (2 * n + i) & 63); };
      auto load_k = [&](int n) __attribute__((always_inline)) {
        load_codes<D, false>(x, c.k_pages, n < n1 ? bid(n, 0) : -1, n < n1 ? bid(n, 1) : -1, m16, g4);
      };
      auto load_v = [&](int n) __attribute__((always_inline)) {
        load_codes<D, true>(x, c.v_pages, n < n1 ? bid(n, 0) : -1, n < n1 ? bid(n, 1) : -1, m16, g4);
      };
      auto scales = [&](int n) __attribute__((always_inline)) {
        // no page: all rows masked, and -inf times a scale of 0 would be NaN
        Scales r;
        r.ka = (bid(n, 0) >= 0 ? readlane_f(ref.ks, 2 * n) : 1.0f) * a.scale_log2;
        r.kb = (bid(n, 1) >= 0 ? readlane_f(ref.ks, 2 * n + 1) : 1.0f) * a.scale_log2;
        r.ea = held_exp(readlane_f(ref.vs, 2 * n));
        r.eb = held_exp(readlane_f(ref.vs, 2 * n + 1));
        return r;
      };
      load_k(0);
      load_v(0);
      // the strips whose rows all columns attend, then the others
      const bool hole = __ballot(blk < blk_end && ref.bid < 0) != 0;
      const int plain = hole ? 0 : min(n1, max(0, open - row0 - n0 * rows + rows - 32) / rows);
      f32x4 sa[kT], sb[kT];
      u32x4 p[kT];
      int n = 0;
      for (; n < plain; ++n) {
        make_scores<D>(sa, sb, x, q);
        __builtin_amdgcn_sched_barrier(0);
        load_k(n + 1);
        __builtin_amdgcn_sched_barrier(0);
        make_weights<D>(p, col, sa, sb, scales(n));
        add_values<D>(col, x, p);
        __builtin_amdgcn_sched_barrier(0);
        load_v(n + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      for (; n < n1; ++n) {
        make_scores<D>(sa, sb, x, q);
        load_k(n + 1);
        const int row = row0 + (n0 + n) * rows;
        const uint32_t held = (bid(n, 0) >= 0 ? 0xffffu : 0u) | (bid(n, 1) >= 0 ? 0xffff0000u : 0u);
        uint32_t keep[kT];
#pragma unroll
        for (int t = 0; t < kT; ++t) keep[t] = attended(a, words_at[t], row, s.base, end) & held;
        mask_scores<D>(sa, sb, keep, g4);
        mend_values<D>(col, x, keep, g4);
        make_weights<D>(p, col, sa, sb, scales(n));
        add_values<D>(col, x, p);
        load_v(n + 1);
      }
    }

    // ---- the waves' results meet ------------------------------------------
    __syncthreads();   // the item before has been read
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const float l = xrow4_sum(col[t].l);
      const int slot = (wave * kT + t) * 16 + m16;
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
    const bool whole = i0 == 0 && i1 == it.units;
    float* rec = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (i0 == 0 ? 1 : 0)) * a.rec_cols * (D + kRecTail);
    const int here = min(16 * tiles, cols - 16 * it.tile0);      // columns of the item
    const int parts = kWaves >> lg;
    for (int idx = threadIdx.x; idx < here * (D / 4); idx += kThreads) {
      const int x = idx / (D / 4), d = idx % (D / 4) * 4;
      const int tile = x >> 4, w0 = tile / per;
      const int slot0 = (w0 * kT + tile - w0 * per) * 16 + (x & 15);
      const int step = lanes * kT * 16;     // the same column, other keys
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
        const int y = 16 * it.tile0 + x, tok = y / a.group;
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
  const int index = min(x0 / (16 * kCap<D>), s.full);
  const Item it = item_at<D>(s, index + (index == s.full && s.half > 0 && x0 >= 16 * (s.full * kCap<D> + s.half) ? 1 : 0));
  const int before = a.units[b], units = a.units[a.B] * c.Hkv, groups = min(launched, units);
  const int first = before * c.Hkv + kvh * (a.units[b + 1] - before) + it.before;
  // workgroup w holds unit x: the largest w with w U / W < x + 1
  const int w0 = static_cast<int>((static_cast<long>(first + 1) * groups - 1) / units);
  const int w1 = static_cast<int>((static_cast<long>(first + it.units) * groups - 1) / units);
  if (w0 == w1) return;   // one workgroup wrote the output
  const int d = static_cast<int>(threadIdx.x) % kQuads * 4, x = static_cast<int>(threadIdx.x) / kQuads % kMergeCols;
  const int ph = static_cast<int>(threadIdx.x) / (kQuads * kMergeCols);
  const int y = min(x0 + x, cols - 1);
  const float* at = a.part + static_cast<size_t>(y - 16 * it.tile0) * (D + kRecTail);
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
  m.items = static_cast<int>(tiles / kCap<D> + 2);    // of the rest, two at most
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
  const size_t lds = static_cast<size_t>(kWaves) * 16 * kTiles<D> * (kAccStride<D> + 2) * sizeof(float) +
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
