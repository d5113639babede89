// GQA attention of drafted token trees over the 8-bit paged cache (gfx950).
//
//   o_i = sum_j softmax_j(q_i . K_j / sqrt(D)) V_j
//
// over the rows j < L - n before a request's n drafted tokens, and the drafted
// rows whose bit is set in token i's mask. The query rows of a KV head are its
// columns: (token, head) pairs, token-major, in tiles of 32, one a wave. Products on
// v_mfma_f32_32x32x16_bf16, a strip of 32 keys at a time:
//   S^T = K Q^T     A = 32 keys, B = the wave's 32 columns
//     lane (m, h) = (l % 32, l / 32) loads 16 codes of key m at 32 kk + 16 h, two
//     operands of 8 dims; it receives keys 8 a + 4 h + c (a, c < 4) of column m.
//   O^T += V^T P^T  A = 32 head dims, B = P of 16 keys, in the registers where S^T
//     left it: step s takes keys 16 s + 4 h + {0..3, 8..11}. A lane loads those
//     rows' dims [D/32 m, D/32 (m + 1)) and pairs the rows' bytes with v_perm.
// Codes go from memory to registers and are converted to bf16 there (exact,
// unscaled: the scales are powers of two and go into the softmax's exponents).
//
// Up to some 40 columns a request it is bound by the bytes and their latency: 32 requests
// of 6000 rows, 8 KV heads, D = 128, 8 columns, 99 us = 4.1 TB/s; wider trees are bound by
// the conversions (64 codes a lane and strip) and the softmax on the vector ALU, 205
// instructions a strip and tile for 512 cycles of products, and take the other walk
// (walks_as_prompt, below). One sequence of 612 rows with 8 drafted tokens: 9.9 us in one
// launch, which is start-up and three strips in a row: lengths -> blocks -> codes.
//
// Tried and left: strips staged by DMA in LDS (no faster: 105 against 112 us for 32
// requests of 26 tokens after 3000 rows), lines touched some strips ahead (129), raised
// priority of either phase or wave (same), two tiles a wave at one wave a SIMD (the compiler
// moves all accumulators through the vector registers in every strip).
#include "paged_fp8.hpp"

#include <algorithm>
#include <type_traits>

namespace aila {
namespace {

constexpr int kTile = 32;              // columns of a wave
constexpr int kMaxSequences = 4096;    // their unit counts live in LDS
constexpr int kRecTail = 4;
constexpr int kCus = 256;
// D = 256: a wave's columns take more than half of a SIMD's registers.
template <int D> constexpr int kWaves = D == 256 ? 4 : 8;     // and column tiles of a workgroup
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
  int chunks;                          // without a split: workgroups of a request and KV head
  int rec_cols;                        // columns of a record
  float scale_log2;
};

// What a request's columns are cut into. An item is up to kWaves column tiles of a
// KV head and all keys, a wave for each tile; the workgroup's other waves take other
// keys (a power of two each), so that a unit - a strip of 32 keys for
// each wave - costs the same whatever the number of columns. Full items first; of
// the rest, more than 3/4 of an item is one, else it is half an item and what is
// left over, or less than that: of 5 tiles in 8 places 3 would idle.
struct Shape {
  int q0, n, len;      // first token, tokens that are computed, rows
  int base;            // first drafted row
  int full;            // items of kWaves tiles (the last may be short of them)
  int half, rest;      // tiles of the others, 0: there is none
};

__device__ __forceinline__ int lanes_log2(int tiles) { return tiles <= 1 ? 0 : 32 - __builtin_clz(tiles - 1); }
template <int D>
__device__ __forceinline__ int item_units(int tiles, int len) {
  const int rows = (32 * kWaves<D>) >> lanes_log2(tiles);
  return max(1, (len + rows - 1) / rows);      // an output without keys is written too
}

template <int D>
__device__ __forceinline__ Shape shape_of(const TreeArgs& a, int b) {
  Shape s;
  const int begin = a.query_start[b], end = a.query_start[b + 1], len = a.seq_lens[b];
  __builtin_amdgcn_sched_barrier(0);      // one round trip
  s.q0 = min(max(begin, 0), a.T);
  s.n = max(min(max(end, 0), a.T) - s.q0, 0);
  s.len = min(max(len, 0), a.max_len);
  s.base = s.len - s.n;
  s.n = min(s.n, 32 * a.words32);   // those behind have no mask
  const int all = (s.n * a.group + kTile - 1) / kTile;
  s.full = all / kWaves<D>;
  s.rest = all % kWaves<D>;
  s.half = 0;
  if (4 * s.rest > 3 * kWaves<D>) {
    ++s.full;
    s.rest = 0;
  } else if (2 * s.rest > kWaves<D>) {
    s.half = kWaves<D> / 2;
    s.rest -= s.half;
  }
  return s;
}
// Units of a KV head.
template <int D>
__device__ __forceinline__ int head_units(const Shape& s) {
  int n = s.full > 0 ? s.full * item_units<D>(kWaves<D>, s.len) : 0;
  if (s.half > 0) n += item_units<D>(s.half, s.len);
  if (s.rest > 0) n += item_units<D>(s.rest, s.len);
  return n;
}

// An item: its first tile, its tiles, its units and its KV head's units before it.
struct Item { int tile0, tiles, units, before; };
template <int D>
__device__ __forceinline__ Item item_at(const Shape& s, int index) {
  Item it;
  const int u = item_units<D>(kWaves<D>, s.len);
  it.tile0 = min(index, s.full) * kWaves<D>;
  it.before = min(index, s.full) * u;
  it.tiles = kWaves<D>;
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
  const int u = item_units<D>(kWaves<D>, s.len);
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

// Codes of a strip's K and V, one strip's registers each: the next strip's K goes
// out when this one's scores are made, its V when this one's products are. A block
// without a page is read as block 0: all its rows are masked.
template <int D>
struct Codes {
  u32x4 k[D / 32];
  static constexpr int VW = D == 256 ? 2 : 1;       // words of a row's run of dims
  uint32_t v[2][VW][8];                             // [step][word][row]
};

template <int D>
__device__ __forceinline__ void load_k(Codes<D>& x, const uint8_t* pages, int bid_a, int bid_b, int m32, int hf) {
  const uint32_t bid = static_cast<uint32_t>(max(m32 < 16 ? bid_a : bid_b, 0));
  const uint8_t* p = pages + static_cast<size_t>(bid) * (kScaleRows * D) + ((m32 & 15) * D + 16 * hf);
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) x.k[kk] = ld16(p + 32 * kk);
}

template <int D>
__device__ __forceinline__ void load_v(Codes<D>& x, const uint8_t* pages, int bid_a, int bid_b, int m32, int hf) {
  const uint32_t at = 4 * hf * D + (D == 64 ? 4 * (m32 & 15) : m32 * (D / 32));
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint8_t* p = pages + static_cast<size_t>(static_cast<uint32_t>(max(s ? bid_b : bid_a, 0))) * (kScaleRows * D);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* r = p + at + ((j & 3) + 8 * (j >> 2)) * D;
      if constexpr (D == 256) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(r);
        x.v[s][0][j] = w[0];
        x.v[s][1][j] = w[1];
      } else {
        x.v[s][0][j] = *reinterpret_cast<const uint32_t*>(r);
      }
    }
  }
}

// Head dim of row m of output part dt.
template <int D>
__device__ __forceinline__ int out_dim(int dt, int m) {
  return D == 64 ? 4 * (m & 15) + 2 * dt + (m >> 4) : (D / 32) * m + dt;
}

// V operands of a step from a word of each of its 8 rows: 4 parts, D = 64: both
// (the lanes of rows 16 .. 31 take the odd bytes).
template <int D>
__device__ __forceinline__ void step_tiles(const uint32_t (&v)[8], bf16x8_t* t, int m32) {
  if constexpr (D == 64) {
    const uint32_t sel = m32 < 16 ? 0x06020400u : 0x07030501u;
    u32x4 o[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], sel);
      o[0][e] = fp8x2_to_bf16x2<false>(w);
      o[1][e] = fp8x2_to_bf16x2<true>(w);
    }
    t[0] = as_bf16x8(o[0]);
    t[1] = as_bf16x8(o[1]);
  } else {
    bf16x8_t x[4];
    v_tiles(v, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = x[i];
  }
}

// A column's running softmax and its output: o[dt][i] is head dim out_dim(dt, 8 (i /
// 4) + 4 h + i % 4).
template <int D>
struct Tile {
  f32x16 o[D / 32];
  float m, l;          // maximum (log2 domain) and this lane's part of the sum
};

// What a strip's blocks contribute: K scales times log2(e) / sqrt(D), exponents of
// the V scales.
struct Scales { float ka, kb, ea, eb, ia, ib; };    // and the V scales' reciprocals

template <int D>
__device__ __forceinline__ f32x16 make_scores(const Codes<D>& x, const bf16x8_t (&q)[D / 16]) {
  f32x16 sc = {};
#pragma unroll
  for (int kk = 0; kk < D / 32; ++kk) {
    bf16x8_t lo, hi;
    fp8x16_to_bf16(x.k[kk], lo, hi);
    sc = mfma32(lo, q[2 * kk], sc);
    sc = mfma32(hi, q[2 * kk + 1], sc);
  }
  return sc;
}

// keep: the rows that this lane's column attends, from row 4 h on.
__device__ __forceinline__ void mask_scores(f32x16& sc, uint32_t keep) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!(keep >> (8 * (i >> 2) + (i & 3)) & 1)) sc[i] = -INFINITY;
}

// A masked row's weight is 0, but 0 times NaN is NaN, and a masked row may hold
// anything: a masked strip's NaN codes are taken out of V, and where there are any
// a second product counts those that each column attends, and puts the NaN back.
template <int D>
__device__ __forceinline__ void mend_values(Tile<D>& c, Codes<D>& x, uint32_t keep, int m32) {
  uint32_t seen = 0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int w = 0; w < Codes<D>::VW; ++w) {
#pragma unroll
      for (int j = 0; j < 8; ++j) seen |= nan_codes(x.v[s][w][j]);
    }
  }
  if (__ballot(seen != 0) == 0) return;
#pragma unroll
  for (int w = 0; w < Codes<D>::VW; ++w) {
    f32x16 count[4] = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t one[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t n = nan_codes(x.v[s][w][j]) >> 7;
        one[j] = n * 0x38u;      // the code of 1
        x.v[s][w][j] &= ~(n * 0xffu);
      }
      u32x4 pa;   // 1 where the column attends the row
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t k = keep >> (16 * s + 8 * (e >> 1) + 2 * (e & 1));
        pa[e] = (k & 1 ? 0x3f80u : 0u) | (k & 2 ? 0x3f800000u : 0u);
      }
      bf16x8_t vt[4];
      step_tiles<D>(one, vt, m32);
#pragma unroll
      for (int i = 0; i < (D == 64 ? 2 : 4); ++i) count[i] = mfma32(vt[i], as_bf16x8(pa), count[i]);
    }
#pragma unroll
    for (int i = 0; i < (D == 64 ? 2 : 4); ++i) {
#pragma unroll
      for (int j = 0; j < 16; ++j)   // count is 0 or at least 1
        c.o[4 * w + i][j] = __uint_as_float(__float_as_uint(c.o[4 * w + i][j]) |
                                            ((0u - min(__float_as_uint(count[i][j]), 1u)) & 0x7fc00000u));
    }
  }
}

// Scores to weights p[step]. The V scales go into the exponents, and out of the
// weights' sums again. A weight is rounded to bf16 once (half a step, 2^-8 of it, at
// random); the sums are taken of the rounded ones, in fp32, so that they add up to 1.
// The sum of two bf16, as the decode takes, would leave the outputs' own rounding alone:
// their error against 64 bits, one / two, 0.00169/0.00161 of their size over 20 rows,
// 0.00159/0.00156 over 100, 0.00155/0.00154 over 612, the same over 4000. It takes 48
// instructions a strip more: 8 tokens after 612 rows 10.4/10.9 us, 32 requests of 8 after 1000
// 17.4/18.3, after 8000 99.7/100.7, 8 of 16 36.6/40.3; in the walk of wide trees 8 of 120
// after 16384 196/246. As a branch for short requests it costs the others 5-16%.
template <int D>
__device__ __forceinline__ void make_weights(u32x4 (&p)[2], Tile<D>& c, const f32x16& sc, const Scales& x) {
  float ta = sc[0], tb = sc[8];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    ta = fmaxf(ta, sc[i]);
    tb = fmaxf(tb, sc[8 + i]);
  }
  const float top = half_max(fmaxf(ta * x.ka, tb * x.kb));
  // the reference maximum moves only when a row exceeds it by 2^8
  if (__ballot(top > c.m + kLazyLog2)) {
    const float mn = fmaxf(c.m, top);
    const float alpha = c.m == -INFINITY ? 0.f : fast_exp2(c.m - mn);
    c.m = mn;
    c.l *= alpha;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) c.o[i] *= alpha;
  }
  const float ref = c.m == -INFINITY ? 0.f : c.m;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float k = s ? x.kb : x.ka, r = (s ? x.eb : x.ea) - ref;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[s][i] = pack_bf16x2(fast_exp2(fmaf(sc[8 * s + 2 * i], k, r)), fast_exp2(fmaf(sc[8 * s + 2 * i + 1], k, r)));
      sum = add_pair(p[s][i], sum);
    }
    c.l = fmaf(sum, s ? x.ib : x.ia, c.l);
  }
}

template <int D>
__device__ __forceinline__ void add_values(Tile<D>& c, const Codes<D>& x, const u32x4 (&p)[2], int m32) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int w = 0; w < Codes<D>::VW; ++w) {
      bf16x8_t vt[4];
      step_tiles<D>(x.v[s][w], vt, m32);
#pragma unroll
      for (int i = 0; i < (D == 64 ? 2 : 4); ++i) c.o[4 * w + i] = mfma32(vt[i], as_bf16x8(p[s]), c.o[4 * w + i]);
    }
  }
}

template <int D>
__global__ __launch_bounds__(64 * kWaves<D>, 1) void gqa_tree_paged_fp8_kernel(PagedFp8 c, TreeArgs a) {
  constexpr int kStride = kAccStride<D>, kThreads = 64 * kWaves<D>;
  extern __shared__ __attribute__((aligned(16))) unsigned char s_dyn[];
  float* s_acc = reinterpret_cast<float*>(s_dyn);             // [kWaves][kTile][kStride]
  float* s_ml = s_acc + kWaves<D> * kTile * kStride;          // [kWaves][kTile][2]
  int* s_pre = reinterpret_cast<int*>(s_ml + kWaves<D> * kTile * 2);   // [B + 1]
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m32 = lane & 31, hf = lane >> 5;

  int u, u1, index = 0;
  if (a.part == nullptr) {
    u = blockIdx.x;       // (request, KV head, first item) here
    u1 = u + 1;
    index = u % a.chunks;
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
      kvh = u / a.chunks % c.Hkv;
      b = u / a.chunks / c.Hkv;
      s = shape_of<D>(a, b);
      if (index >= item_count(s)) return;
      it = item_at<D>(s, index);
      index += a.chunks;
      i0 = 0;
      i1 = it.units;
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
    const int lg = lanes_log2(it.tiles);
    const int lanes = 1 << lg, rows = (32 * kWaves<D>) >> lg;               // keys of a unit
    const int cols = s.n * a.group;                                         // the request's
    const int tile = it.tile0 + (wave & (lanes - 1));
    const bool mine = (wave & (lanes - 1)) < it.tiles && tile * kTile < cols;

    // this lane's column; past the last: its copy, not stored
    const int y0 = min(tile * kTile + m32, cols - 1), tok0 = y0 / a.group;
    const uint32_t* words = a.mask + static_cast<size_t>(s.q0 + tok0) * a.words32;
    bf16x8_t q[D / 16];
    {
      const bf16* src = a.q + static_cast<size_t>(s.q0 + tok0) * a.q_stride + static_cast<size_t>(kvh * a.group + y0 - tok0 * a.group) * D + 16 * hf;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) q[i] = as_bf16x8(ld16(src + 32 * (i >> 1) + 8 * (i & 1)));
    }
    Tile<D> col;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) col.o[i] = f32x16{};
    col.m = -INFINITY;
    col.l = 0.f;

    // strips of this wave: row0 + rows * n, n < ns
    const int row0 = i0 * rows + 32 * (wave >> lg);
    const int end = min(i1 * rows, s.len);
    const int ns = mine && row0 < end ? (end - row0 + rows - 1) / rows : 0;
    const int blk_end = (end + kScaleRows - 1) / kScaleRows;
    const int open = min(end, s.base);        // rows that every column attends
    for (int n0 = 0; n0 < ns; n0 += 32) {
      // lane l holds block l % 2 of strip n0 + l / 2
      const int blk = (row0 + (n0 + (lane >> 1)) * rows) / kScaleRows + (lane & 1);
      // without branches, at whose ends the loads would be waited for
      BlockRef ref;
      {
        const int at = min(blk, blk_end - 1), p = at / c.page_blocks;
        const int page = c.table[static_cast<size_t>(b) * c.max_pages + p];
        ref.bid = blk < blk_end && page >= 0 && page < c.num_pages ? (page * c.Hkv + kvh) * c.page_blocks + at - p * c.page_blocks : -1;
        ref.ks = c.k_scale[max(ref.bid, 0)];
        ref.vs = c.v_scale[max(ref.bid, 0)];
      }
      const int n1 = min(ns - n0, 32);
      Codes<D> x;
      auto bid = [&](int n, int i) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(ref.bid, (2 * n + i) & 63); };
      auto next_k = [&](int n) __attribute__((always_inline)) {
        if (n < n1) load_k<D>(x, c.k_pages, bid(n, 0), bid(n, 1), m32, hf);
      };
      auto next_v = [&](int n) __attribute__((always_inline)) {
        if (n < n1) load_v<D>(x, c.v_pages, bid(n, 0), bid(n, 1), m32, hf);
      };
      next_k(0);
      next_v(0);
      __builtin_amdgcn_sched_barrier(0);      // the codes do not wait for the scales
      // within its range, which leaves a scale as it is: a block that no token attends may
      // hold any (NaN too), and -inf times 0 or NaN would not mask its rows
      const float my_k = fminf(fmaxf(ref.ks, kMinScale), kMaxScale) * a.scale_log2;
      const int my_e = held_exp(ref.vs);
      const float my_ef = static_cast<float>(my_e), my_i = pow2f(-my_e);
      auto scales = [&](int n) __attribute__((always_inline)) {
        Scales r;
        r.ka = readlane_f(my_k, 2 * n);
        r.kb = readlane_f(my_k, 2 * n + 1);
        r.ea = readlane_f(my_ef, 2 * n);
        r.eb = readlane_f(my_ef, 2 * n + 1);
        r.ia = readlane_f(my_i, 2 * n);
        r.ib = readlane_f(my_i, 2 * n + 1);
        return r;
      };
      // the strips whose rows all columns attend, then the others
      const bool hole = __ballot(blk < blk_end && ref.bid < 0) != 0;
      const int plain = hole ? 0 : min(n1, max(0, open - row0 - n0 * rows + rows - 32) / rows);
      u32x4 p[2];
      int n = 0;
      for (; n < plain; ++n) {
        const f32x16 sc = make_scores<D>(x, q);
        __builtin_amdgcn_sched_barrier(0);
        next_k(n + 1);
        __builtin_amdgcn_sched_barrier(0);
        make_weights<D>(p, col, sc, scales(n));
        add_values<D>(col, x, p, m32);
        __builtin_amdgcn_sched_barrier(0);
        next_v(n + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      for (; n < n1; ++n) {
        const int row = row0 + (n0 + n) * rows;
        const uint32_t held = (bid(n, 0) >= 0 ? 0xffffu : 0u) | (bid(n, 1) >= 0 ? 0xffff0000u : 0u);
        const uint32_t keep = (tree_rows(words, a.words32, row, s.base, end) & held) >> (4 * hf);
        f32x16 sc = make_scores<D>(x, q);
        next_k(n + 1);
        mask_scores(sc, keep);
        mend_values<D>(col, x, keep, m32);
        make_weights<D>(p, col, sc, scales(n));
        add_values<D>(col, x, p, m32);
        next_v(n + 1);
      }
    }

    // ---- the waves' results meet ------------------------------------------
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));      // places in LDS are made here, not held over the strips
    __syncthreads();   // the item before has been read
    {
      const float l = half_sum(col.l);
      float* row = s_acc + (wave * kTile + m32) * kStride;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int m = 8 * (i >> 2) + 4 * hf + (i & 3);
        if constexpr (D == 64) {
          if (i < 8) *reinterpret_cast<f32x4*>(row + 4 * m) = f32x4{col.o[0][i], col.o[0][i + 8], col.o[1][i], col.o[1][i + 8]};
        } else {
#pragma unroll
          for (int w = 0; w < D / 128; ++w)
            *reinterpret_cast<f32x4*>(row + (D / 32) * m + 4 * w) =
                f32x4{col.o[4 * w][i], col.o[4 * w + 1][i], col.o[4 * w + 2][i], col.o[4 * w + 3][i]};
        }
      }
      if (hf == 0) {
        s_ml[(wave * kTile + m32) * 2] = col.m;
        s_ml[(wave * kTile + m32) * 2 + 1] = l;
      }
    }
    __syncthreads();
    const bool whole = i0 == 0 && i1 == it.units;
    float* rec = a.part + (static_cast<size_t>(blockIdx.x) * 2 + (i0 == 0 ? 1 : 0)) * a.rec_cols * (D + kRecTail);
    const int here = min(kTile * it.tiles, cols - kTile * it.tile0);      // columns of the item
    // a column's results are those of waves x / kTile + i * lanes; the loads of all go out
    // together (one after the other they took 2.6 us of 14.4, D = 256, 32 columns)
    auto join = [&](auto parts) __attribute__((always_inline)) {
      constexpr int N = decltype(parts)::value;
      for (int idx = tid; idx < here * (D / 4); idx += kThreads) {
        const int x = idx / (D / 4), d = idx % (D / 4) * 4;
        f32x2 ml[N];
        f32x4 v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int slot = x + i * lanes * kTile;
          ml[i] = *reinterpret_cast<const f32x2*>(s_ml + slot * 2);
          v[i] = *reinterpret_cast<const f32x4*>(s_acc + slot * kStride + d);
        }
        float M = ml[0][0], L = 0.f;
#pragma unroll
        for (int i = 1; i < N; ++i) M = fmaxf(M, ml[i][0]);
        f32x4 A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float f = ml[i][0] == -INFINITY ? 0.f : fast_exp2(ml[i][0] - M);
          A += f * v[i];
          L += f * ml[i][1];
        }
        if (whole) {
          const int y = kTile * it.tile0 + x, tok = y / a.group;
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
    };
    if (lg == 0) join(std::integral_constant<int, kWaves<D>>{});
    else if (lg == 1) join(std::integral_constant<int, kWaves<D> / 2>{});
    else if (lg == 2) join(std::integral_constant<int, kWaves<D> / 4>{});
    else join(std::integral_constant<int, 1>{});
  }
}

// The records of column y of a request and KV head that several workgroups walked:
// those of the workgroups w0 .. w1, none if one wrote the output.
struct Records { const float* at; int w0, w1; };
template <int D>
__device__ __forceinline__ Records records_of(const PagedFp8& c, const TreeArgs& a, const Shape& s, int b, int kvh, int y, int launched) {
  const int index = min(y / (kTile * kWaves<D>), s.full);
  const Item it = item_at<D>(s, index + (index == s.full && s.half > 0 && y >= kTile * (s.full * kWaves<D> + s.half) ? 1 : 0));
  const int before = a.units[b], units = a.units[a.B] * c.Hkv, groups = min(launched, units);
  const int first = before * c.Hkv + kvh * (a.units[b + 1] - before) + it.before;
  // workgroup w holds unit x: the largest w with w U / W < x + 1
  return Records{a.part + static_cast<size_t>(y - kTile * it.tile0) * (D + kRecTail),
                 static_cast<int>((static_cast<long>(first + 1) * groups - 1) / units),
                 static_cast<int>((static_cast<long>(first + it.units) * groups - 1) / units)};
}

// A thread's running sum over records.
struct Joined {
  f32x4 A = {0.f, 0.f, 0.f, 0.f};
  float M = -INFINITY, L = 0.f;
  __device__ __forceinline__ void add(const f32x4& v, float m, float l) {
    const float mn = fmaxf(M, m);
    const float fo = M == -INFINITY ? 0.f : fast_exp2(M - mn), fn = m == -INFINITY ? 0.f : fast_exp2(m - mn);
    A = A * fo + v * fn;
    L = L * fo + l * fn;
    M = mn;
  }
};
template <int D>
__device__ __forceinline__ void store_joined(const TreeArgs& a, const Shape& s, int kvh, int y, int d, const Joined& x) {
  const float inv = x.L == 0.f ? 0.f : 1.0f / x.L;
  const int tok = y / a.group;
  *reinterpret_cast<u32x2*>(a.out + (static_cast<size_t>(s.q0 + tok) * a.Hq + kvh * a.group + y - tok * a.group) * D + d) =
      u32x2{pack_bf16x2(x.A[0] * inv, x.A[1] * inv), pack_bf16x2(x.A[2] * inv, x.A[3] * inv)};
}

// Joins the records: o = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i. Few
// columns, many records each: a workgroup takes one column of a request and KV head,
// its threads other records, kBatch at a time (past the last: the last again, with
// weight 0).
constexpr int kMergeThreads = 256, kBatch = 4;
template <int D>
__device__ __forceinline__ void join_batch(Joined* sum, const float* at, const Records& r, int w, int stride, size_t step, int d) {
  f32x4 v[kBatch];
  float m[kBatch], l[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int u = min(w + i * stride, r.w1);
    const float* p = at + (static_cast<size_t>(u) * 2 + (u == r.w0 ? 1 : 0)) * step;
    v[i] = *reinterpret_cast<const f32x4*>(p + d);
    m[i] = p[D];
    l[i] = p[D + 1];
  }
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (w + i * stride <= r.w1) sum->add(v[i], m[i], l[i]);
}
template <int D>
__global__ __launch_bounds__(kMergeThreads) void gqa_tree_paged_fp8_merge_kernel(PagedFp8 c, TreeArgs a, int launched) {
  constexpr int kQuads = D / 4, kPhases = kMergeThreads / kQuads;
  __shared__ f32x4 s_a[kMergeThreads];
  __shared__ float s_m[kMergeThreads], s_l[kMergeThreads];
  const int b = blockIdx.y, kvh = blockIdx.x, y = blockIdx.z;
  const Shape s = shape_of<D>(a, b);
  if (y >= s.n * a.group) return;
  const int d = static_cast<int>(threadIdx.x) % kQuads * 4, ph = static_cast<int>(threadIdx.x) / kQuads;
  const Records r = records_of<D>(c, a, s, b, kvh, y, launched);
  if (r.w0 == r.w1) return;
  const size_t step = static_cast<size_t>(a.rec_cols) * (D + kRecTail);
  Joined sum;
  for (int w = r.w0 + ph; w <= r.w1; w += kBatch * kPhases) join_batch<D>(&sum, r.at, r, w, kPhases, step, d);
  s_a[threadIdx.x] = sum.A;
  s_m[threadIdx.x] = sum.M;
  s_l[threadIdx.x] = sum.L;
  __syncthreads();
  if (ph > 0) return;
#pragma unroll
  for (int i = 1; i < kPhases; ++i) {
    const int j = threadIdx.x + i * kQuads;
    sum.add(s_a[j], s_m[j], s_l[j]);
  }
  store_joined<D>(a, s, kvh, y, d, sum);
}

// The same for many columns, few records each: a workgroup takes as many columns as it
// has threads for, and then those gridDim.z times as many further on.
template <int D>
__global__ __launch_bounds__(kMergeThreads) void gqa_tree_paged_fp8_merge_few_kernel(PagedFp8 c, TreeArgs a, int launched) {
  constexpr int kQuads = D / 4, kColumns = kMergeThreads / kQuads;
  const int b = blockIdx.y, kvh = blockIdx.x;
  const Shape s = shape_of<D>(a, b);
  const int cols = s.n * a.group, d = static_cast<int>(threadIdx.x) % kQuads * 4, mine = static_cast<int>(threadIdx.x) / kQuads;
  const size_t step = static_cast<size_t>(a.rec_cols) * (D + kRecTail);
  for (int x0 = static_cast<int>(blockIdx.z) * kColumns; x0 < cols; x0 += static_cast<int>(gridDim.z) * kColumns) {
    const Records r = records_of<D>(c, a, s, b, kvh, x0, launched);      // the columns are one item's
    if (r.w0 == r.w1) continue;
    const int x = min(mine, cols - 1 - x0);
    Joined sum;
    for (int w = r.w0; w <= r.w1; w += kBatch) join_batch<D>(&sum, r.at + x * (D + kRecTail), r, w, 1, step, d);
    if (mine < cols - x0) store_joined<D>(a, s, kvh, x0 + x, d, sum);
  }
}

// The most that a request may have: columns, column tiles, items of a KV head.
struct Most { long cols; int items, rec_cols; };
template <int D>
Most most_of(int T, int words, int group) {
  Most m;
  m.cols = static_cast<long>(std::min<long>(T, 64L * words)) * group;
  const long tiles = (m.cols + kTile - 1) / kTile;
  m.items = static_cast<int>(tiles / kWaves<D> + 2);    // of the rest, two at most
  m.rec_cols = static_cast<int>(kTile * std::min<long>(tiles, kWaves<D>));
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

// Whether a request and KV head is one workgroup's, for all keys: up to a length that
// grows with the CUs they fill, and is shared by the tiles of a request (of average
// size), since a workgroup's waves that have no tile take other keys. us in a graph, whole
// / split, lengths between half the bound and all of it, trees of up to 4 tokens (16: in
// parentheses), G = 4. D = 128, 8 KV heads: 1 request of 600 rows 10.3/12.2 (15.3/14.1), 1000
// 12.3/12.5 (18.7/14.4), 2000 17.0/12.5 (27.8/15.8); 4 of 1000 12.5/12.8 (19.0/17.0), 1500
// 14.7/13.1 (23.5/23.7); 8 of 1500 15.6/19.8 (24.3/23.8), 3000 23.0/22.5 (38.4/26.5); 16 of
// 2000 18.8/23.0 (30.1/29.6), 3000 23.4/25.6 (39.4/32.8). D = 64: 1 of 1000 9.5/11.4
// (14.0/12.7), 2000 13.2/11.6 (21.1/13.4); 8 of 2000 13.4/16.3 (21.4/18.9). D = 256, 4 heads:
// 1 of 200 11.8/13.1 (18.1/16.0), 400 14.7/13.2 (22.8/16.7); 8 of 400 15.0/13.8 (23.1/21.7),
// 800 19.2/15.0 (31.7/28.7); 16 of 800 20.2/22.1 (32.9/33.1), 2000 33.7/26.7 (60.5/36.8).
bool walks_whole(long columns, int B, int Hkv, int max_len, int D) {
  const long items = static_cast<long>(B) * Hkv, tiles = (columns + 32L * B - 1) / (32L * B);
  const long most = D == 256 ? 300 + items * items / 5 : (D == 128 ? 1000 : 1500) + items * items * 3 / 10;
  return max_len <= (D == 256 ? 2048 : 4096) && max_len * std::min<long>(tiles, D == 256 ? 4 : 8) <= most;
}

// Records of a column, where requests share evenly, from which a workgroup joins one
// column's. us, the whole call, columns by columns / each, 8000 rows (30000: in
// parentheses), all columns of a KV head. 1 request, D = 256, 4 heads: 4 26.2/16.7
// (33.8/23.8), 64 35.1/24.8 (45.0/34.9); 2: 52 33.4/27.7 (44.4/38.2); 8: 332 48.1/46.8, 676
// 68.8/67.9; 32: 128 91.8/94.6, 272 95.1/104.4. D = 128, 8 heads: 1: 4 18.4/13.2 (26.3/21.2),
// 128 28.7/24.3 (44.1/39.1); 4: 92 27.2/26.5, 192 31.3/32.1, 388 40.8/43.0; 8: 36 28.7/27.8,
// 160 31.8/34.3; 32: 128 92.6/104.5. D = 64: 1: 4 16.3/11.9, 128 23.9/19.3; 4: 92 20.8/20.2,
// 192 23.9/24.9; 32: 128 56.7/68.2.
// Up to 1024 columns of all heads, D = 256 (a quarter of the phases, so less to meet) 4096.
constexpr int kEachRecords = 8;

template <int D>
int launch(const PagedFp8& c, TreeArgs a, int words, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Most m = most_of<D>(a.T, words, a.group);
  // a workgroup for each item that a request of average size has
  a.chunks = static_cast<int>(std::min<long>(m.items, (static_cast<long>(a.T) * a.group + 32L * kWaves<D> * a.B - 1) / (32L * kWaves<D> * a.B)));
  a.rec_cols = m.rec_cols;
  constexpr int kThreads = 64 * kWaves<D>;
  const long items = static_cast<long>(a.B) * c.Hkv * m.items;
  AILA_REQUIRE(items * most_units(a.max_len) < (1L << 31) && items * kThreads < (1L << 32),
               "gqa_tree_paged_fp8: B=%d requests of up to %ld query rows and %d keys are too many", a.B, m.cols, a.max_len);
  const long joins = (m.cols * (D / 4) + kMergeThreads - 1) / kMergeThreads;      // workgroups of a request and KV head
  AILA_REQUIRE(joins <= 65535, "gqa_tree_paged_fp8: %ld query rows of a KV head are too many", m.cols);
  // fewer than 2^32 threads, the most of a launch
  const long few = std::min(joins, ((1L << 32) - 1) / kMergeThreads / (static_cast<long>(a.B) * c.Hkv));
  long groups = static_cast<long>(a.B) * c.Hkv * a.chunks;
  if (workspace != nullptr) {
    const size_t rec = record_bytes<D>(m);
    if (workspace_bytes < units_bytes(a.B) + 2 * rec)
      return set_error(AILA_HIP_EWORKSPACE, "gqa_tree_paged_fp8: workspace %zu bytes, %zu are the least", workspace_bytes,
                       units_bytes(a.B) + 2 * rec);
    if (!walks_whole(static_cast<long>(a.T) * a.group, a.B, c.Hkv, a.max_len, D)) {
      groups = std::min<long>(split_groups<D>(a.B, c.Hkv, m, a.max_len), static_cast<long>((workspace_bytes - units_bytes(a.B)) / rec));
      a.units = static_cast<int*>(workspace);
      a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + units_bytes(a.B));
    }
  }
  const size_t lds = static_cast<size_t>(kWaves<D>) * kTile * (kAccStride<D> + 2) * sizeof(float) +
                     (a.part ? static_cast<size_t>(a.B + 1) * sizeof(int) : 0);
  hipLaunchKernelGGL((gqa_tree_paged_fp8_kernel<D>), dim3(groups), dim3(kThreads), lds, st, c, a);
  const long all = static_cast<long>(a.T) * a.group * c.Hkv;      // columns
  const bool each = kEachRecords * a.B * c.Hkv <= kCus && all <= (D == 256 ? 4096 : 1024);
  if (a.part && each)
    hipLaunchKernelGGL((gqa_tree_paged_fp8_merge_kernel<D>), dim3(c.Hkv, a.B, m.cols), dim3(kMergeThreads), 0, st, c, a,
                       static_cast<int>(groups));
  else if (a.part)
    hipLaunchKernelGGL((gqa_tree_paged_fp8_merge_few_kernel<D>), dim3(c.Hkv, a.B, few), dim3(kMergeThreads), 0, st, c, a,
                       static_cast<int>(groups));
  return check_launch("gqa_tree_paged_fp8");
}

// Wide trees walk as prompts do, 128 columns a workgroup with their codes converted
// once in LDS (gqa_prefill_paged_fp8.hip): from some columns a request on, which the
// host knows on average, and the more of them the fewer requests share the device.
// us, here split / as prompts, trees of up to 16, 32, 64, 128 columns (two thirds of it
// on average where there are more than one), 8000 rows. D = 128: 1 request 14/23, 16/23,
// 19/24, 25/26; 2 19/24, 22/24, 27/25, 35/29; 4 24/32, 27/32, 31/35, 41/38; 8 30/44, 32/44,
// 37/47, 53/50; 32 97/138, 100/133, 123/136, 173/149. D = 64: 1 12/18, 13/18, 16/19, 19/20; 2
// 16/19, 18/19, 21/20, 26/22; 8 23/35, 23/35, 28/36, 39/38; 32 57/101, 58/95, 77/97,
// 119/100. D = 256: 1 19/27, 21/27, 25/29, 33/32; 2 24/28, 28/28, 35/30, 45/36; 4 28/32,
// 32/33, 37/36, 53/43; 8 33/44, 36/45, 48/49, 70/56; 32 95/129, 100/133, 128/132, 188/144.
// (One request of D = 256, whose records are joined a column each, keeps to itself longer.)
// But not if requests that fill the device are short for their columns: each is one
// workgroup's here then. us, here whole / as prompts, of up to 500, 1000, 2000, 4000 rows.
// D = 128, 8 heads: 16 requests of up to 128 columns 22/27, 31/34, 50/40, 85/53; 32 23/40,
// 33/46, 52/60, 101/90; 32 of up to 256 columns 39/51, 58/64, 96/85, 175/137. D = 64: 32 of
// 256 28/38, 43/48, 72/62, 127/92. D = 256, 4 heads: 32 of 64 27/35, 38/41, 61/54, 120/84.
bool walks_as_prompt(int T, int B, int Hkv, int group, int words, int max_len, int D) {
  const long columns = static_cast<long>(T) * group;
  const long each = D == 64 ? 62 : D == 128 ? 54 : 40, more = D == 64 ? 80 : D == 128 ? 60 : B == 1 ? 70 : 10;
  if (columns <= each * B + more) return false;
  if (static_cast<double>(max_len) * columns <= (D == 64 ? 800.0 : D == 128 ? 700.0 : 250.0) * B * B * Hkv) return false;
  // its line of key tiles and its merge's threads have to fit
  const long tiles = (std::min<long>(T, 64L * words) * group + 127) / 128 * B;
  return tiles * (max_len / 32 + 16) < (1L << 31) && tiles * Hkv * 8 * 256 < (1L << 32);
}

}  // namespace
}  // namespace aila

extern "C" size_t aila_hip_gqa_tree_paged_fp8_workspace_size(int T, int B, int Hq, int Hkv, int D, int max_len,
                                                             int mask_words) {
  using namespace aila;
  if (T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_len < 0 || mask_words <= 0) return 0;
  if (D != 64 && D != 128 && D != 256) return 0;
  // enough for fewer tokens too, which may take the other walk
  const size_t wide = walks_as_prompt(T, B, Hkv, Hq / Hkv, mask_words, max_len, D) ? tree_as_prefill_workspace(D, B, Hkv) : 0;
  switch (D) {
    case 64: return std::max(wide, workspace_need<64>(T, B, Hkv, Hq / Hkv, mask_words, max_len));
    case 128: return std::max(wide, workspace_need<128>(T, B, Hkv, Hq / Hkv, mask_words, max_len));
    default: return std::max(wide, workspace_need<256>(T, B, Hkv, Hq / Hkv, mask_words, max_len));
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
  if (walks_as_prompt(T, B, Hkv, Hq / Hkv, mask_words, max_len, D) && workspace != nullptr && workspace_bytes >= tree_as_prefill_workspace(D, B, Hkv))
    return tree_as_prefill(D, c, TreeCall{a.q, q_stride, a.out, a.mask, a.words32, query_start, seq_lens, T, B, Hq, max_len, workspace}, st);
  switch (D) {
    case 64: return launch<64>(c, a, mask_words, workspace, workspace_bytes, st);
    case 128: return launch<128>(c, a, mask_words, workspace, workspace_bytes, st);
    default: return launch<256>(c, a, mask_words, workspace, workspace_bytes, st);
  }
}
