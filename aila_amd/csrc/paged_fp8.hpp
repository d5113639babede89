// The 8-bit paged KV cache: e4m3 (OCP) codes in pages [P, Hkv, page_size, D]
// and a scale for each block of 16 rows and head, [P, Hkv, page_size / 16]
// fp32, always a power of two. Block `bid` = (page * Hkv + head) * (page_size /
// 16) + row / 16 is 16 * D contiguous codes and one scale.
//
// Powers of two, because a block is filled over many decode steps: when a new
// row outgrows the scale, the rows before it are requantised, and a code times
// a power of two is again a code (but for underflow), so no row is rounded
// twice. They also make every dequantised value exact in bf16 (4 significant
// bits), which is what the matrix instructions take.
#pragma once

#include "common.hpp"

namespace aila {

constexpr int kScaleRows = 16;
// Exponents of a scale: the smallest e with amax <= 448 * 2^e, bounded so that
// 448 * 2^e stays finite and the smallest code times it stays a normal bf16.
constexpr int kMinScaleExp = -100, kMaxScaleExp = 119;
constexpr float kMinScale = 0x1p-100f, kMaxScale = 0x1p119f;
constexpr float kE4m3Max = 448.0f;

// 2^e in fp32; 0 below its normal range.
__device__ __forceinline__ float pow2f(int e) {
  return e < -126 ? 0.0f : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Two codes (the low or the high half of w) as a pair of bf16, exact.
template <bool HI>
__device__ __forceinline__ uint32_t fp8x2_to_bf16x2(uint32_t w, float scale = 1.0f) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// 16 bytes of codes -> two MFMA operands of 8 bf16.
__device__ __forceinline__ void fp8x16_to_bf16(const u32x4& w, bf16x8_t& lo, bf16x8_t& hi) {
  lo = as_bf16x8(u32x4{fp8x2_to_bf16x2<false>(w[0]), fp8x2_to_bf16x2<true>(w[0]), fp8x2_to_bf16x2<false>(w[1]),
                       fp8x2_to_bf16x2<true>(w[1])});
  hi = as_bf16x8(u32x4{fp8x2_to_bf16x2<false>(w[2]), fp8x2_to_bf16x2<true>(w[2]), fp8x2_to_bf16x2<false>(w[3]),
                       fp8x2_to_bf16x2<true>(w[3])});
}

// Exponent of a block's scale.
__device__ __forceinline__ int held_exp(float scale) {
  return min(max(static_cast<int>(__float_as_uint(scale) >> 23 & 0xff) - 127, kMinScaleExp), kMaxScaleExp);
}

// x * 2^-e as a value to be rounded to e4m3: saturated (at kMaxScaleExp alone
// a finite x exceeds 448), NaN for what is not finite (e4m3 has no infinity).
__device__ __forceinline__ float to_code_range(float x, float inv) {
  const float y = fminf(fmaxf(x * inv, -kE4m3Max), kE4m3Max);
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : y;
}

__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

template <int CTRL>
__device__ __forceinline__ int dpp_i(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xF, 0xF, false);
}
// Maximum of the wave's values, in every lane.
__device__ __forceinline__ int wave_max(int x) {
  x = max(x, dpp_i<kDppQuadXor1>(x));
  x = max(x, dpp_i<kDppQuadXor2>(x));
  x = max(x, dpp_i<kDppRowHalfMirror>(x));
  x = max(x, dpp_i<kDppRowMirror>(x));
  const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max(static_cast<int>(a[0]), static_cast<int>(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max(static_cast<int>(b[0]), static_cast<int>(b[1]));
}

// ---- of the walks on 32x32 products --------------------------------------------
__device__ __forceinline__ f32x16 mfma32(const bf16x8_t& a, const bf16x8_t& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Max / sum over lanes l and l ^ 32.
__device__ __forceinline__ float half_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// acc + the two bf16 of x.
__device__ __forceinline__ float add_pair(uint32_t x, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc, false);
}

// What the attention kernels are given of the cache and its tables.
struct PagedFp8 {
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* k_scale;
  const float* v_scale;
  const int* table;      // [B, max_pages]
  int max_pages, num_pages, Hkv;
  int page_blocks;       // page_size / 16
};

int check_paged_fp8(const char* what, const void* k_pages, const void* v_pages, const float* k_scale,
                    const float* v_scale, int Hkv, int D, int page_size, int num_pages);

// A block of a sequence as a lane looks it up: its index in the pool (-1: the
// table holds no page for it, or it is past the rows looked at) and its scales.
struct BlockRef {
  int bid;
  float ks, vs;
};
// Index of a sequence's block in the pool; -1: its table entry is no page.
__device__ __forceinline__ int block_id(const PagedFp8& c, int b, int head, int blk) {
  const int p = blk / c.page_blocks;
  const int page = c.table[static_cast<size_t>(b) * c.max_pages + p];
  return page >= 0 && page < c.num_pages ? (page * c.Hkv + head) * c.page_blocks + blk - p * c.page_blocks : -1;
}
__device__ __forceinline__ BlockRef block_ref(const PagedFp8& c, int b, int head, int blk, int blk_end) {
  BlockRef r{-1, 0.f, 0.f};
  if (blk < blk_end) r.bid = block_id(c, b, head, blk);
  if (r.bid >= 0) {
    r.ks = c.k_scale[r.bid];
    r.vs = c.v_scale[r.bid];
  }
  return r;
}

// One strip: two blocks of 16 rows, as a wave holds it. Orientation of the
// products (both on v_mfma_f32_16x16x32_bf16, whose A and B operands have the
// same lane layout):
//   S^T = K Q^T    A = 16 rows of K, B = 16 query rows (columns)
//     lane (m, g) = (l % 16, l / 16) loads 16 codes of row m at 64 kk + 16 g, two
//     operands of 8 dims; it receives rows 4g + j of column m.
//   O^T += V^T P^T A = 16 head dims of V, B = P of 32 rows
//     lane (m, g) holds the scores of column m for rows 4g + j of both blocks,
//     which are the 8 k-slots it has to supply: P never leaves its registers. It
//     loads those rows' dims [D/16 m, D/16 (m + 1)), neighbouring lanes one row
//     side by side, and pairs the rows' bytes with v_perm: dim t of each lane's
//     run makes the A operand of tile t, whose row m is head dim D/16 m + t.
template <int D>
struct Strip {
  static constexpr int KK = D / 64;
  static constexpr int VW = D / 64;        // words of a lane's run of dims
  u32x4 k[2][KK];
  uint32_t v[8][VW];
};

// Buffer loads, each block a buffer of its own: one that has no page (bid < 0)
// has no bytes, and its loads return zeros without going to memory, so a
// pipeline of strips needs no branch around its loads.
template <int D, bool NT>
__device__ __forceinline__ void load_strip(Strip<D>& s, const PagedFp8& c, int bid_a, int bid_b, int m16, int g4) {
  constexpr int kAux = NT ? 2 : 0;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int bid = x ? bid_b : bid_a;
    const size_t base = static_cast<size_t>(max(bid, 0)) * (kScaleRows * D);
    const int bytes = bid >= 0 ? kScaleRows * D : 0;
    const __amdgpu_buffer_rsrc_t kr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.k_pages) + base, 0, bytes, kBufferRsrcWord3);
    const __amdgpu_buffer_rsrc_t vr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.v_pages) + base, 0, bytes, kBufferRsrcWord3);
#pragma unroll
    for (int kk = 0; kk < Strip<D>::KK; ++kk)
      s.k[x][kk] = __builtin_amdgcn_raw_buffer_load_b128(kr, m16 * D + 16 * g4 + 64 * kk, 0, kAux);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = (4 * g4 + j) * D + m16 * (D / 16);
      if constexpr (D == 256) {
        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(vr, at, 0, kAux);
#pragma unroll
        for (int i = 0; i < 4; ++i) s.v[4 * x + j][i] = w[i];
      } else if constexpr (D == 128) {
        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vr, at, 0, kAux);
        s.v[4 * x + j][0] = w[0];
        s.v[4 * x + j][1] = w[1];
      } else {
        s.v[4 * x + j][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, at, 0, kAux);
      }
    }
  }
}

// Running softmax of one column (query row) per lane m, and its output.
template <int D>
struct Column {
  f32x4 acc[D / 16];   // acc[t][i]: head dim D/16 (4 g + i) + t of column m
  float m, l;          // maximum (log2 domain) and this lane's part of the sum
};

template <int D>
__device__ __forceinline__ void clear_column(Column<D>& c) {
#pragma unroll
  for (int t = 0; t < D / 16; ++t) c.acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  c.m = -INFINITY;
  c.l = 0.f;
}

// The V operands of word w, both halves: tiles 4w .. 4w + 3.
__device__ __forceinline__ void v_tiles(const uint32_t (&v)[8], bf16x8_t (&t)[4]) {
  u32x4 o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t a = v[2 * e], b = v[2 * e + 1];
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u);   // a0 b0 a1 b1
    const uint32_t hi = __builtin_amdgcn_perm(b, a, 0x07030602u);   // a2 b2 a3 b3
    o[0][e] = fp8x2_to_bf16x2<false>(lo);
    o[1][e] = fp8x2_to_bf16x2<true>(lo);
    o[2][e] = fp8x2_to_bf16x2<false>(hi);
    o[3][e] = fp8x2_to_bf16x2<true>(hi);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = as_bf16x8(o[i]);
}

// One strip into a column's softmax. `row` is the strip's first row; if masked,
// a column attends rows < lim of the blocks that have a page (ok_a, ok_b).
// ka, kb: the K scales times log2(e) / sqrt(D). The V scales go into P, where
// they are exact. P goes in as the sum of two bf16 (16 bits): one
// would double the output's rounding error, and the matrix cores are idle most of
// the time here.
//
// A masked row's P is 0, but 0 times NaN is NaN, and a masked row may hold
// anything. So a masked strip's NaN codes are taken out of V; where there are
// any, a second product counts those that each column attends, and puts the NaN
// back there.
constexpr float kLazyLog2 = 8.0f;

// The bytes of w that are NaN codes (0x7f, 0xff), as 0x80 each.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Takes the NaN codes out of a masked strip's V and puts NaN into the outputs
// of the columns that attend them.
template <int D>
__device__ __forceinline__ void mend_strip(Column<D>& c, Strip<D>& s, int row, int lim, bool ok_a, bool ok_b, int g4) {
  uint32_t seen = 0;
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) seen |= nan_codes(s.v[j][w]);
  }
  if (__ballot(seen != 0) == 0) return;
  u32x4 pa;   // 1 where the column attends the row
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = row + (e < 2 ? 0 : 16) + 4 * g4 + 2 * (e & 1);
    const bool ok = e < 2 ? ok_a : ok_b;
    pa[e] = (ok && r < lim ? 0x3f80u : 0u) | (ok && r + 1 < lim ? 0x3f800000u : 0u);
  }
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
    uint32_t one[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t n = nan_codes(s.v[j][w]) >> 7;
      one[j] = n * 0x38u;      // the code of 1
      s.v[j][w] &= ~(n * 0xffu);
    }
    bf16x8_t t[4];
    v_tiles(one, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 n = mfma16x16x32(t[i], as_bf16x8(pa), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int j = 0; j < 4; ++j)   // n[j] is 0 or at least 1
        c.acc[4 * w + i][j] = __uint_as_float(__float_as_uint(c.acc[4 * w + i][j]) |
                                              ((0u - min(__float_as_uint(n[j]), 1u)) & 0x7fc00000u));
    }
  }
}

template <int D>
__device__ __forceinline__ void strip_step(Column<D>& c, Strip<D>& s, const bf16x8_t (&q)[D / 32], float ka, float kb,
                                           float va, float vb, bool masked, int row, int lim, bool ok_a, bool ok_b, int g4) {
  f32x4 sa = {0.f, 0.f, 0.f, 0.f}, sb = sa;
#pragma unroll
  for (int kk = 0; kk < D / 64; ++kk) {
    bf16x8_t lo, hi;
    fp8x16_to_bf16(s.k[0][kk], lo, hi);
    sa = mfma16x16x32(lo, q[2 * kk], sa);
    sa = mfma16x16x32(hi, q[2 * kk + 1], sa);
    fp8x16_to_bf16(s.k[1][kk], lo, hi);
    sb = mfma16x16x32(lo, q[2 * kk], sb);
    sb = mfma16x16x32(hi, q[2 * kk + 1], sb);
  }
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = sa[j] * ka;
    x[4 + j] = sb[j] * kb;
  }
  if (masked) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!(ok_a && row + 4 * g4 + j < lim)) x[j] = -INFINITY;
      if (!(ok_b && row + 16 + 4 * g4 + j < lim)) x[4 + j] = -INFINITY;
    }
    mend_strip<D>(c, s, row, lim, ok_a, ok_b, g4);
  }
  float top = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
  top = xrow4_max(top);
  // The reference maximum moves only when a row exceeds it by 2^8: until then
  // P <= 2^8 and nothing is lost, and the accumulators need no rescaling.
  if (__ballot(top > c.m + kLazyLog2)) {
    const float mn = fmaxf(c.m, top);
    const float alpha = c.m == -INFINITY ? 0.f : fast_exp2(c.m - mn);
    c.m = mn;
    c.l *= alpha;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) c.acc[t] *= alpha;
  }
  const float ref = c.m == -INFINITY ? 0.f : c.m;
  u32x4 ph, pl;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = fast_exp2(x[j] - ref);
    c.l += x[j];
    x[j] *= j < 4 ? va : vb;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ph[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
    pl[e] = pack_bf16x2(x[2 * e] - __uint_as_float(ph[e] << 16), x[2 * e + 1] - __uint_as_float(ph[e] & 0xffff0000u));
  }
#pragma unroll
  for (int w = 0; w < D / 64; ++w) {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s.v[j][w];
    bf16x8_t t[4];
    v_tiles(v, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c.acc[4 * w + i] = mfma16x16x32(t[i], as_bf16x8(ph), c.acc[4 * w + i]);
      c.acc[4 * w + i] = mfma16x16x32(t[i], as_bf16x8(pl), c.acc[4 * w + i]);
    }
  }
}

// ---- drafted trees ----------------------------------------------------------
// The rows [row, row + 32) that a token attends, as bits: those before the draft
// (row < base), the drafted ones by its mask words, none from len on.
__device__ __forceinline__ uint32_t tree_rows(const uint32_t* words, int words32, int row, int base, int len) {
  const int o = row - base, i = o >> 5, sh = o & 31;
  auto word = [&](int w) __attribute__((always_inline)) -> uint32_t {
    return w < 0 ? ~0u : w < words32 ? words[w] : 0u;
  };
  const uint64_t both = static_cast<uint64_t>(word(i + 1)) << 32 | word(i);
  const uint32_t keep = static_cast<uint32_t>(both >> sh);
  const int left = len - row;
  return left >= 32 ? keep : left > 0 ? keep & ((1u << left) - 1) : 0u;
}

// The tree attention's arguments, for the kernel that walks wide trees as prompts.
struct TreeCall {
  const bf16* q;
  long q_stride;
  bf16* out;
  const uint32_t* mask;
  int words32;
  const int* query_start;
  const int* seq_lens;
  int T, B, Hq, max_len;
  void* workspace;      // of at least tree_as_prefill_workspace bytes
};
size_t tree_as_prefill_workspace(int D, int B, int Hkv);
int tree_as_prefill(int D, const PagedFp8& c, const TreeCall& t, hipStream_t st);

}  // namespace aila
