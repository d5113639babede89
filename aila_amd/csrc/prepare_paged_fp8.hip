// What stands between a layer's fused projection and its attention over the 8-bit
// paged cache, for a ragged batch of tokens: per-head RMSNorm of q and k, rotation
// at each token's own position, k and v quantised into the pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_d, y_{d + rot/2}) turned by p theta^(-2 d / rot), d < rot / 2
//
// in fp32, rounded once: q to bf16, k by the append's rule to e4m3 (the calls
// for the single steps round k to bf16 twice on its way there). An angle is a product in
// fp64 of whole turns, taken modulo 1 there: at position 2^20 an fp32 product is
// off by 2^-4 radians.
//
// A lane holds dims 4 s .. 4 s + 3 of both halves of the rotated part (or of the
// rest), so a pair is never apart, at two 8-byte loads instead of one of 16. The
// cosines and sines of a workgroup's tokens are made once, in LDS, for all its waves.
//
// Many tokens, 8191 of 16 / 4 heads, D = 256 (184 MB): 54.3 us where tokens follow each
// other, 58.8 with gates between the queries, where a large copy takes 38. Queries alone 30
// us for 135 MB = 4.5 TB/s, their vector ALU busy for 84% of it. Rows 25 to 30 us for 50 MB:
// a wave holds a whole block, so a CU has 10 of them, which wait for 45% of their time with
// the vector ALU busy for 56%; loads, arithmetic and stores of a wave's one run follow each
// other. (The append alone takes 14; without the rotation 7 us go.) Few tokens are bound
// by launch and the chain slots -> rows -> codes: 26 tokens, 32 / 8, D = 128, 5.9 us. The rows,
// or a wave's first head, are on their way while the turns are made (26 tokens 6.3 -> 5.9 us,
// 4096 of 32 / 8, D = 128, 25.2 -> 23.9). Rows and queries interleaved in one launch were
// slower (83 us for the 8191 tokens): what stores rows takes longest, and comes last.
#include "paged_fp8.hpp"

#include <type_traits>

namespace aila {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Turns a position of pair j, r^j / (2 pi) with r = theta^(-2 / rot), from powers of r
// that stay in scalar registers.
struct Powers {
  double base;       // 1 / (2 pi)
  double bit[7];     // r, r^2, ..., r^64
};

struct PrepareArgs {
  const bf16 *q, *k, *v;
  long q_stride, q_head_stride, k_stride, v_stride;
  bf16* q_out;
  const bf16 *q_norm, *k_norm;     // null: 1
  uint8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  const int* slots;
  const int *pos_t, *pos_h, *pos_w;     // the same three times: one position
  int section_h, section_w;
  const float* inv_freq;
  int T, tile, Hq, Hkv, page_size, num_slots, rot;
  int kv_groups;       // workgroups that store rows; the others take a token's queries each
  float eps;
};

template <int LR>
__device__ __forceinline__ float row_sum(float x) {
  x += dpp_f<kDppQuadXor1>(x);
  x += dpp_f<kDppQuadXor2>(x);
  x += dpp_f<kDppRowHalfMirror>(x);
  if constexpr (LR >= 16) x += dpp_f<kDppRowMirror>(x);
  if constexpr (LR >= 32) {
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return x;
}

// A lane's place in a row: dims lo .. lo + 3 and hi .. hi + 3, which are turned
// pairwise (pairs j .. j + 3) if `turns`.
struct Place { int lo, hi, j; bool turns; };
template <int D>
__device__ __forceinline__ Place place_of(int s, int rot) {
  const int x = 4 * s, half = rot / 2;
  return x < half ? Place{x, x + half, x, true} : Place{x + half, x + D / 2, 0, false};
}

// (cosine, sine) of x turns, |x| <= 1/2, each rounded once: Taylor's series within an eighth
// of a turn, in fp64 (the first terms left out are below 2^-32 of them). The fp32 functions
// of the angle in fp32 are off by up to 2^-22, which shows in codes next to a border.
__device__ __forceinline__ f32x2 turn_of(double x) {
  const double k = __builtin_rint(4.0 * x);
  const double a = (x - 0.25 * k) * 6.283185307179586, z = a * a;
  double s = -1.0 / 39916800, c = -1.0 / 3628800;
  s = fma(s, z, 1.0 / 362880);
  c = fma(c, z, 1.0 / 40320);
  s = fma(s, z, -1.0 / 5040);
  c = fma(c, z, -1.0 / 720);
  s = fma(s, z, 1.0 / 120);
  c = fma(c, z, 1.0 / 24);
  s = fma(s, z, -1.0 / 6);
  c = fma(c, z, -0.5);
  const float sn = static_cast<float>(fma(a * z, s, a)), cs = static_cast<float>(fma(z, c, 1.0));
  const int q = static_cast<int>(k) & 3;      // quarter turns
  const float u = q & 1 ? sn : cs, v = q & 1 ? cs : sn;
  return f32x2{q == 1 || q == 2 ? -u : u, q >= 2 ? -v : v};
}

// (cosine, sine) of the pairs of `count` tokens from `token` on, [token][pair] in LDS:
// each once for the workgroup, whose waves all need the same. A thread keeps to a pair.
__device__ __forceinline__ void fill_turns(const PrepareArgs& a, const Powers& pw, int token, int count, f32x2* s_turn) {
  const int half = a.rot / 2;
  if (half == 0) return;
  const int first = static_cast<int>(threadIdx.x) / half, j = static_cast<int>(threadIdx.x) - first * half, step = kThreads / half;
  if (first >= step) return;
  const int n = j / 3, m = j - 3 * n;
  const int* from = a.pos_t;
  if (m == 1 && n < a.section_h) from = a.pos_h;
  if (m == 2 && n < a.section_w) from = a.pos_w;
  double f;
  if (a.inv_freq != nullptr) {
    f = static_cast<double>(a.inv_freq[j]) * 0.15915494309189535;
  } else {
    f = pw.base;
#pragma unroll
    for (int b = 0; b < 7; ++b) f *= j >> b & 1 ? pw.bit[b] : 1.0;
  }
  for (int t = first; t < count; t += step) {
    double x = static_cast<double>(from[token + t]) * f;
    s_turn[t * half + j] = turn_of(x - __builtin_rint(x));
  }
}

struct Turn { float c[4], s[4]; };
__device__ __forceinline__ Turn load_turn(const f32x2* p) {      // 16-byte aligned where rot is a multiple of 8
  Turn t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(p + 2 * i);
    t.c[2 * i] = x[0];
    t.s[2 * i] = x[1];
    t.c[2 * i + 1] = x[2];
    t.s[2 * i + 1] = x[3];
  }
  return t;
}

__device__ __forceinline__ u32x2 load4(const bf16* p) { return *reinterpret_cast<const u32x2*>(p); }
__device__ __forceinline__ void widen4(const u32x2& w, float* f) {
  f[0] = __uint_as_float(w[0] << 16);
  f[1] = __uint_as_float(w[0] & 0xffff0000u);
  f[2] = __uint_as_float(w[1] << 16);
  f[3] = __uint_as_float(w[1] & 0xffff0000u);
}
__device__ __forceinline__ void load_weights(const bf16* w, const Place& p, float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 1.0f;
  if (w != nullptr) {
    widen4(load4(w + p.lo), f);
    widen4(load4(w + p.hi), f + 4);
  }
}

// x: a lane's 8 values of a head, normalised and turned in place.
template <int D>
__device__ __forceinline__ void norm_turn(float* x, const float* w, const Turn& t, bool turns, float eps) {
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
  // x / root, rounded once: the reciprocal in two parts (the second of an infinite root,
  // which makes finite x 0, from the largest finite one)
  const float root = sqrtf(row_sum<D / 8>(ss) * (1.0f / D) + eps), r = 1.0f / root;
  const float rest = r * fmaf(-fminf(root, 0x1.fffffep127f), r, 1.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], r, x[i] * rest) * w[i];
  if (turns) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[i], b = x[4 + i];
      x[i] = a * t.c[i] - b * t.s[i];
      x[4 + i] = fmaf(a, t.s[i], b * t.c[i]);
    }
  }
}

// The queries of one token.
template <int D>
__device__ __forceinline__ void prepare_queries(const PrepareArgs& a, const Powers& pw, int token, f32x2* s_turn) {
  constexpr int LR = D / 8, RI = 64 / LR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Place p = place_of<D>(lane % LR, a.rot);
  float w[8];
  load_weights(a.q_norm, p, w);
  const bf16* src = a.q + static_cast<size_t>(token) * a.q_stride;
  bf16* dst = a.q_out + static_cast<size_t>(token) * a.Hq * D;
  u32x2 lo, hi;      // of the next head, on their way while the turns are made
  auto fetch = [&](int h0) __attribute__((always_inline)) {
    const bf16* row = src + min(h0 + lane / LR, a.Hq - 1) * a.q_head_stride;
    lo = load4(row + p.lo);
    hi = load4(row + p.hi);
  };
  fetch(wave * RI);
  fill_turns(a, pw, token, 1, s_turn);
  __syncthreads();
  Turn t{};
  if (p.turns) t = load_turn(s_turn + p.j);
  for (int h0 = wave * RI; h0 < a.Hq; h0 += kWaves * RI) {
    const int h = h0 + lane / LR;
    float x[8];
    widen4(lo, x);
    widen4(hi, x + 4);
    if (h0 + kWaves * RI < a.Hq) fetch(h0 + kWaves * RI);
    norm_turn<D>(x, w, t, p.turns, a.eps);
    if (h < a.Hq) {
      *reinterpret_cast<u32x2*>(dst + h * D + p.lo) = u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
      *reinterpret_cast<u32x2*>(dst + h * D + p.hi) = u32x2{pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
  }
}

// Smallest e with a <= 448 * 2^e (448 = 1.75 * 2^8) for the fp32 of these bits, bounded.
__device__ __forceinline__ int scale_exp_f32(int bits) {
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, kMinScaleExp), kMaxScaleExp);
}

// Rows into the pages: as the append (a wave takes K or V of a head, the runs that
// begin in its tile of tokens), K normalised and turned on the way.
template <int D>
__device__ __forceinline__ void prepare_rows(const PrepareArgs& a, const Powers& pw, int bx, int by, f32x2* s_turn) {
  constexpr int LR = D / 8;
  constexpr int RI = 64 / LR;
  constexpr int NI = kScaleRows / RI;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = by * 2 + (wave >> 1);
  const bool isv = wave & 1;
  const bf16* src = (isv ? a.v : a.k) + static_cast<size_t>(head) * D;
  const long stride = isv ? a.v_stride : a.k_stride;
  uint8_t* pages = isv ? a.v_pages : a.k_pages;
  float* scale = isv ? a.v_scale : a.k_scale;
  const int t0 = bx * a.tile;
  const int rr = lane / LR, s = lane % LR;
  Place p = place_of<D>(s, a.rot);
  if (isv) p = Place{8 * s, 8 * s + 4, 0, false};
  float w[8];
  load_weights(isv ? nullptr : a.k_norm, p, w);

  // Lane i holds the slot of token t0 + i - 1: a tile's runs end 31 tokens after
  // its begin at most.
  const int ti = t0 + lane - 1;
  const int win = ti >= 0 && ti < a.T && lane < 2 * kScaleRows + 1 ? a.slots[ti] : -1;
  const int before = __shfl_up(win, 1);
  const bool begins = lane >= 1 && lane <= a.tile && win >= 0 && win < a.num_slots &&
                      !(before >= 0 && before + 1 == win && win % kScaleRows != 0);
  unsigned long long todo = __ballot(begins);      // the same in all waves
  if (todo == 0) return;
  // the run that begins at lane i: its tokens' slots go on, to the block's end
  auto run_length = [&](int i) __attribute__((always_inline)) {
    const int slot = __builtin_amdgcn_readlane(win, i);
    const unsigned long long off = ~(__ballot(lane >= i && lane - i < kScaleRows - slot % kScaleRows && win == slot + (lane - i)) >> i);
    return __builtin_ctzll(off);      // 1 .. 16 - slot % 16
  };
  auto block_of = [&](int slot) __attribute__((always_inline)) {
    const int page = slot / a.page_size, blk = slot % a.page_size / kScaleRows;
    return (static_cast<size_t>(page) * a.Hkv + head) * (a.page_size / kScaleRows) + blk;
  };
  // a run's rows, the first's on their way while the turns are made
  u32x2 lo[NI], hi[NI];
  float old = 0.f;     // its block's scale
  auto fetch = [&]() __attribute__((always_inline)) {
    const int i = __builtin_ctzll(todo), n = run_length(i);
    const bf16* from = src + static_cast<size_t>(t0 + i - 1) * stride;
    old = scale[block_of(__builtin_amdgcn_readlane(win, i))];
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const bf16* row = from + min(k * RI + rr, n - 1) * stride;      // past the last: its copy
      lo[k] = load4(row + p.lo);
      hi[k] = load4(row + p.hi);
    }
  };
  if (head < a.Hkv) fetch();
  const int i1 = 63 - __builtin_clzll(todo);
  const int first = t0 + __builtin_ctzll(todo) - 1, last = t0 + i1 - 1 + run_length(i1);      // tokens of all runs: tile + 15 at most
  fill_turns(a, pw, first, last - first, s_turn);
  __syncthreads();
  if (head >= a.Hkv) return;
  while (todo) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int t = t0 + i - 1;
    const int slot = __builtin_amdgcn_readlane(win, i);
    const int r0 = slot % kScaleRows;
    const int n = run_length(i);

    const size_t bid = block_of(slot);
    uint8_t* block = pages + bid * (kScaleRows * D);
    const int held = held_exp(old);
    float x[NI][8];
    int top = 0;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      widen4(lo[k], x[k]);
      widen4(hi[k], x[k] + 4);
    }
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      if (k * RI >= n) break;
      if (!isv) {
        Turn r{};
        if (p.turns) r = load_turn(s_turn + (t - first + min(k * RI + rr, n - 1)) * (a.rot / 2) + p.j);
        norm_turn<D>(x[k], w, r, p.turns, a.eps);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int m = __float_as_uint(x[k][e]) & 0x7fffffff;
        if (m < 0x7f800000) top = max(top, m);
      }
    }
    int e = scale_exp_f32(wave_max(top));
    if (r0 > 0) {
      if (e > held) {
        // requantise rows [0, r0): x 2^(held - e) is exact but for underflow
        const float f = pow2f(held - e);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const int j = k * RI + rr;
          if (j < r0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t* at = reinterpret_cast<uint32_t*>(block + j * D + (h ? p.hi : p.lo));
              const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(*at, false);
              const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(*at, true);
              *at = pack_fp8x4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
            }
          }
        }
      }
      e = max(e, held);
    }
    const float inv = pow2f(-e);
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const int j = k * RI + rr;
      if (j < n) {
        float f[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) f[y] = to_code_range(x[k][y], inv);
        *reinterpret_cast<uint32_t*>(block + (r0 + j) * D + p.lo) = pack_fp8x4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<uint32_t*>(block + (r0 + j) * D + p.hi) = pack_fp8x4(f[4], f[5], f[6], f[7]);
      }
    }
    if (lane == 0) scale[bid] = pow2f(e);
    if (todo) fetch();     // behind the stores: it may be the same block's next run
  }
}

enum class Part { kBoth, kRows, kQueries };
template <int D, Part P>
__global__ __launch_bounds__(kThreads, P == Part::kQueries ? 8 : D == 256 ? 3 : 4) void prepare_qkv_paged_fp8_kernel(PrepareArgs a, Powers pw) {
  extern __shared__ __attribute__((aligned(16))) f32x2 s_turn[];
  const int x = blockIdx.x;
  if (P == Part::kRows || (P == Part::kBoth && x < a.kv_groups)) {
    const int pairs = (a.Hkv + 1) / 2;
    prepare_rows<D>(a, pw, x / pairs, x % pairs, s_turn);
  } else {
    prepare_queries<D>(a, pw, P == Part::kBoth ? x - a.kv_groups : x, s_turn);
  }
}

// Whether [o, o + n) meets one of `count` runs of w elements from x on, `step` (>= w) apart.
bool meets(const bf16* o, long n, const bf16* x, long count, long step, long w) {
  const intptr_t at = (reinterpret_cast<intptr_t>(o) - reinterpret_cast<intptr_t>(x)) / static_cast<intptr_t>(sizeof(bf16));
  const long i = at < w ? 0 : (at - w) / step + 1;      // the first run that ends behind o
  return i < count && i * step < at + n;
}

Powers powers_of(float theta, int rot) {
  Powers p{};
  const double r = -2.0 / rot;
  p.base = 0.15915494309189535;
  for (int i = 0; i < 7; ++i) p.bit[i] = std::pow(static_cast<double>(theta), r * (1 << i));
  return p;
}

}  // namespace
}  // namespace aila

extern "C" int aila_hip_prepare_qkv_paged_fp8(const void* q, long q_stride, long q_head_stride, const void* k,
                                              long k_stride, const void* v, long v_stride, void* q_out,
                                              const void* q_norm_w, const void* k_norm_w, void* k_pages, void* v_pages,
                                              float* k_scale, float* v_scale, const int* slots, const int* positions,
                                              const int* pos_h, const int* pos_w, int section_h, int section_w, int T,
                                              int Hq, int Hkv, int D, int page_size, int num_pages, int rotary_dim,
                                              float theta, const float* inv_freq, float eps, void* stream) {
  using namespace aila;
  const char* what = "prepare_qkv_paged_fp8";
  AILA_REQUIRE(q && k && v && q_out && slots, "%s: null pointer", what);
  if (int rc = check_paged_fp8(what, k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages)) return rc;
  AILA_REQUIRE(Hq > 0 && Hq <= 65535, "%s: bad Hq=%d", what, Hq);
  AILA_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 8 == 0, "%s: rotary_dim=%d must be a multiple of 8 up to D=%d", what,
               rotary_dim, D);
  AILA_REQUIRE(rotary_dim == 0 || positions != nullptr, "%s: positions are required", what);
  AILA_REQUIRE((pos_h == nullptr) == (pos_w == nullptr), "%s: pos_h and pos_w go together", what);
  AILA_REQUIRE(section_h >= 0 && section_w >= 0, "%s: bad sections h=%d w=%d", what, section_h, section_w);
  AILA_REQUIRE(rotary_dim == 0 || inv_freq != nullptr || theta > 0.f, "%s: theta=%g must be positive", what, static_cast<double>(theta));
  AILA_REQUIRE(q_head_stride >= D && q_head_stride % 8 == 0 && q_stride % 8 == 0 && q_stride >= (Hq - 1) * q_head_stride + D,
               "%s: query strides %ld (token) and %ld (head) must be multiples of 8 and hold %d heads of %d", what, q_stride,
               q_head_stride, Hq, D);
  AILA_REQUIRE(q_out != q || ((Hq == 1 || q_head_stride == D) && (T == 1 || q_stride == static_cast<long>(Hq) * D)),
               "%s: q_out may be q where its heads and tokens follow each other", what);
  AILA_REQUIRE(k_stride >= static_cast<long>(Hkv) * D && k_stride % 8 == 0 && v_stride >= static_cast<long>(Hkv) * D && v_stride % 8 == 0,
               "%s: token strides %ld (k) and %ld (v) must be multiples of 8 and hold Hkv * D = %ld values", what, k_stride, v_stride,
               static_cast<long>(Hkv) * D);
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                        reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q_norm_w) | reinterpret_cast<uintptr_t>(k_norm_w);
  AILA_REQUIRE(all % 16 == 0, "%s: q, k, v, q_out and the weights must be 16-byte aligned", what);
  // A wave takes the runs that begin in its tile one after the other. us, tiles of 1, 4, 8
  // and 16 tokens, a run a token / prompts of T / 4, 32 / 8 heads, D = 128: T = 256
  // 8.0/7.5, 9.1/7.9, 13.6/8.0, 22.8/8.8; 512 12.6/10.7, 10.8/7.9, 14.2/8.4, 23.3/8.3; 1024
  // 23.0/16.3, 17.0/11.1, 18.0/9.7, 25.9/10.7; 2048 41.1/27.4, 29.0/16.7, 26.8/14.5,
  // 29.6/13.7; 4096 77.3/48.6, 52.4/33.7, 48.2/27.5, 46.2/22.3. 16 / 4, D = 256: 256 7.1/9.0,
  // 10.2/10.6, 15.6/10.6, 26.6/12.3; 1024 19.0/20.3, 14.8/11.9, 17.9/12.1, 29.1/13.9; 4096
  // 60.9/64.2, 45.0/35.7, 41.4/29.2, 40.3/24.2.
  const int tile = T <= 256 ? 1 : T <= 1024 ? 4 : T <= 2048 ? 8 : kScaleRows;
  // fewer than 2^32 threads, the most of a launch
  const long kv_groups = (static_cast<long>(T) + tile - 1) / tile * ((Hkv + 1) / 2);
  AILA_REQUIRE(T > 0 && T <= (1 << 30) && (kv_groups + T) * kThreads < (1L << 32), "%s: T=%d tokens are none or too many for one call", what, T);
  {
    const bf16 *o = static_cast<const bf16*>(q_out), *x = static_cast<const bf16*>(q);
    const long n = static_cast<long>(T) * Hq * D, span = (Hq - 1) * q_head_stride + D, row = static_cast<long>(Hkv) * D;
    bool over = meets(o, n, static_cast<const bf16*>(k), T, k_stride, row) || meets(o, n, static_cast<const bf16*>(v), T, v_stride, row);
    if (o != x) {
      // the first token that ends behind q_out's begin may have it between two heads; the next one may not
      const long at = (reinterpret_cast<intptr_t>(o) - reinterpret_cast<intptr_t>(x)) / static_cast<long>(sizeof(bf16));
      const long i = at < span ? 0 : (at - span) / q_stride + 1;
      over |= (i < T && meets(o, n, x + i * q_stride, Hq, q_head_stride, D)) || (i + 1 < T && (i + 1) * q_stride < at + n);
    }
    AILA_REQUIRE(!over, "%s: q_out overlaps q, k or v", what);
  }
  PrepareArgs a{};
  a.q = static_cast<const bf16*>(q);
  a.k = static_cast<const bf16*>(k);
  a.v = static_cast<const bf16*>(v);
  a.q_stride = q_stride; a.q_head_stride = q_head_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_out = static_cast<bf16*>(q_out);
  a.q_norm = static_cast<const bf16*>(q_norm_w);
  a.k_norm = static_cast<const bf16*>(k_norm_w);
  a.k_pages = static_cast<uint8_t*>(k_pages);
  a.v_pages = static_cast<uint8_t*>(v_pages);
  a.k_scale = k_scale; a.v_scale = v_scale;
  a.slots = slots;
  a.pos_t = positions;
  a.pos_h = pos_h != nullptr ? pos_h : positions;
  a.pos_w = pos_w != nullptr ? pos_w : positions;
  a.section_h = section_h; a.section_w = section_w;
  a.inv_freq = inv_freq;
  a.T = T; a.tile = tile; a.Hq = Hq; a.Hkv = Hkv; a.page_size = page_size; a.num_slots = num_pages * page_size;
  a.rot = rotary_dim;
  a.kv_groups = static_cast<int>(kv_groups);
  a.eps = eps;
  const Powers pw = rotary_dim > 0 && inv_freq == nullptr ? powers_of(theta, rotary_dim) : Powers{};
  // One launch, rows first, or two (us, one / two). 16 / 4, D = 256: T = 32 7.0 / 10.1, 1024
  // 12.0 / 16.4, 4096 (92 MB) 24.9 / 28.6, 6000 (135 MB) 43.3 / 38.4, 8191 (184 MB) 63.4 / 54.3;
  // 32 / 8, D = 128: 4096 24.4 / 26.7, 6000 38.2 / 38.0, 8191 55.2 / 50.8; 16 / 8, D = 128: 8191
  // (117 MB) 34.0 / 34.6. Where the data do not stay in the caches, queries alone run at
  // twice the waves a SIMD.
  constexpr long kOneLaunchBytes = 120L << 20;
  const long moved = static_cast<long>(T) * D * (4L * Hq + 6L * Hkv);
  const size_t lds = static_cast<size_t>(tile + kScaleRows - 1) * (rotary_dim / 2) * sizeof(f32x2);
  auto go = [&](auto kernel, long groups, size_t bytes) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(kThreads), bytes, static_cast<hipStream_t>(stream), a, pw);
  };
  auto launch = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    if (moved <= kOneLaunchBytes) {
      go(prepare_qkv_paged_fp8_kernel<kD, Part::kBoth>, kv_groups + T, lds);
    } else {
      go(prepare_qkv_paged_fp8_kernel<kD, Part::kRows>, kv_groups, lds);
      go(prepare_qkv_paged_fp8_kernel<kD, Part::kQueries>, T, (rotary_dim / 2) * sizeof(f32x2));
    }
  };
  if (D == 64) launch(std::integral_constant<int, 64>{});
  else if (D == 128) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 256>{});
  return check_launch(what);
}
