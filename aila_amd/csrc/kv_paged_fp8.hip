// Rows of the 8-bit paged KV cache: written (quantised) and read back by slot.
//
// Append: the tokens that fall into one block of 16 rows form a run (adjacent
// tokens with consecutive slots). For the run and each head
//   a = max |x| over its finite values, e = smallest with a <= 448 * 2^e,
//   e = max(e, the block's exponent) when rows stand before the run,
//   code = rne_e4m3(x * 2^-e),
// and when e grew, the rows before are requantised from the old exponent. A
// wave owns a run for one head and one of K and V, so block and scale have one
// writer, and it is bound by the bytes: 2 in and 1 out a value. A long prompt of
// 8191 tokens, 4 heads, D = 256: 15-17 us for 50 MB (a large copy reaches 4.7
// TB/s, 10.6 us); reading the rows back 9.9 us for the same. 32 single tokens,
// 8 heads, D = 128: 3.7 and 3.0 us, which are the launch and the chain slot ->
// rows and block -> codes.
#include "paged_fp8.hpp"

namespace aila {
namespace {

constexpr int kThreads = 256;

// Smallest e with |x| <= 448 * 2^e for the bf16 whose magnitude bits are
// `mag` (448 = 1.75 * 2^8), bounded.
__device__ __forceinline__ int scale_exp(int mag) {
  const int e = (mag >> 7) - 127 - 8 + ((mag & 0x7f) > 0x60 ? 1 : 0);
  return min(max(e, kMinScaleExp), kMaxScaleExp);
}

// Grid (ceil(T / tile), ceil(Hkv / 2)); wave w: K or V (w & 1) of head
// 2 * blockIdx.y + w / 2, the runs that begin in the workgroup's `tile` tokens.
template <int D>
__global__ __launch_bounds__(kThreads) void kv_append_paged_fp8_kernel(
    const bf16* __restrict__ k_new, const bf16* __restrict__ v_new, long new_stride, uint8_t* __restrict__ k_pages,
    uint8_t* __restrict__ v_pages, float* __restrict__ k_scale, float* __restrict__ v_scale,
    const int* __restrict__ slots, int T, int tile, int Hkv, int page_size, int num_slots) {
  constexpr int LR = D / 8;                 // lanes per row (8 values each)
  constexpr int RI = 64 / LR;               // rows per instruction
  constexpr int NI = kScaleRows / RI;       // instructions per block
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = static_cast<int>(blockIdx.y) * 2 + (wave >> 1);
  if (head >= Hkv) return;
  const bool isv = wave & 1;
  const bf16* src = (isv ? v_new : k_new) + static_cast<size_t>(head) * D;
  uint8_t* pages = isv ? v_pages : k_pages;
  float* scale = isv ? v_scale : k_scale;
  const int t0 = static_cast<int>(blockIdx.x) * tile;
  const int rr = lane / LR, c8 = (lane % LR) * 8;

  // Lane i holds the slot of token t0 + i - 1: a tile's runs end 31 tokens after
  // its begin at most.
  const int ti = t0 + lane - 1;
  const int win = ti >= 0 && ti < T && lane < 2 * kScaleRows + 1 ? slots[ti] : -1;
  const int before = __shfl_up(win, 1);
  const bool begins = lane >= 1 && lane <= tile && win >= 0 && win < num_slots &&
                      !(before >= 0 && before + 1 == win && win % kScaleRows != 0);
  unsigned long long todo = __ballot(begins);
  while (todo) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int t = t0 + i - 1;
    const int slot = __builtin_amdgcn_readlane(win, i);
    const int r0 = slot % kScaleRows;
    // the run: the tokens from i on whose slots go on, to the block's end
    const unsigned long long off = ~(__ballot(lane >= i && lane - i < kScaleRows - r0 && win == slot + (lane - i)) >> i);
    const int n = __builtin_ctzll(off);      // 1 .. 16 - r0

    u32x4 x[NI];
    int top = 0;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const int j = k * RI + rr;
      x[k] = u32x4{0u, 0u, 0u, 0u};
      if (j < n) x[k] = ld16(src + static_cast<size_t>(t + j) * new_stride + c8);
    }
    const int page = slot / page_size, blk = slot % page_size / kScaleRows;
    const size_t bid = (static_cast<size_t>(page) * Hkv + head) * (page_size / kScaleRows) + blk;
    uint8_t* block = pages + bid * (kScaleRows * D);
    const int e_old = static_cast<int>(__float_as_uint(scale[bid]) >> 23 & 0xff) - 127;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int a = x[k][w] & 0x7fff, b = x[k][w] >> 16 & 0x7fff;
        if (a < 0x7f80) top = max(top, a);
        if (b < 0x7f80) top = max(top, b);
      }
    }
    int e = scale_exp(wave_max(top));
    if (r0 > 0) {
      const int held = min(max(e_old, kMinScaleExp), kMaxScaleExp);
      if (e > held) {
        // requantise rows [0, r0): x 2^(held - e) is exact but for underflow
        const float f = pow2f(held - e);
#pragma unroll
        for (int k = 0; k < NI; ++k) {
          const int j = k * RI + rr;
          if (j < r0) {
            u32x2* p = reinterpret_cast<u32x2*>(block + j * D + c8);
            u32x2 w = *p;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], false);
              const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], true);
              w[h] = pack_fp8x4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
            }
            *p = w;
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
        unpack8(x[k], f);
#pragma unroll
        for (int w = 0; w < 8; ++w) f[w] = to_code_range(f[w], inv);
        *reinterpret_cast<u32x2*>(block + (r0 + j) * D + c8) =
            u32x2{pack_fp8x4(f[0], f[1], f[2], f[3]), pack_fp8x4(f[4], f[5], f[6], f[7])};
      }
    }
    if (lane == 0) scale[bid] = pow2f(e);
  }
}

// One thread: 8 values of K and of V of a token and head, so that a wave's stores
// are a contiguous KiB each (16 values a thread: 11.8 us against 10.5 for the
// 8191 tokens above).
template <int D>
__global__ __launch_bounds__(kThreads) void kv_read_paged_fp8_kernel(
    const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, const int* __restrict__ slots, bf16* __restrict__ k_out,
    bf16* __restrict__ v_out, long n, int Hkv, int page_size, int num_slots) {
  const long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n) return;
  const int c = static_cast<int>(i) & (D / 8 - 1);
  const unsigned th = static_cast<unsigned>(i / (D / 8)), t = th / Hkv;     // below 2^31
  const int head = static_cast<int>(th - t * Hkv);
  const int slot = slots[t];
  u32x4 k = {0u, 0u, 0u, 0u}, v = k;
  if (slot >= 0 && slot < num_slots) {
    const int page = slot / page_size, row = slot % page_size;
    const size_t bid = (static_cast<size_t>(page) * Hkv + head) * (page_size / kScaleRows) + row / kScaleRows;
    const size_t at = bid * (static_cast<size_t>(kScaleRows) * D) + (row % kScaleRows) * D + c * 8;
    const u32x2 kw = *reinterpret_cast<const u32x2*>(k_pages + at), vw = *reinterpret_cast<const u32x2*>(v_pages + at);
    const float ks = k_scale[bid], vs = v_scale[bid];
    k = u32x4{fp8x2_to_bf16x2<false>(kw[0], ks), fp8x2_to_bf16x2<true>(kw[0], ks), fp8x2_to_bf16x2<false>(kw[1], ks),
              fp8x2_to_bf16x2<true>(kw[1], ks)};
    v = u32x4{fp8x2_to_bf16x2<false>(vw[0], vs), fp8x2_to_bf16x2<true>(vw[0], vs), fp8x2_to_bf16x2<false>(vw[1], vs),
              fp8x2_to_bf16x2<true>(vw[1], vs)};
  }
  *reinterpret_cast<u32x4*>(k_out + i * 8) = k;
  *reinterpret_cast<u32x4*>(v_out + i * 8) = v;
}

}  // namespace

// Shape and pointer checks shared by the entry points over the 8-bit pages.
int check_paged_fp8(const char* what, const void* k_pages, const void* v_pages, const float* k_scale,
                    const float* v_scale, int Hkv, int D, int page_size, int num_pages) {
  AILA_REQUIRE(k_pages && v_pages && k_scale && v_scale, "%s: null pointer", what);
  AILA_REQUIRE(Hkv > 0 && Hkv <= 65535, "%s: bad Hkv=%d", what, Hkv);
  if (D != 64 && D != 128 && D != 256)
    return set_error(AILA_HIP_EUNSUPPORTED, "%s: D=%d not in {64,128,256}", what, D);
  AILA_REQUIRE(page_size > 0 && page_size % kScaleRows == 0, "%s: page_size=%d must be a positive multiple of %d", what,
               page_size, kScaleRows);
  AILA_REQUIRE(num_pages > 0 && static_cast<long>(num_pages) * page_size < (1L << 31),
               "%s: num_pages=%d pages of %d rows: slots must fit 31 bits", what, num_pages, page_size);
  AILA_REQUIRE(static_cast<long>(num_pages) * Hkv * (page_size / kScaleRows) < (1L << 31),
               "%s: more than 2^31 blocks of %d rows and heads", what, kScaleRows);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(k_pages) % 16 == 0 && reinterpret_cast<uintptr_t>(v_pages) % 16 == 0,
               "%s: k_pages and v_pages must be 16-byte aligned", what);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(k_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(v_scale) % 4 == 0,
               "%s: k_scale and v_scale must be 4-byte aligned", what);
  return AILA_HIP_OK;
}

}  // namespace aila

extern "C" int aila_hip_kv_append_paged_fp8(const void* k_new, const void* v_new, long new_stride, void* k_pages,
                                            void* v_pages, float* k_scale, float* v_scale, const int* slots, int T,
                                            int Hkv, int D, int page_size, int num_pages, void* stream) {
  using namespace aila;
  AILA_REQUIRE(k_new && v_new && slots, "kv_append_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("kv_append_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  // 16 tokens a workgroup at least where T is large: fewer than 2^32 threads, the most of a launch
  AILA_REQUIRE(T > 0 && T <= (1 << 28) - kScaleRows, "kv_append_paged_fp8: T=%d outside [1, 2^28 - 16]", T);
  AILA_REQUIRE(new_stride >= static_cast<long>(Hkv) * D && new_stride % 8 == 0,
               "kv_append_paged_fp8: token stride %ld must be a multiple of 8 and hold Hkv * D = %ld values", new_stride,
               static_cast<long>(Hkv) * D);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(k_new) % 16 == 0 && reinterpret_cast<uintptr_t>(v_new) % 16 == 0,
               "kv_append_paged_fp8: k_new and v_new must be 16-byte aligned");
  // Single tokens are a run each, which a wave takes one after the other; of a
  // prompt 15 of 16 tokens begin none, and a wave that finds none is a waste. us,
  // single tokens / prompt, 8 heads, D = 128, tiles of 1, 4, 8 and 16 tokens:
  // T = 32 3.2/3.3, 6.0/3.3, 11.1/3.4, 20.8/4.5; 512 6.3/8.3, 7.3/4.2, 10.4/3.6,
  // 18.0/4.5; 1024 10.1/14.1, 10.3/5.9, 12.4/4.3, 18.4/4.5; 2048 18.1/25.0,
  // 16.5/9.2, 18.6/5.9, 22.0/5.4; 4096 32.9/45.8, 29.3/15.3, 29.9/9.3, 34.3/8.3. T is
  // all that the host knows: single tokens that stand together in a large T take the
  // long tiles too, and a wave stores up to 16 runs in a row (32 of them padded to
  // 4096 31.4 us, to 256 4.5; 30 behind prompts of 3 x 1300 tokens 24.3, prompts of as
  // many alone 9.6).
  const int tile = T <= 256 ? 1 : T <= 1024 ? 4 : T <= 2048 ? 8 : kScaleRows;
  const dim3 grid((T + tile - 1) / tile, (Hkv + 1) / 2);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const bf16*>(k_new), static_cast<const bf16*>(v_new), new_stride,
                       static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), k_scale, v_scale, slots, T, tile,
                       Hkv, page_size, num_pages * page_size);
  };
  if (D == 64) go(kv_append_paged_fp8_kernel<64>);
  else if (D == 128) go(kv_append_paged_fp8_kernel<128>);
  else go(kv_append_paged_fp8_kernel<256>);
  return check_launch("kv_append_paged_fp8");
}

extern "C" int aila_hip_kv_read_paged_fp8(const void* k_pages, const void* v_pages, const float* k_scale,
                                          const float* v_scale, const int* slots, void* k_out, void* v_out, int T,
                                          int Hkv, int D, int page_size, int num_pages, void* stream) {
  using namespace aila;
  AILA_REQUIRE(slots && k_out && v_out, "kv_read_paged_fp8: null pointer");
  if (int rc = check_paged_fp8("kv_read_paged_fp8", k_pages, v_pages, k_scale, v_scale, Hkv, D, page_size, num_pages))
    return rc;
  AILA_REQUIRE(T > 0, "kv_read_paged_fp8: bad T=%d", T);
  AILA_REQUIRE(reinterpret_cast<uintptr_t>(k_out) % 16 == 0 && reinterpret_cast<uintptr_t>(v_out) % 16 == 0,
               "kv_read_paged_fp8: k_out and v_out must be 16-byte aligned");
  // a thread 8 values: fewer than 2^32 of them, the most of a launch
  const long n = static_cast<long>(T) * Hkv * (D / 8);
  AILA_REQUIRE(n < (1L << 32) - kThreads, "kv_read_paged_fp8: T=%d rows of %d heads are too many for one call", T, Hkv);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), static_cast<const uint8_t*>(k_pages),
                       static_cast<const uint8_t*>(v_pages), k_scale, v_scale, slots, static_cast<bf16*>(k_out),
                       static_cast<bf16*>(v_out), n, Hkv, page_size, num_pages * page_size);
  };
  if (D == 64) go(kv_read_paged_fp8_kernel<64>);
  else if (D == 128) go(kv_read_paged_fp8_kernel<128>);
  else go(kv_read_paged_fp8_kernel<256>);
  return check_launch("kv_read_paged_fp8");
}
