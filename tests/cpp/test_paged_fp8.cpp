// The ops:: forms of the 8-bit paged cache on the GPU: a prompt step and decode
// steps of two requests, attention checked in doubles over the rows that the
// cache reads back, rows against what was written. Exit code 0 = all passed.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <stdexcept>
#include <vector>

#include "Ops.hpp"
#include "aila_hip.h"

static int g_fail = 0;
static void expect(bool ok, const char* name, double err) {
  std::printf("%-44s %s (err %.3g)\n", name, ok ? "OK" : "FAIL", err);
  if (!ok) ++g_fail;
}
static uint64_t g_state = 0x1234567ull;
static float rnd() {   // uniform in [-2, 2)
  g_state = g_state * 6364136223846793005ull + 1442695040888963407ull;
  return static_cast<float>((g_state >> 40) * (4.0 / 16777216.0) - 2.0);
}
static uint16_t bf16_of(float x) {
  uint32_t u;
  std::memcpy(&u, &x, 4);
  return static_cast<uint16_t>((u + 0x7fff + (u >> 16 & 1)) >> 16);
}
static double value(uint16_t b) {
  const uint32_t u = static_cast<uint32_t>(b) << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
template <typename T>
static Tensor upload(Context& ctx, const std::vector<T>& h, std::vector<int64_t> shape, DType dt) {
  Tensor t = Tensor::allocate(ctx, shape, dt);
  ctx.memcpy_h2d(t.data(), h.data(), h.size() * sizeof(T));
  return t;
}
template <typename T>
static std::vector<T> download(Context& ctx, Tensor& t) {
  std::vector<T> h(t.numel());
  ctx.memcpy_d2h(h.data(), t.data(), h.size() * sizeof(T));
  return h;
}
template <typename F>
static void refuses(F&& f, const char* name) {
  bool thrown = false;
  try {
    f();
  } catch (const std::runtime_error&) {
    thrown = true;
  }
  expect(thrown, name, 0);
}

int main() {
  Context ctx;
  const int B = 2, Hq = 8, Hkv = 2, D = 128, page = 32, P = 20, mp = 8, T = 64, max_len = mp * page;
  std::vector<int> zero(B, 0), fresh = {50, 7}, none(B * mp, -1), pool(P), count = {P};
  for (int i = 0; i < P; ++i) pool[i] = i;
  Tensor cached = upload(ctx, zero, {B}, DType::s32), added = upload(ctx, fresh, {B}, DType::s32);
  Tensor table = upload(ctx, none, {B, mp}, DType::s32), free_pages = upload(ctx, pool, {P}, DType::s32);
  Tensor free_count = upload(ctx, count, {1}, DType::s32);
  Tensor slots = Tensor::allocate(ctx, {T}, DType::s32), starts = Tensor::allocate(ctx, {B + 1}, DType::s32);
  Tensor lens = Tensor::allocate(ctx, {B}, DType::s32);
  const std::vector<uint8_t> codes(size_t(P) * Hkv * page * D, 0);
  const std::vector<float> ones(size_t(P) * Hkv * page / 16, 1.0f);
  Tensor kp = upload(ctx, codes, {P, Hkv, page, D}, DType::u8), vp = upload(ctx, codes, {P, Hkv, page, D}, DType::u8);
  Tensor ks = upload(ctx, ones, {P, Hkv, page / 16}, DType::f32), vs = upload(ctx, ones, {P, Hkv, page / 16}, DType::f32);
  const size_t need = std::max(aila_hip_gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len),
                               aila_hip_gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len));
  Tensor ws = Tensor::allocate(ctx, {static_cast<int64_t>(need)}, DType::u8);

  for (int step = 0; step < 4; ++step) {
    const bool decode = step > 0;
    const int rows = decode ? B : T;       // one token a request, or a batch with room behind it
    ops::kv_pages_reserve(ctx, cached, added, table, free_pages, free_count, page, slots, starts, lens);
    std::vector<uint16_t> q(size_t(rows) * Hq * D), k(size_t(rows) * Hkv * D), v(k.size());
    for (auto* x : {&q, &k, &v})
      for (auto& e : *x) e = bf16_of(rnd());
    Tensor tq = upload(ctx, q, {rows, Hq * D}, DType::bf16), tk = upload(ctx, k, {rows, Hkv * D}, DType::bf16);
    Tensor tv = upload(ctx, v, {rows, Hkv * D}, DType::bf16), out = Tensor::allocate(ctx, {rows, Hq * D});
    ops::copy_to_cache_paged_fp8(ctx, tk, tv, kp, vp, ks, vs, slots);
    if (decode) ops::attention_decode_paged_fp8(ctx, tq, kp, vp, ks, vs, table, lens, out, Hq, max_len, &ws);
    else ops::attention_prefill_paged_fp8(ctx, tq, kp, vp, ks, vs, table, starts, lens, out, Hq, max_len, &ws);
    const auto got = download<uint16_t>(ctx, out);
    const auto tab = download<int>(ctx, table), len = download<int>(ctx, lens), start = download<int>(ctx, starts);
    double worst = 0, row_err = 0;
    for (int b = 0; b < B; ++b) {
      std::vector<int> at(len[b]);
      for (int r = 0; r < len[b]; ++r) at[r] = tab[b * mp + r / page] * page + r % page;
      Tensor ts = upload(ctx, at, {len[b]}, DType::s32);
      Tensor ko = Tensor::allocate(ctx, {len[b], Hkv * D}), vo = Tensor::allocate(ctx, {len[b], Hkv * D});
      ops::read_cache_paged_fp8(ctx, kp, vp, ks, vs, ts, ko, vo);
      const auto kr = download<uint16_t>(ctx, ko), vr = download<uint16_t>(ctx, vo);
      const int n = start[b + 1] - start[b];
      for (int i = 0; i < n; ++i) {
        const int t = start[b] + i, attended = len[b] - n + i + 1;
        // the row just written: |x| < 2, so a code is within 2^-4 of its value or, at the bottom, 2^-10 of a scale of 2^-7
        for (int e = 0; e < Hkv * D; ++e) {
          const double x = value(k[size_t(t) * Hkv * D + e]), y = value(kr[size_t(attended - 1) * Hkv * D + e]);
          row_err = std::fmax(row_err, std::fabs(x - y) / (std::fabs(x) / 16 + std::ldexp(1.0, -17)));
        }
        for (int h = 0; h < Hq; ++h) {
          const uint16_t* qr = &q[(size_t(t) * Hq + h) * D];
          std::vector<double> s(attended);
          double top = -1e300, sum = 0;
          for (int r = 0; r < attended; ++r) {
            double x = 0;
            for (int d = 0; d < D; ++d) x += value(qr[d]) * value(kr[(size_t(r) * Hkv + h / (Hq / Hkv)) * D + d]);
            s[r] = x / std::sqrt(double(D));
            top = std::fmax(top, s[r]);
          }
          for (auto& x : s) sum += x = std::exp(x - top);
          for (int d = 0; d < D; ++d) {
            double o = 0, mag = 0;
            for (int r = 0; r < attended; ++r) {
              const double x = s[r] / sum * value(vr[(size_t(r) * Hkv + h / (Hq / Hkv)) * D + d]);
              o += x;
              mag += std::fabs(x);
            }
            // half a step of bf16; weights rounded to 2^-8 (decode: 2^-16); 2^-12 for fp32 sums of terms below 46 and the exponentials
            const double tol = std::fabs(o) / 256 + mag * ((decode ? 1.0 / 65536 : 1.0 / 256) + 1.0 / 4096);
            worst = std::fmax(worst, std::fabs(value(got[(size_t(t) * Hq + h) * D + d]) - o) / (tol + 1e-30));
          }
        }
      }
    }
    expect(worst <= 1, decode ? "attention_decode_paged_fp8" : "attention_prefill_paged_fp8", worst);
    expect(row_err <= 1, "copy_to_cache_paged_fp8 / read_cache_paged_fp8", row_err);
    expect(len[0] == 50 + step && len[1] == 7 + step, "kv_pages_reserve", 0);
    cached = upload(ctx, len, {B}, DType::s32);
    added = upload(ctx, std::vector<int>(B, 1), {B}, DType::s32);
  }
  Tensor ended = upload(ctx, std::vector<int>{1, 1}, {B}, DType::s32);
  ops::kv_pages_release(ctx, ended, table, free_pages, free_count);
  expect(download<int>(ctx, free_count)[0] == P && download<int>(ctx, table) == none, "kv_pages_release", 0);

  Tensor q = Tensor::allocate(ctx, {B, Hq * D}), wrong = Tensor::allocate(ctx, {B, mp}, DType::f32);
  refuses([&] { ops::attention_decode_paged_fp8(ctx, q, kp, vp, ks, vs, wrong, lens, q, Hq, max_len); }, "a table of floats");
  refuses([&] { ops::attention_decode_paged_fp8(ctx, q, kp, vp, vs, wrong, table, lens, q, Hq, max_len); }, "scales of another shape");
  refuses([&] { ops::attention_decode_paged_fp8(ctx, q, kp, vp, ks, vs, table, lens, q, Hq + 1, max_len); }, "heads that the rows do not hold");
  refuses([&] { ops::attention_decode_paged_fp8(ctx, q, kp, vp, ks, vs, table, lens, q, Hq, max_len + 1); }, "more rows than the table");
  refuses([&] { ops::kv_pages_reserve(ctx, lens, added, table, free_pages, free_count, page, slots, starts, lens); }, "lengths over lengths");
  std::printf(g_fail ? "%d FAILED\n" : "ALL OK\n", g_fail);
  return g_fail ? 1 : 0;
}
