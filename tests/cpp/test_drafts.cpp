// The ops:: forms of drafted trees on the 8-bit paged cache on the GPU: prompts,
// one step of trees (prepare, tree attention checked in doubles over the rows that
// the cache reads back, keep, trim), and a fork. Exit code 0 = all passed.
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
  const int B = 3, Hq = 8, Hkv = 2, D = 128, page = 32, P = 20, mp = 8, T = 20, max_len = mp * page, rot = 64, G = Hq / Hkv;
  const double theta = 1e4, eps = 1e-6;
  const std::vector<int> prompt = {50, 7, 0}, drafted = {6, 6, 2}, none(B * mp, -1);
  std::vector<int> pool(P);
  for (int i = 0; i < P; ++i) pool[i] = i;
  Tensor cached = upload(ctx, std::vector<int>(B, 0), {B}, DType::s32), added = upload(ctx, prompt, {B}, DType::s32);
  Tensor table = upload(ctx, none, {B, mp}, DType::s32), free_pages = upload(ctx, pool, {P}, DType::s32);
  Tensor free_count = upload(ctx, std::vector<int>{P}, {1}, DType::s32);
  Tensor first = Tensor::allocate(ctx, {64}, DType::s32), slots = Tensor::allocate(ctx, {T}, DType::s32);
  Tensor starts = Tensor::allocate(ctx, {B + 1}, DType::s32), lens = Tensor::allocate(ctx, {B}, DType::s32);
  const std::vector<uint8_t> codes(size_t(P) * Hkv * page * D, 0);
  const std::vector<float> ones(size_t(P) * Hkv * page / 16, 1.0f);
  std::vector<Tensor> kp, vp, ks, vs;      // two layers
  for (int l = 0; l < 2; ++l) {
    kp.push_back(upload(ctx, codes, {P, Hkv, page, D}, DType::u8));
    vp.push_back(upload(ctx, codes, {P, Hkv, page, D}, DType::u8));
    ks.push_back(upload(ctx, ones, {P, Hkv, page / 16}, DType::f32));
    vs.push_back(upload(ctx, ones, {P, Hkv, page / 16}, DType::f32));
  }
  std::vector<ops::PagedLayerFp8> layers;
  for (int l = 0; l < 2; ++l) layers.push_back({&kp[l], &vp[l], &ks[l], &vs[l]});
  const auto random = [&](size_t n) {
    std::vector<uint16_t> x(n);
    for (auto& e : x) e = bf16_of(rnd());
    return x;
  };
  // rows [0, n) of a request as the cache reads them, K then V
  const auto rows = [&](int l, int b, int n) {
    const auto tab = download<int>(ctx, table);
    std::vector<int> at(n);
    for (int r = 0; r < n; ++r) at[r] = tab[b * mp + r / page] * page + r % page;
    Tensor ts = upload(ctx, at, {n}, DType::s32);
    Tensor ko = Tensor::allocate(ctx, {n, Hkv * D}), vo = Tensor::allocate(ctx, {n, Hkv * D});
    ops::read_cache_paged_fp8(ctx, kp[l], vp[l], ks[l], vs[l], ts, ko, vo);
    auto x = download<uint16_t>(ctx, ko);
    const auto v = download<uint16_t>(ctx, vo);
    x.insert(x.end(), v.begin(), v.end());
    return x;
  };

  ops::kv_pages_reserve(ctx, cached, added, table, free_pages, free_count, page, first, starts, lens);
  for (int l = 0; l < 2; ++l) {
    Tensor tk = upload(ctx, random(size_t(64) * Hkv * D), {64, Hkv * D}, DType::bf16);
    Tensor tv = upload(ctx, random(size_t(64) * Hkv * D), {64, Hkv * D}, DType::bf16);
    ops::copy_to_cache_paged_fp8(ctx, tk, tv, kp[l], vp[l], ks[l], vs[l], first);
  }

  cached = upload(ctx, prompt, {B}, DType::s32);
  added = upload(ctx, drafted, {B}, DType::s32);
  ops::kv_pages_reserve(ctx, cached, added, table, free_pages, free_count, page, slots, starts, lens);
  const auto start = download<int>(ctx, starts), len = download<int>(ctx, lens);
  // tokens 0 .. 5 of a tree: 0 its root, 1 and 2 below 0, 3 below 1, 4 below 2, 5 below 4; the third
  // request's first token attends nothing, its second itself
  const uint64_t tree[6] = {1, 3, 5, 11, 21, 53}, pair[2] = {0, 2};
  std::vector<int> mask(2 * T, 0), pos(3 * T, 0);
  for (int b = 0; b < B; ++b)
    for (int i = 0; i < drafted[b]; ++i) {
      mask[2 * (start[b] + i)] = static_cast<int>(b < 2 ? tree[i] : pair[i]);
      for (int s = 0; s < 3; ++s) pos[s * T + start[b] + i] = 1000 * s + prompt[b] + i;
    }
  Tensor tmask = upload(ctx, mask, {T, 2}, DType::s32), tpos = upload(ctx, pos, {3, T}, DType::s32);
  const auto wq = random(D), wk = random(D);
  Tensor twq = upload(ctx, wq, {D}, DType::bf16), twk = upload(ctx, wk, {D}, DType::bf16);
  const int section_h = 11, section_w = 10;
  // the turned and normalised value of dim d of a row, and the size of what it is a sum of
  const auto prepared = [&](const uint16_t* x, const std::vector<uint16_t>& w, int t, int d, double* size) {
    double ss = 0;
    for (int e = 0; e < D; ++e) ss += value(x[e]) * value(x[e]);
    const double r = 1 / std::sqrt(ss / D + eps);
    const auto y = [&](int e) { return value(x[e]) * r * value(w[e]); };
    if (d >= rot) return *size = std::fabs(y(d)), y(d);
    const int p = d % (rot / 2);
    const int s = p % 3 == 1 && p / 3 < section_h ? 1 : p % 3 == 2 && p / 3 < section_w ? 2 : 0;
    const double a = pos[s * T + t] * std::pow(theta, -2.0 * p / rot), c = std::cos(a), n = std::sin(a);
    *size = std::fabs(y(p)) + std::fabs(y(p + rot / 2));
    return d < rot / 2 ? y(p) * c - y(p + rot / 2) * n : y(p + rot / 2) * c + y(p) * n;
  };
  const size_t need = aila_hip_gqa_tree_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len, 1);
  Tensor ws = Tensor::allocate(ctx, {static_cast<int64_t>(need)}, DType::u8);
  for (int l = 0; l < 2; ++l) {
    // q in rows of q|gate, each head's gate behind it
    const auto q = random(size_t(T) * Hq * 2 * D), k = random(size_t(T) * Hkv * D), v = random(size_t(T) * Hkv * D);
    Tensor tq = upload(ctx, q, {T, Hq * 2 * D}, DType::bf16), tk = upload(ctx, k, {T, Hkv * D}, DType::bf16);
    Tensor tv = upload(ctx, v, {T, Hkv * D}, DType::bf16), qr = Tensor::allocate(ctx, {T, Hq * D});
    const std::vector<uint16_t> before(size_t(T) * Hq * D, 0x1234);
    Tensor out = upload(ctx, before, {T, Hq * D}, DType::bf16);
    ops::prepare_qkv_paged_fp8(ctx, tq, tk, tv, kp[l], vp[l], ks[l], vs[l], slots, tpos, &twq, &twk, qr, Hq, rot, theta, eps, 2 * D,
                               section_h, section_w);
    ops::attention_tree_paged_fp8(ctx, qr, kp[l], vp[l], ks[l], vs[l], table, starts, lens, tmask, out, Hq, max_len, l ? &ws : nullptr);
    const auto got = download<uint16_t>(ctx, out), query = download<uint16_t>(ctx, qr);
    double q_err = 0, row_err = 0, worst = 0;
    bool untouched = true;
    for (size_t e = size_t(start[B]) * Hq * D; e < got.size(); ++e) untouched &= got[e] == 0x1234;
    for (int b = 0; b < B; ++b) {
      const auto kv = rows(l, b, len[b]);
      const uint16_t *kr = kv.data(), *vr = kr + size_t(len[b]) * Hkv * D;
      for (int i = 0; i < drafted[b]; ++i) {
        const int t = start[b] + i;
        for (int e = 0; e < Hkv * D; ++e) {
          // a code is within 2^-4 of its value or 2^-10 of its scale, which stays below 2^-3 (448 of it cover 56; |k| < 8);
          // 2^-16 of the sum's terms for fp32 and the angle
          const size_t at = size_t(prompt[b] + i) * Hkv * D + e;
          double size = 0;
          const double y = prepared(&k[(size_t(t) * Hkv + e / D) * D], wk, t, e % D, &size), x = value(v[size_t(t) * Hkv * D + e]);
          row_err = std::fmax(row_err, std::fabs(value(kr[at]) - y) / (std::fabs(y) / 16 + std::ldexp(1.0, -13) + std::ldexp(size, -16)));
          row_err = std::fmax(row_err, std::fabs(value(vr[at]) - x) / (std::fabs(x) / 16 + std::ldexp(1.0, -13)));
        }
        std::vector<int> attended;
        for (int r = 0; r < prompt[b]; ++r) attended.push_back(r);
        for (int j = 0; j < drafted[b]; ++j)
          if (static_cast<uint32_t>(mask[2 * t]) >> j & 1) attended.push_back(prompt[b] + j);
        for (int h = 0; h < Hq; ++h) {
          const uint16_t* row = &query[(size_t(t) * Hq + h) * D];
          for (int d = 0; d < D; ++d) {
            double size = 0;
            const double y = prepared(&q[(size_t(t) * Hq + h) * 2 * D], wq, t, d, &size);
            q_err = std::fmax(q_err, std::fabs(value(row[d]) - y) / (std::fabs(y) / 256 + std::ldexp(size, -16)));
          }
          std::vector<double> s(attended.size());
          double top = -1e300, sum = 0;
          for (size_t r = 0; r < s.size(); ++r) {
            double x = 0;
            for (int d = 0; d < D; ++d) x += value(row[d]) * value(kr[(size_t(attended[r]) * Hkv + h / G) * D + d]);
            s[r] = x / std::sqrt(double(D));
            top = std::fmax(top, s[r]);
          }
          for (auto& x : s) sum += x = std::exp(x - top);
          for (int d = 0; d < D; ++d) {
            double o = 0, mag = 0;
            for (size_t r = 0; r < s.size(); ++r) {
              const double x = s[r] / sum * value(vr[(size_t(attended[r]) * Hkv + h / G) * D + d]);
              o += x;
              mag += std::fabs(x);
            }
            // half a step of bf16, weights rounded to 2^-8, and 2^-10 for scores below 48 (|q| and |k| below 23, over
            // sqrt(D)) off by 128 roundings of 2^-24, above and below the line
            const double tol = std::fabs(o) / 256 + mag * (1.0 / 256 + 1.0 / 1024);
            worst = std::fmax(worst, std::fabs(value(got[(size_t(t) * Hq + h) * D + d]) - o) / (tol + 1e-30));
          }
        }
      }
    }
    expect(q_err <= 1, "prepare_qkv_paged_fp8: queries", q_err);
    expect(row_err <= 1, "prepare_qkv_paged_fp8: rows", row_err);
    expect(worst <= 1, "attention_tree_paged_fp8", worst);
    expect(untouched, "rows behind the last request", 0);
  }

  const std::vector<int> path = {0, 2, 4, 0, 1, 3, 0, 0, 0}, paths = {3, 3, 0};
  std::vector<std::vector<uint16_t>> was;
  for (int l = 0; l < 2; ++l)
    for (int b = 0; b < 2; ++b) was.push_back(rows(l, b, len[b]));
  Tensor kept = upload(ctx, path, {B, 3}, DType::s32), kept_lens = upload(ctx, paths, {B}, DType::s32);
  Tensor now = Tensor::allocate(ctx, {B}, DType::s32);
  ops::kv_keep_paged_fp8(ctx, layers, table, cached, kept, kept_lens, now);
  expect(download<int>(ctx, now) == std::vector<int>{53, 10, 0}, "kv_keep_paged_fp8: lengths", 0);
  double err = 0;
  for (int l = 0; l < 2; ++l)
    for (int b = 0; b < 2; ++b) {
      const auto is = rows(l, b, prompt[b] + 3);
      const auto& old = was[2 * l + b];
      for (int part = 0; part < 2; ++part)
        for (int r = 0; r < prompt[b] + 3; ++r) {
          const int from = r < prompt[b] ? r : prompt[b] + path[3 * b + r - prompt[b]];
          for (int e = 0; e < Hkv * D; ++e) {   // as it was, but for what underflows at a scale below 2^-3
            const double x = value(is[(size_t(part) * (prompt[b] + 3) + r) * Hkv * D + e]);
            err = std::fmax(err, std::fabs(x - value(old[(size_t(part) * len[b] + from) * Hkv * D + e])) * std::ldexp(1.0, 13));
          }
        }
    }
  expect(err <= 1, "kv_keep_paged_fp8: rows", err);
  ops::kv_pages_trim(ctx, now, table, free_pages, free_count, page);
  expect(download<int>(ctx, free_count)[0] == P - 3, "kv_pages_trim", 0);   // two pages and one stay

  added = upload(ctx, std::vector<int>{0, 0, 53}, {B}, DType::s32);
  ops::kv_pages_reserve(ctx, now, added, table, free_pages, free_count, page, first, starts, lens);
  Tensor from = upload(ctx, std::vector<int>{0}, {1}, DType::s32), to = upload(ctx, std::vector<int>{2}, {1}, DType::s32);
  Tensor count = upload(ctx, std::vector<int>{53}, {1}, DType::s32);
  ops::kv_copy_paged_fp8(ctx, layers, table, from, to, count, max_len);
  expect(rows(0, 0, 53) == rows(0, 2, 53) && rows(1, 0, 53) == rows(1, 2, 53), "kv_copy_paged_fp8", 0);

  Tensor q = Tensor::allocate(ctx, {T, Hq * D}), k = Tensor::allocate(ctx, {T, Hkv * D});
  Tensor odd = upload(ctx, std::vector<int>(T, 1), {T, 1}, DType::s32);
  Tensor small = Tensor::allocate(ctx, {P, Hkv, page / 2, D}, DType::u8);
  Tensor small_scale = Tensor::allocate(ctx, {P, Hkv, page / 32}, DType::f32);
  refuses([&] { ops::attention_tree_paged_fp8(ctx, q, kp[0], vp[0], ks[0], vs[0], table, starts, lens, odd, q, Hq, max_len); }, "masks of half a word");
  refuses([&] { ops::attention_tree_paged_fp8(ctx, q, kp[0], vp[0], ks[0], vs[0], table, starts, lens, tmask, q, Hq, max_len + 1); }, "more rows than the table");
  refuses([&] { ops::prepare_qkv_paged_fp8(ctx, q, k, k, kp[0], vp[0], ks[0], vs[0], slots, tpos, &q, &twk, q, Hq, rot, theta, eps); }, "a norm of another size");
  refuses([&] { ops::prepare_qkv_paged_fp8(ctx, q, k, k, kp[0], vp[0], ks[0], vs[0], slots, tpos, &twq, &twk, q, Hq, rot + 2, theta, eps); }, "pairs that are no multiple of 8");
  refuses([&] { ops::prepare_qkv_paged_fp8(ctx, q, k, k, kp[0], vp[0], ks[0], vs[0], slots, kept_lens, &twq, &twk, q, Hq, rot, theta, eps); }, "too few positions");
  refuses([&] { ops::kv_keep_paged_fp8(ctx, {}, table, cached, kept, kept_lens, now); }, "no layers");
  refuses([&] { ops::kv_keep_paged_fp8(ctx, layers, table, cached, kept, kept_lens, cached); }, "lengths over lengths");
  layers.push_back({&small, &small, &small_scale, &small_scale});
  refuses([&] { ops::kv_copy_paged_fp8(ctx, layers, table, from, to, count, max_len); }, "layers of different pages");
  std::printf(g_fail ? "%d FAILED\n" : "ALL OK\n", g_fail);
  return g_fail ? 1 : 0;
}
