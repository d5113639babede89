// What the ops:: forms of the draft operators refuse before any device work: runs
// on the host alone, over addresses that are never read. Exit code 0 = all passed.
#include <cstdio>
#include <cstring>
#include <stdexcept>

#include "Ops.hpp"

static int g_fail = 0;
template <typename F>
static void refuses(F&& f, const char* why) {
  std::string got = "no refusal";
  try {
    f();
  } catch (const std::runtime_error& e) {
    got = e.what();
  }
  const bool ok = got.find(why) != std::string::npos;
  std::printf("%-28s %s (%s)\n", why, ok ? "OK" : "FAIL", got.c_str());
  if (!ok) ++g_fail;
}

int main() {
  Context ctx(nullptr);
  const int T = 5, Hq = 4, Hkv = 2, D = 128, page = 32, P = 6, rot = 64;
  char* at = reinterpret_cast<char*>(size_t{1} << 20);
  const auto tensor = [&](std::vector<int64_t> shape, DType dt) {
    Tensor t = Tensor::view(ctx, at, shape, dt);
    at += size_t{1} << 20;
    return t;
  };
  Tensor q = tensor({T, Hq * D}, DType::bf16), k = tensor({T, Hkv * D}, DType::bf16), v = tensor({T, Hkv * D}, DType::bf16);
  Tensor out = tensor({T, Hq * D}, DType::bf16), norm = tensor({D}, DType::bf16);
  Tensor kp = tensor({P, Hkv, page, D}, DType::u8), vp = tensor({P, Hkv, page, D}, DType::u8);
  Tensor ks = tensor({P, Hkv, page / 16}, DType::f32), vs = tensor({P, Hkv, page / 16}, DType::f32);
  Tensor slots = tensor({T}, DType::s32), pos = tensor({3, T}, DType::s32), wrong = tensor({2, T}, DType::s32);
  const auto prepare = [&](Tensor& positions, auto... sections) {
    ops::prepare_qkv_paged_fp8(ctx, q, k, v, kp, vp, ks, vs, slots, positions, &norm, &norm, out, Hq, rot, 1e4f, 1e-6f, sections...);
  };
  refuses([&] { prepare(pos); }, "need section_h and section_w");
  refuses([&] { prepare(pos, 0, 10); }, "need section_h and section_w");
  refuses([&] { prepare(pos, 0, -1, 10); }, "need section_h and section_w");
  refuses([&] { prepare(wrong, 0, 10, 10); }, "positions");
  std::printf(g_fail ? "%d FAILED\n" : "ALL OK\n", g_fail);
  return g_fail ? 1 : 0;
}
