// ops:: over the C ABI (see Ops.hpp).
#include "Ops.hpp"

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <stdexcept>
#include <string>

#include "aila_hip.h"

namespace ops {
namespace {

void check(int rc, const char* what) {
  if (rc != AILA_HIP_OK)
    throw std::runtime_error(std::string(what) + ": " + aila_hip_last_error());
}

void need_dtype(const Tensor& t, DType dt, const char* name) {
  if (!t.valid()) throw std::runtime_error(std::string(name) + ": invalid tensor");
  if (t.dtype() != dt) throw std::runtime_error(std::string(name) + ": wrong dtype");
}

}  // namespace

void copy_to_cache(Context& ctx, Tensor& new_kv, Tensor& cache, int seq_len, int start_pos,
                   int num_heads, int head_dim, int max_seq_len) {
  need_dtype(new_kv, DType::bf16, "copy_to_cache new_kv");
  need_dtype(cache, DType::bf16, "copy_to_cache cache");
  check(aila_hip_copy_to_cache(new_kv.data(), cache.data(), seq_len, start_pos, num_heads, head_dim,
                               max_seq_len, ctx.stream()),
        "copy_to_cache");
}

namespace {
int env_int(const char* name, int dflt) {
  const char* v = std::getenv(name);
  if (v == nullptr || *v == '\0') return dflt;
  char* end = nullptr;
  const long x = std::strtol(v, &end, 10);
  return end && *end == '\0' ? static_cast<int>(x) : dflt;
}
}  // namespace

void attention_decode(Context& ctx, Tensor& q, Tensor& k_cache, Tensor& v_cache, Tensor& output,
                      Tensor& scores_buf, int num_heads, int num_kv_heads, int head_dim,
                      int cached_len, Tensor* exact_partials_buf) {
  // The reference's decode window knobs, read once (AttentionOps.cpp:517-551).
  static const int window = std::max(0, env_int("AILA_ATTN_DECODE_WINDOW", 0));
  static const int window_start = env_int("AILA_ATTN_DECODE_WINDOW_START", -1);
  static const int sink = std::max(0, env_int("AILA_ATTN_DECODE_SINK", 0));
  attention_decode_window(ctx, q, k_cache, v_cache, output, scores_buf, num_heads, num_kv_heads, head_dim,
                          cached_len, exact_partials_buf, window, window_start, sink);
}

void attention_decode_window(Context& ctx, Tensor& q, Tensor& k_cache, Tensor& v_cache, Tensor& output,
                             Tensor& scores_buf, int num_heads, int num_kv_heads, int head_dim, int cached_len,
                             Tensor* exact_partials_buf, int window, int window_start, int sink) {
  (void)scores_buf;
  need_dtype(q, DType::bf16, "attention_decode q");
  need_dtype(k_cache, DType::bf16, "attention_decode k_cache");
  need_dtype(v_cache, DType::bf16, "attention_decode v_cache");
  need_dtype(output, DType::bf16, "attention_decode output");
  const int max_seq = static_cast<int>(k_cache.shape(1));
  void* ws = nullptr;
  size_t ws_bytes = 0;
  if (exact_partials_buf && exact_partials_buf->valid()) {
    ws = exact_partials_buf->data();
    ws_bytes = exact_partials_buf->size_bytes();
    // a buffer too small for two records per head falls back to one pass
    if (ws_bytes < 2 * static_cast<size_t>(num_heads) * (16 + head_dim) * sizeof(float)) {
      ws = nullptr;
      ws_bytes = 0;
    }
  }
  if (window > 0)
    check(aila_hip_gqa_decode_window(q.data(), k_cache.data(), v_cache.data(), output.data(), ws, ws_bytes, 1,
                                     num_heads, num_kv_heads, head_dim, max_seq, cached_len, nullptr, window,
                                     window_start, sink, ctx.stream()),
          "attention_decode");
  else
    check(aila_hip_gqa_decode(q.data(), k_cache.data(), v_cache.data(), output.data(), ws, ws_bytes, 1,
                              num_heads, num_kv_heads, head_dim, max_seq, cached_len, nullptr,
                              ctx.stream()),
          "attention_decode");
}

void attention_decode_paged(Context& ctx, Tensor& q, Tensor& k_pages, Tensor& v_pages, Tensor& block_table,
                            Tensor& seq_lens, Tensor& output, int num_heads, int num_kv_heads, int head_dim,
                            int max_len, Tensor* exact_partials_buf) {
  need_dtype(q, DType::bf16, "attention_decode_paged q");
  need_dtype(k_pages, DType::bf16, "attention_decode_paged k_pages");
  need_dtype(v_pages, DType::bf16, "attention_decode_paged v_pages");
  need_dtype(output, DType::bf16, "attention_decode_paged output");
  need_dtype(block_table, DType::s32, "attention_decode_paged block_table");
  need_dtype(seq_lens, DType::s32, "attention_decode_paged seq_lens");
  const int B = static_cast<int>(block_table.shape(0));
  const int max_pages = static_cast<int>(block_table.shape(1));
  const int page_size = static_cast<int>(k_pages.shape(2));
  void* ws = nullptr;
  size_t ws_bytes = 0;
  if (exact_partials_buf && exact_partials_buf->valid() &&
      exact_partials_buf->size_bytes() >= 2 * static_cast<size_t>(B) * num_heads * (16 + head_dim) * sizeof(float)) {
    ws = exact_partials_buf->data();
    ws_bytes = exact_partials_buf->size_bytes();
  }
  check(aila_hip_gqa_decode_paged(q.data(), k_pages.data(), v_pages.data(), output.data(), ws, ws_bytes, B,
                                  num_heads, num_kv_heads, head_dim, page_size,
                                  static_cast<const int*>(block_table.data()), max_pages, max_len,
                                  static_cast<const int*>(seq_lens.data()), ctx.stream()),
        "attention_decode_paged");
}

namespace {

const int* s32(const Tensor& t, const char* name, int64_t least) {
  need_dtype(t, DType::s32, name);
  if (t.numel() < least) throw std::runtime_error(std::string(name) + ": too few elements");
  return static_cast<const int*>(t.data());
}

// An 8-bit paged cache's sizes, checked against each other.
struct PagesFp8 {
  int num_pages, Hkv, page_size, D;
  const float *k_scale, *v_scale;
};
PagesFp8 pages_fp8(const Tensor& k_pages, const Tensor& v_pages, const Tensor& k_scale, const Tensor& v_scale,
                   const char* what) {
  need_dtype(k_pages, DType::u8, what);
  need_dtype(v_pages, DType::u8, what);
  need_dtype(k_scale, DType::f32, what);
  need_dtype(v_scale, DType::f32, what);
  if (k_pages.ndim() != 4 || v_pages.shape() != k_pages.shape())
    throw std::runtime_error(std::string(what) + ": k_pages and v_pages must be [num_pages, Hkv, page_size, D]");
  const PagesFp8 p{static_cast<int>(k_pages.shape(0)), static_cast<int>(k_pages.shape(1)), static_cast<int>(k_pages.shape(2)),
                   static_cast<int>(k_pages.shape(3)), static_cast<const float*>(k_scale.data()),
                   static_cast<const float*>(v_scale.data())};
  const std::vector<int64_t> want = {p.num_pages, p.Hkv, p.page_size / 16};
  if (k_scale.shape() != want || v_scale.shape() != want)
    throw std::runtime_error(std::string(what) + ": k_scale and v_scale must be [num_pages, Hkv, page_size / 16]");
  return p;
}

// Tokens of a [T, width] bf16 tensor.
int rows_of(const Tensor& t, int64_t width, const char* name) {
  need_dtype(t, DType::bf16, name);
  if (t.ndim() < 1 || t.numel() != t.shape(0) * width) throw std::runtime_error(std::string(name) + ": wrong row size");
  return static_cast<int>(t.shape(0));
}

}  // namespace

void kv_pages_reserve(Context& ctx, Tensor& cached_lens, Tensor& new_lens, Tensor& block_table, Tensor& free_pages,
                      Tensor& free_count, int page_size, Tensor& slots, Tensor& query_start, Tensor& seq_lens) {
  need_dtype(block_table, DType::s32, "kv_pages_reserve block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("kv_pages_reserve block_table: must be [B, max_pages]");
  const int B = static_cast<int>(block_table.shape(0));
  const int* cached = s32(cached_lens, "kv_pages_reserve cached_lens", B);
  const int* fresh = s32(new_lens, "kv_pages_reserve new_lens", B);
  const int* pool = s32(free_pages, "kv_pages_reserve free_pages", 1);
  s32(free_count, "kv_pages_reserve free_count", 1);
  s32(slots, "kv_pages_reserve slots", 1);
  s32(query_start, "kv_pages_reserve query_start", B + 1);
  s32(seq_lens, "kv_pages_reserve seq_lens", B);
  check(aila_hip_kv_pages_reserve(cached, fresh, block_table.data_as<int>(), pool, free_count.data_as<int>(),
                                  query_start.data_as<int>(), seq_lens.data_as<int>(), slots.data_as<int>(), B,
                                  static_cast<int>(block_table.shape(1)), page_size, static_cast<int>(free_pages.numel()),
                                  static_cast<int>(slots.numel()), ctx.stream()),
        "kv_pages_reserve");
}

void kv_pages_release(Context& ctx, Tensor& ended, Tensor& block_table, Tensor& free_pages, Tensor& free_count) {
  need_dtype(block_table, DType::s32, "kv_pages_release block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("kv_pages_release block_table: must be [B, max_pages]");
  const int B = static_cast<int>(block_table.shape(0));
  const int* flags = s32(ended, "kv_pages_release ended", B);
  s32(free_pages, "kv_pages_release free_pages", 1);
  s32(free_count, "kv_pages_release free_count", 1);
  check(aila_hip_kv_pages_release(flags, block_table.data_as<int>(), free_pages.data_as<int>(), free_count.data_as<int>(), B,
                                  static_cast<int>(block_table.shape(1)), static_cast<int>(free_pages.numel()), ctx.stream()),
        "kv_pages_release");
}

void copy_to_cache_paged_fp8(Context& ctx, Tensor& new_k, Tensor& new_v, Tensor& k_pages, Tensor& v_pages,
                             Tensor& k_scale, Tensor& v_scale, Tensor& slots) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "copy_to_cache_paged_fp8");
  const int T = rows_of(new_k, int64_t{p.Hkv} * p.D, "copy_to_cache_paged_fp8 new_k");
  if (rows_of(new_v, int64_t{p.Hkv} * p.D, "copy_to_cache_paged_fp8 new_v") != T)
    throw std::runtime_error("copy_to_cache_paged_fp8: new_k and new_v differ in rows");
  check(aila_hip_kv_append_paged_fp8(new_k.data(), new_v.data(), static_cast<long>(p.Hkv) * p.D, k_pages.data(), v_pages.data(),
                                     k_scale.data_as<float>(), v_scale.data_as<float>(),
                                     s32(slots, "copy_to_cache_paged_fp8 slots", T), T, p.Hkv, p.D, p.page_size, p.num_pages,
                                     ctx.stream()),
        "copy_to_cache_paged_fp8");
}

void read_cache_paged_fp8(Context& ctx, Tensor& k_pages, Tensor& v_pages, Tensor& k_scale, Tensor& v_scale,
                          Tensor& slots, Tensor& k_out, Tensor& v_out) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "read_cache_paged_fp8");
  const int T = rows_of(k_out, int64_t{p.Hkv} * p.D, "read_cache_paged_fp8 k_out");
  if (rows_of(v_out, int64_t{p.Hkv} * p.D, "read_cache_paged_fp8 v_out") != T)
    throw std::runtime_error("read_cache_paged_fp8: k_out and v_out differ in rows");
  check(aila_hip_kv_read_paged_fp8(k_pages.data(), v_pages.data(), p.k_scale, p.v_scale, s32(slots, "read_cache_paged_fp8 slots", T),
                                   k_out.data(), v_out.data(), T, p.Hkv, p.D, p.page_size, p.num_pages, ctx.stream()),
        "read_cache_paged_fp8");
}

void attention_decode_paged_fp8(Context& ctx, Tensor& q, Tensor& k_pages, Tensor& v_pages, Tensor& k_scale,
                                Tensor& v_scale, Tensor& block_table, Tensor& seq_lens, Tensor& output, int num_heads,
                                int max_len, Tensor* workspace) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "attention_decode_paged_fp8");
  const int B = rows_of(q, int64_t{num_heads} * p.D, "attention_decode_paged_fp8 q");
  if (rows_of(output, int64_t{num_heads} * p.D, "attention_decode_paged_fp8 output") != B)
    throw std::runtime_error("attention_decode_paged_fp8: q and output differ in rows");
  need_dtype(block_table, DType::s32, "attention_decode_paged_fp8 block_table");
  if (block_table.ndim() != 2 || block_table.shape(0) != B)
    throw std::runtime_error("attention_decode_paged_fp8 block_table: must be [B, max_pages]");
  const bool ws = workspace && workspace->valid();
  check(aila_hip_gqa_decode_paged_fp8(q.data(), static_cast<long>(num_heads) * p.D, k_pages.data(), v_pages.data(), p.k_scale,
                                      p.v_scale, output.data(), ws ? workspace->data() : nullptr,
                                      ws ? workspace->size_bytes() : 0, B, num_heads, p.Hkv, p.D, p.page_size, p.num_pages,
                                      block_table.data_as<int>(), static_cast<int>(block_table.shape(1)), max_len,
                                      s32(seq_lens, "attention_decode_paged_fp8 seq_lens", B), ctx.stream()),
        "attention_decode_paged_fp8");
}

void attention_prefill_paged_fp8(Context& ctx, Tensor& q, Tensor& k_pages, Tensor& v_pages, Tensor& k_scale,
                                 Tensor& v_scale, Tensor& block_table, Tensor& query_start, Tensor& seq_lens,
                                 Tensor& output, int num_heads, int max_len, Tensor* workspace) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "attention_prefill_paged_fp8");
  const int T = rows_of(q, int64_t{num_heads} * p.D, "attention_prefill_paged_fp8 q");
  if (rows_of(output, int64_t{num_heads} * p.D, "attention_prefill_paged_fp8 output") != T)
    throw std::runtime_error("attention_prefill_paged_fp8: q and output differ in rows");
  need_dtype(block_table, DType::s32, "attention_prefill_paged_fp8 block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("attention_prefill_paged_fp8 block_table: must be [B, max_pages]");
  const int B = static_cast<int>(block_table.shape(0));
  const bool ws = workspace && workspace->valid();
  check(aila_hip_gqa_prefill_paged_fp8(q.data(), static_cast<long>(num_heads) * p.D, k_pages.data(), v_pages.data(), p.k_scale,
                                       p.v_scale, output.data(), ws ? workspace->data() : nullptr,
                                       ws ? workspace->size_bytes() : 0, T, B, num_heads, p.Hkv, p.D, p.page_size, p.num_pages,
                                       block_table.data_as<int>(), static_cast<int>(block_table.shape(1)), max_len,
                                       s32(query_start, "attention_prefill_paged_fp8 query_start", B + 1),
                                       s32(seq_lens, "attention_prefill_paged_fp8 seq_lens", B), ctx.stream()),
        "attention_prefill_paged_fp8");
}

void prepare_qkv_paged_fp8(Context& ctx, Tensor& q, Tensor& new_k, Tensor& new_v, Tensor& k_pages, Tensor& v_pages,
                           Tensor& k_scale, Tensor& v_scale, Tensor& slots, Tensor& positions, Tensor* q_norm,
                           Tensor* k_norm, Tensor& q_out, int num_heads, int rotary_dim, float theta, float eps,
                           int q_head_stride, int section_h, int section_w, Tensor* inv_freq) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "prepare_qkv_paged_fp8");
  const int64_t step = q_head_stride ? q_head_stride : p.D, q_row = num_heads * step, row = int64_t{p.Hkv} * p.D;
  const int T = rows_of(q, q_row, "prepare_qkv_paged_fp8 q");
  if (rows_of(new_k, row, "prepare_qkv_paged_fp8 new_k") != T || rows_of(new_v, row, "prepare_qkv_paged_fp8 new_v") != T ||
      rows_of(q_out, int64_t{num_heads} * p.D, "prepare_qkv_paged_fp8 q_out") != T)
    throw std::runtime_error("prepare_qkv_paged_fp8: q, new_k, new_v and q_out differ in rows");
  for (Tensor* w : {q_norm, k_norm})
    if (w && w->valid() && rows_of(*w, 1, "prepare_qkv_paged_fp8 norm") != p.D)
      throw std::runtime_error("prepare_qkv_paged_fp8: q_norm and k_norm must be [D]");
  const bool freqs = inv_freq && inv_freq->valid();
  if (freqs) {
    need_dtype(*inv_freq, DType::f32, "prepare_qkv_paged_fp8 inv_freq");
    if (inv_freq->numel() < rotary_dim / 2) throw std::runtime_error("prepare_qkv_paged_fp8 inv_freq: too few elements");
  }
  const int* pos = nullptr;
  bool streams = false;
  if (rotary_dim != 0) {
    streams = positions.ndim() == 2;
    pos = s32(positions, "prepare_qkv_paged_fp8 positions", streams ? 3 * int64_t{T} : T);
    if (streams && (positions.shape(0) != 3 || positions.shape(1) != T))
      throw std::runtime_error("prepare_qkv_paged_fp8 positions: must be [T] or [3, T]");
    if (streams && (section_h < 0 || section_w < 0))
      throw std::runtime_error("prepare_qkv_paged_fp8: positions [3, T] need section_h and section_w");
  }
  check(aila_hip_prepare_qkv_paged_fp8(
            q.data(), q_row, step, new_k.data(), row, new_v.data(), row, q_out.data(),
            q_norm && q_norm->valid() ? q_norm->data() : nullptr, k_norm && k_norm->valid() ? k_norm->data() : nullptr,
            k_pages.data(), v_pages.data(), k_scale.data_as<float>(), v_scale.data_as<float>(),
            s32(slots, "prepare_qkv_paged_fp8 slots", T), pos, streams ? pos + T : nullptr, streams ? pos + 2 * int64_t{T} : nullptr,
            streams ? section_h : 0, streams ? section_w : 0, T, num_heads, p.Hkv, p.D, p.page_size, p.num_pages, rotary_dim, theta,
            freqs ? inv_freq->data_as<float>() : nullptr, eps, ctx.stream()),
        "prepare_qkv_paged_fp8");
}

void attention_tree_paged_fp8(Context& ctx, Tensor& q, Tensor& k_pages, Tensor& v_pages, Tensor& k_scale,
                              Tensor& v_scale, Tensor& block_table, Tensor& query_start, Tensor& seq_lens,
                              Tensor& tree_mask, Tensor& output, int num_heads, int max_len, Tensor* workspace) {
  const PagesFp8 p = pages_fp8(k_pages, v_pages, k_scale, v_scale, "attention_tree_paged_fp8");
  const int T = rows_of(q, int64_t{num_heads} * p.D, "attention_tree_paged_fp8 q");
  if (rows_of(output, int64_t{num_heads} * p.D, "attention_tree_paged_fp8 output") != T)
    throw std::runtime_error("attention_tree_paged_fp8: q and output differ in rows");
  need_dtype(block_table, DType::s32, "attention_tree_paged_fp8 block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("attention_tree_paged_fp8 block_table: must be [B, max_pages]");
  need_dtype(tree_mask, DType::s32, "attention_tree_paged_fp8 tree_mask");
  if (tree_mask.ndim() != 2 || tree_mask.shape(0) != T || tree_mask.shape(1) % 2)
    throw std::runtime_error("attention_tree_paged_fp8 tree_mask: must be [T, 2 * mask_words]");
  const int B = static_cast<int>(block_table.shape(0));
  const bool ws = workspace && workspace->valid();
  check(aila_hip_gqa_tree_paged_fp8(q.data(), static_cast<long>(num_heads) * p.D, k_pages.data(), v_pages.data(), p.k_scale,
                                    p.v_scale, output.data(), ws ? workspace->data() : nullptr, ws ? workspace->size_bytes() : 0,
                                    T, B, num_heads, p.Hkv, p.D, p.page_size, p.num_pages, block_table.data_as<int>(),
                                    static_cast<int>(block_table.shape(1)), max_len,
                                    s32(query_start, "attention_tree_paged_fp8 query_start", B + 1),
                                    s32(seq_lens, "attention_tree_paged_fp8 seq_lens", B), tree_mask.data(),
                                    static_cast<int>(tree_mask.shape(1) / 2), ctx.stream()),
        "attention_tree_paged_fp8");
}

namespace {

// The layers' pointers, every layer checked to have the first one's sizes.
struct LayersFp8 {
  PagesFp8 p;
  std::vector<void*> k, v;
  std::vector<float*> ks, vs;
};
LayersFp8 layers_fp8(const std::vector<PagedLayerFp8>& layers, const char* what) {
  LayersFp8 out{};
  for (const auto& l : layers) {
    if (!l.k_pages || !l.v_pages || !l.k_scale || !l.v_scale) throw std::runtime_error(std::string(what) + ": a layer lacks a tensor");
    const PagesFp8 p = pages_fp8(*l.k_pages, *l.v_pages, *l.k_scale, *l.v_scale, what);
    if (l.k_pages->shape() != layers[0].k_pages->shape()) throw std::runtime_error(std::string(what) + ": layers differ in shape");
    out.p = p;
    out.k.push_back(l.k_pages->data());
    out.v.push_back(l.v_pages->data());
    out.ks.push_back(l.k_scale->data_as<float>());
    out.vs.push_back(l.v_scale->data_as<float>());
  }
  if (layers.empty()) throw std::runtime_error(std::string(what) + ": no layers");
  return out;
}

}  // namespace

void kv_keep_paged_fp8(Context& ctx, const std::vector<PagedLayerFp8>& layers, Tensor& block_table, Tensor& cached_lens,
                       Tensor& kept, Tensor& kept_lens, Tensor& lens) {
  const LayersFp8 l = layers_fp8(layers, "kv_keep_paged_fp8");
  need_dtype(block_table, DType::s32, "kv_keep_paged_fp8 block_table");
  need_dtype(kept, DType::s32, "kv_keep_paged_fp8 kept");
  if (block_table.ndim() != 2 || kept.ndim() != 2 || kept.shape(0) != block_table.shape(0))
    throw std::runtime_error("kv_keep_paged_fp8: block_table must be [B, max_pages], kept [B, max_kept]");
  const int B = static_cast<int>(block_table.shape(0));
  s32(lens, "kv_keep_paged_fp8 lens", B);
  check(aila_hip_kv_keep_paged_fp8(l.k.data(), l.v.data(), l.ks.data(), l.vs.data(), static_cast<int>(layers.size()),
                                   block_table.data_as<int>(), s32(cached_lens, "kv_keep_paged_fp8 cached_lens", B),
                                   kept.data_as<int>(), s32(kept_lens, "kv_keep_paged_fp8 kept_lens", B), lens.data_as<int>(), B,
                                   static_cast<int>(kept.shape(1)), l.p.Hkv, l.p.D, l.p.page_size, l.p.num_pages,
                                   static_cast<int>(block_table.shape(1)), ctx.stream()),
        "kv_keep_paged_fp8");
}

void kv_pages_trim(Context& ctx, Tensor& lens, Tensor& block_table, Tensor& free_pages, Tensor& free_count, int page_size) {
  need_dtype(block_table, DType::s32, "kv_pages_trim block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("kv_pages_trim block_table: must be [B, max_pages]");
  const int B = static_cast<int>(block_table.shape(0));
  s32(free_pages, "kv_pages_trim free_pages", 1);
  s32(free_count, "kv_pages_trim free_count", 1);
  check(aila_hip_kv_pages_trim(s32(lens, "kv_pages_trim lens", B), block_table.data_as<int>(), free_pages.data_as<int>(),
                               free_count.data_as<int>(), B, static_cast<int>(block_table.shape(1)), page_size,
                               static_cast<int>(free_pages.numel()), ctx.stream()),
        "kv_pages_trim");
}

void kv_copy_paged_fp8(Context& ctx, const std::vector<PagedLayerFp8>& layers, Tensor& block_table, Tensor& src,
                       Tensor& dst, Tensor& lens, int max_len) {
  const LayersFp8 l = layers_fp8(layers, "kv_copy_paged_fp8");
  need_dtype(block_table, DType::s32, "kv_copy_paged_fp8 block_table");
  if (block_table.ndim() != 2) throw std::runtime_error("kv_copy_paged_fp8 block_table: must be [B, max_pages]");
  const int n = static_cast<int>(src.numel());
  check(aila_hip_kv_copy_paged_fp8(l.k.data(), l.v.data(), l.ks.data(), l.vs.data(), static_cast<int>(layers.size()),
                                   block_table.data_as<int>(), s32(src, "kv_copy_paged_fp8 src", n),
                                   s32(dst, "kv_copy_paged_fp8 dst", n), s32(lens, "kv_copy_paged_fp8 lens", n), n, max_len,
                                   static_cast<int>(block_table.shape(0)), l.p.Hkv, l.p.D, l.p.page_size, l.p.num_pages,
                                   static_cast<int>(block_table.shape(1)), ctx.stream()),
        "kv_copy_paged_fp8");
}

void attention_prefill(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& output,
                       Tensor& scores_buf, int seq_len, int num_heads, int num_kv_heads,
                       int head_dim) {
  (void)scores_buf;
  need_dtype(q, DType::bf16, "attention_prefill q");
  check(aila_hip_gqa_prefill(q.data(), k.data(), v.data(), output.data(), nullptr, nullptr, 0, 0, seq_len,
                             num_heads, num_kv_heads, head_dim, ctx.stream()),
        "attention_prefill");
}

void attention_prefill_write_cache(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& output,
                                   Tensor& k_cache, Tensor& v_cache, int seq_len, int start_pos,
                                   int num_heads, int num_kv_heads, int head_dim, int max_seq_len) {
  need_dtype(q, DType::bf16, "attention_prefill_write_cache q");
  check(aila_hip_gqa_prefill(q.data(), k.data(), v.data(), output.data(), k_cache.data(), v_cache.data(),
                             start_pos, max_seq_len, seq_len, num_heads, num_kv_heads, head_dim,
                             ctx.stream()),
        "attention_prefill_write_cache");
}

void attention_prefill_cached(Context& ctx, Tensor& q, Tensor& k_cache, Tensor& v_cache,
                              Tensor& output, Tensor& scores_buf, int seq_len, int start_pos,
                              int num_heads, int num_kv_heads, int head_dim, int max_seq_len) {
  need_dtype(q, DType::bf16, "attention_prefill_cached q");
  // The reference's score buffer ([heads, seq, total] fp32, never
  // materialised here) serves as the key-split workspace.
  const bool ws = scores_buf.valid();
  check(aila_hip_gqa_prefill_cached_ws(q.data(), k_cache.data(), v_cache.data(), output.data(),
                                       ws ? scores_buf.data() : nullptr, ws ? scores_buf.size_bytes() : 0, seq_len,
                                       start_pos, num_heads, num_kv_heads, head_dim, max_seq_len, ctx.stream()),
        "attention_prefill_cached");
}

void linear_delta_decode(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& a, Tensor& b,
                         Tensor* dt_bias, Tensor* A_log, Tensor& state, Tensor& out,
                         int num_k_heads, int num_v_heads, int head_k_dim, int head_v_dim,
                         float eps, float scale) {
  need_dtype(state, DType::f32, "linear_delta_decode state");
  const int B = state.ndim() == 4 ? static_cast<int>(state.shape(0)) : 1;
  check(aila_hip_deltanet_decode(q.data(), k.data(), v.data(), a.data(), b.data(),
                                 dt_bias ? dt_bias->data() : nullptr,
                                 A_log ? static_cast<const float*>(A_log->data()) : nullptr,
                                 static_cast<float*>(state.data()), out.data(), B, num_k_heads,
                                 num_v_heads, head_k_dim, head_v_dim, eps, scale, ctx.stream()),
        "linear_delta_decode");
}

size_t linear_delta_prefill_workspace_bytes(int seq_len, int num_v_heads, int head_k_dim,
                                            int head_v_dim) {
  return aila_hip_deltanet_prefill_workspace_size(1, seq_len, num_v_heads, head_k_dim, head_v_dim);
}

void linear_delta_prefill(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& a, Tensor& b,
                          Tensor* dt_bias, Tensor* A_log, Tensor& state, Tensor& out,
                          Tensor& workspace, int seq_len, int num_k_heads, int num_v_heads,
                          int head_k_dim, int head_v_dim, float eps, float scale) {
  need_dtype(state, DType::f32, "linear_delta_prefill state");
  check(aila_hip_deltanet_prefill(q.data(), k.data(), v.data(), a.data(), b.data(),
                                  dt_bias ? dt_bias->data() : nullptr,
                                  A_log ? static_cast<const float*>(A_log->data()) : nullptr,
                                  static_cast<float*>(state.data()), out.data(), workspace.data(),
                                  workspace.size_bytes(), 1, seq_len, num_k_heads, num_v_heads,
                                  head_k_dim, head_v_dim, eps, scale, ctx.stream()),
        "linear_delta_prefill");
}

namespace {

void* opt(Tensor& t) { return t.valid() ? t.data() : nullptr; }

// The reference's rotary position arguments (ElementwiseOps.cpp:33-103,
// 555-863) as the C ABI's position record. The position streams are the
// engine's device arrays, indexed by cache row.
aila_hip_rope_pos rope_pos(bool interleaved, const int* pos_t, const int* pos_h, const int* pos_w,
                           int prompt_pos_len, int text_pos_delta, int sec_t, int sec_h, int sec_w) {
  aila_hip_rope_pos rp{};
  rp.interleaved = interleaved ? 1 : 0;
  rp.pos_t = pos_t;
  rp.pos_h = pos_h;
  rp.pos_w = pos_w;
  rp.pos_stride = 0;
  rp.prompt_pos_len = prompt_pos_len;
  rp.text_pos_delta = text_pos_delta;
  rp.mrope_section_t = sec_t;
  rp.mrope_section_h = sec_h;
  rp.mrope_section_w = sec_w;
  return rp;
}

}  // namespace

void head_rms_norm(Context& ctx, Tensor& x, Tensor& weight, float eps, int seq_len, int num_heads,
                   int head_dim) {
  need_dtype(x, DType::bf16, "head_rms_norm x");
  if (weight.valid()) need_dtype(weight, DType::bf16, "head_rms_norm weight");
  check(aila_hip_head_rms_norm(x.data(), opt(weight), seq_len, num_heads, head_dim, eps, ctx.stream()),
        "head_rms_norm");
}

void sigmoid_mul(Context& ctx, Tensor& input, Tensor& gate, Tensor& output, int n) {
  need_dtype(input, DType::bf16, "sigmoid_mul input");
  need_dtype(gate, DType::bf16, "sigmoid_mul gate");
  need_dtype(output, DType::bf16, "sigmoid_mul output");
  check(aila_hip_sigmoid_mul(input.data(), gate.data(), output.data(), n, ctx.stream()), "sigmoid_mul");
}

void apply_rope(Context& ctx, Tensor& q, Tensor& k, int seq_len, int start_pos, int num_heads_q,
                int num_kv_heads, int head_dim, float theta) {
  apply_rope_partial(ctx, q, k, seq_len, start_pos, num_heads_q, num_kv_heads, head_dim, head_dim, theta);
}

void apply_rope_partial(Context& ctx, Tensor& q, Tensor& k, int seq_len, int start_pos, int num_heads_q,
                        int num_kv_heads, int head_dim, int rotary_dim, float theta, bool interleaved,
                        const int* pos_t, const int* pos_h, const int* pos_w, int prompt_pos_len,
                        int text_pos_delta, int mrope_section_t, int mrope_section_h, int mrope_section_w) {
  need_dtype(q, DType::bf16, "apply_rope q");
  need_dtype(k, DType::bf16, "apply_rope k");
  const aila_hip_rope_pos rp = rope_pos(interleaved, pos_t, pos_h, pos_w, prompt_pos_len, text_pos_delta,
                                        mrope_section_t, mrope_section_h, mrope_section_w);
  check(aila_hip_apply_rope(q.data(), k.data(), seq_len, start_pos, num_heads_q, num_kv_heads, head_dim, rotary_dim,
                            theta, &rp, ctx.stream()),
        "apply_rope_partial");
}

void decode_prepare_qkv(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& rope_freq,
                        Tensor& q_norm_weight, Tensor& k_norm_weight, Tensor& k_cache, Tensor& v_cache,
                        int start_pos, int num_heads_q, int num_kv_heads, int head_dim, float eps,
                        float theta) {
  // angle = start_pos * rope_freq[d] (ElementwiseOps.cpp:159, 198): the
  // table is used as given (an invalid tensor falls back to theta)
  for (Tensor* t : {&q, &k, &v, &k_cache, &v_cache}) need_dtype(*t, DType::bf16, "decode_prepare_qkv");
  aila_hip_rope_pos rp{};
  if (rope_freq.valid()) {
    need_dtype(rope_freq, DType::f32, "decode_prepare_qkv rope_freq");
    if (rope_freq.numel() < head_dim / 2) throw std::runtime_error("decode_prepare_qkv: rope_freq holds < head_dim/2 values");
    rp.inv_freq = rope_freq.data_as<float>();
  }
  check(aila_hip_decode_prepare_qkv(q.data(), 0, q.data(), nullptr, k.data(), v.data(), opt(q_norm_weight),
                                    opt(k_norm_weight), k_cache.data(), v_cache.data(), 1, num_heads_q,
                                    num_kv_heads, head_dim, static_cast<int>(k_cache.shape(1)), head_dim, theta,
                                    eps, start_pos, nullptr, &rp, ctx.stream()),
        "decode_prepare_qkv");
}

void decode_prepare_qkv_partial(Context& ctx, Tensor& q, Tensor& k, Tensor& v, Tensor& q_norm_weight,
                                Tensor& k_norm_weight, Tensor& k_cache, Tensor& v_cache, int start_pos,
                                int num_heads_q, int num_kv_heads, int head_dim, float eps, int rotary_dim,
                                float theta, bool interleaved, const int* pos_t, const int* pos_h,
                                const int* pos_w, int prompt_pos_len, int text_pos_delta, int mrope_section_t,
                                int mrope_section_h, int mrope_section_w) {
  const aila_hip_rope_pos rp = rope_pos(interleaved, pos_t, pos_h, pos_w, prompt_pos_len, text_pos_delta,
                                        mrope_section_t, mrope_section_h, mrope_section_w);
  for (Tensor* t : {&q, &k, &v, &k_cache, &v_cache}) need_dtype(*t, DType::bf16, "decode_prepare_qkv");
  check(aila_hip_decode_prepare_qkv(q.data(), 0, q.data(), nullptr, k.data(), v.data(), opt(q_norm_weight),
                                    opt(k_norm_weight), k_cache.data(), v_cache.data(), 1, num_heads_q,
                                    num_kv_heads, head_dim, static_cast<int>(k_cache.shape(1)), rotary_dim,
                                    theta, eps, start_pos, nullptr, &rp, ctx.stream()),
        "decode_prepare_qkv");
}

void decode_prepare_qgkv_packed_partial(Context& ctx, Tensor& q_gate_packed, Tensor& k, Tensor& v,
                                        Tensor& q_out, Tensor& gate_out, Tensor& q_norm_weight,
                                        Tensor& k_norm_weight, Tensor& k_cache, Tensor& v_cache,
                                        int start_pos, int num_heads_q, int num_kv_heads, int head_dim,
                                        float eps, int rotary_dim, float theta, bool interleaved,
                                        const int* pos_t, const int* pos_h, const int* pos_w,
                                        int prompt_pos_len, int text_pos_delta, int mrope_section_t,
                                        int mrope_section_h, int mrope_section_w) {
  const aila_hip_rope_pos rp = rope_pos(interleaved, pos_t, pos_h, pos_w, prompt_pos_len, text_pos_delta,
                                        mrope_section_t, mrope_section_h, mrope_section_w);
  for (Tensor* t : {&q_gate_packed, &k, &v, &q_out, &gate_out, &k_cache, &v_cache})
    need_dtype(*t, DType::bf16, "decode_prepare_qgkv_packed_partial");
  check(aila_hip_decode_prepare_qkv(q_gate_packed.data(), 1, q_out.data(), gate_out.data(), k.data(), v.data(),
                                    opt(q_norm_weight), opt(k_norm_weight), k_cache.data(), v_cache.data(), 1,
                                    num_heads_q, num_kv_heads, head_dim, static_cast<int>(k_cache.shape(1)),
                                    rotary_dim, theta, eps, start_pos, nullptr, &rp, ctx.stream()),
        "decode_prepare_qgkv_packed_partial");
}

void linear_delta_layer_decode(Context& ctx, Tensor& qkv, Tensor& z, Tensor& a, Tensor& b, Tensor& conv1d_weight,
                               Tensor& conv_state, int& conv_head, Tensor* dt_bias, Tensor* A_log,
                               Tensor& norm_weight, Tensor& state, Tensor& out, int num_k_heads, int num_v_heads,
                               int head_k_dim, int head_v_dim, int conv_kernel, float eps, Tensor* arrivals) {
  for (Tensor* t : {&qkv, &z, &a, &b, &conv1d_weight, &out}) need_dtype(*t, DType::bf16, "linear_delta_layer_decode");
  if (arrivals) need_dtype(*arrivals, DType::s32, "linear_delta_layer_decode arrivals");
  for (Tensor* t : {&conv_state, &state, &norm_weight}) need_dtype(*t, DType::f32, "linear_delta_layer_decode");
  const int ch = 2 * num_k_heads * head_k_dim + num_v_heads * head_v_dim;
  const float scale = 1.0f / std::sqrt(static_cast<float>(head_k_dim));
  check(aila_hip_deltanet_layer_decode(qkv.data(), ch, z.data(), num_v_heads * head_v_dim, a.data(), b.data(),
                                       num_v_heads, conv1d_weight.data(), conv_state.data_as<float>(), conv_head,
                                       nullptr, dt_bias ? dt_bias->data() : nullptr,
                                       A_log ? A_log->data_as<float>() : nullptr, norm_weight.data_as<float>(),
                                       state.data_as<float>(), out.data(), 1, num_k_heads, num_v_heads, head_k_dim,
                                       head_v_dim, conv_kernel, eps, scale,
                                       arrivals ? static_cast<unsigned int*>(arrivals->data()) : nullptr, ctx.stream()),
        "linear_delta_layer_decode");
  if (conv_kernel > 1) conv_head = (conv_head + 1) % (conv_kernel - 1);
}

size_t linear_delta_layer_prefill_workspace_bytes(int seq_len, int num_k_heads, int num_v_heads, int head_k_dim,
                                                  int head_v_dim) {
  return aila_hip_deltanet_layer_prefill_workspace_size(1, seq_len, num_k_heads, num_v_heads, head_k_dim,
                                                        head_v_dim);
}

void linear_delta_layer_prefill(Context& ctx, Tensor& fused_all, Tensor& out, int seq_len, Tensor& conv1d_weight,
                                Tensor& conv_state, int& conv_head, Tensor* dt_bias, Tensor* A_log,
                                Tensor& norm_weight, Tensor& state, Tensor& workspace, int num_k_heads,
                                int num_v_heads, int head_k_dim, int head_v_dim, int conv_kernel, float eps) {
  for (Tensor* t : {&fused_all, &conv1d_weight, &out}) need_dtype(*t, DType::bf16, "linear_delta_layer_prefill");
  for (Tensor* t : {&conv_state, &state, &norm_weight}) need_dtype(*t, DType::f32, "linear_delta_layer_prefill");
  const int ch = 2 * num_k_heads * head_k_dim + num_v_heads * head_v_dim;
  const int zd = num_v_heads * head_v_dim;
  const int all_dim = ch + zd + 2 * num_v_heads;
  const float scale = 1.0f / std::sqrt(static_cast<float>(head_k_dim));
  uint16_t* row = fused_all.data_as<uint16_t>();
  check(aila_hip_deltanet_layer_prefill(row, all_dim, row + ch, all_dim, row + ch + zd, row + ch + zd + num_v_heads,
                                        all_dim, conv1d_weight.data(), conv_state.data_as<float>(), conv_head,
                                        dt_bias ? dt_bias->data() : nullptr, A_log ? A_log->data_as<float>() : nullptr,
                                        norm_weight.data_as<float>(), state.data_as<float>(), out.data(),
                                        workspace.data(), workspace.size_bytes(), 1, seq_len, num_k_heads,
                                        num_v_heads, head_k_dim, head_v_dim, conv_kernel, eps, scale, ctx.stream()),
        "linear_delta_layer_prefill");
  if (conv_kernel > 1) conv_head = (conv_head + seq_len) % (conv_kernel - 1);
}

}  // namespace ops
