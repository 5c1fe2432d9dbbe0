// Torch op registration of the operators of sonar_attention.h, in the library's own namespace `sonar_amd`.  No kernels live
// here: argument checks, the tensors of the results, and the call of the C ABI on the current stream of the inputs' device.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/EmptyTensor.h>
#include <hip/hip_runtime_api.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "sonar_attention.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void raise_if_failed(int rc) {
  if (rc != SONAR_OK) TORCH_CHECK(false, sonar_attention_last_error());
}

void* current_stream(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

int dtype_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kHalf) return SONAR_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return SONAR_DTYPE_BF16;
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float16, bfloat16 or float32; got ", t.scalar_type());
  return SONAR_DTYPE_F32;
}

Tensor new_tensor(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, at::kStrided, t.device(), std::nullopt, std::nullopt);
}

// The heads (tokens, heads, dim) of a tensor, each one's numbers behind each other: `t` itself where its strides say so, else a
// copy.  A stride that nothing is multiplied by counts as that of a tensor without gaps.
struct Heads {
  Tensor t;
  int64_t token_stride, head_stride;
  Heads(const Tensor& x, bool aligned) : t(x) {
    auto fits = [&] { return (x.size(2) <= 1 || x.stride(2) == 1) && (!aligned || ((uintptr_t)x.const_data_ptr() % 16 == 0 &&
                             (x.size(0) <= 1 || x.stride(0) % 8 == 0) && (x.size(1) <= 1 || x.stride(1) % 8 == 0))); };
    if (x.numel() > 0 && !fits()) t = x.clone(at::MemoryFormat::Contiguous);
    head_stride = t.size(1) > 1 ? t.stride(1) : t.size(2);
    token_stride = t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
  }
};

void check_heads(const Tensor& t, const Tensor& like, int64_t tokens, int64_t dim, const char* name) {
  TORCH_CHECK(t.dim() == 3 && t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.size(0) == tokens &&
                  t.size(1) >= 1 && t.size(2) == dim, name, " must be (", tokens, ", heads, ", dim, ") of query's type on its device; got ",
              t.sizes(), " ", t.scalar_type());
}

bool is_index(const Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }

// A cache (pages, page_size, kv_heads, dim) with its scales.
sonar_kv_cache cache_of(const Tensor& cache, const OptTensor& scale, const Tensor& query, int64_t kv_heads, int64_t dim, const char* name,
                        const char* scale_name) {
  TORCH_CHECK(cache.dim() == 4 && cache.device() == query.device() && cache.size(2) == kv_heads && cache.size(3) == dim, name,
              " must be (pages, page_size, ", kv_heads, ", ", dim, ") on query's device; got ", cache.sizes());
  TORCH_CHECK(cache.size(3) <= 1 || cache.stride(3) == 1 || cache.numel() == 0, name, " must have the numbers of a head behind each other: its strides are ",
              cache.strides());
  TORCH_CHECK(cache.size(1) >= 1, name, " must have at least one slot a page");
  const bool fp8 = cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || cache.scalar_type() == query.scalar_type(), name, " must be of query's type or float8_e4m3fn; got ", cache.scalar_type());
  TORCH_CHECK(fp8 == scale.has_value(), scale_name, fp8 ? " is needed with a cache of float8_e4m3fn" : " goes with a cache of float8_e4m3fn");
  if (fp8)
    TORCH_CHECK(scale->device() == query.device() && scale->scalar_type() == at::kFloat && scale->is_contiguous() &&
                    (scale->numel() == 1 || scale->numel() == kv_heads), scale_name, " must hold 1 or ", kv_heads, " float32 numbers on query's device");
  // (a stride that nothing is multiplied by may be anything)
  const int64_t head = cache.size(2) > 1 ? cache.stride(2) : 0, slot = cache.size(1) > 1 ? cache.stride(1) : 0;
  return sonar_kv_cache{const_cast<void*>(cache.const_data_ptr()), cache.size(0) > 1 ? cache.stride(0) : 0, slot, head,
                        fp8 ? static_cast<const float*>(scale->const_data_ptr()) : nullptr, fp8 ? scale->numel() : 0};
}

int cache_code(const Tensor& cache, int dtype) { return cache.scalar_type() == at::kFloat8_e4m3fn ? SONAR_CACHE_FP8 : dtype; }

// ---------------------------------------------------------------- norms and rotation
struct Rope {
  Tensor table, positions, q_weight, k_weight;
  Rope(const Tensor& query, int64_t tokens, int64_t dim, const OptTensor& positions_, const OptTensor& table_, const OptTensor& q_weight_,
       const OptTensor& k_weight_) {
    TORCH_CHECK(positions_.has_value() == table_.has_value(), "positions and cos_sin_cache go together");
    if (table_.has_value()) {
      TORCH_CHECK(positions_->device() == query.device() && is_index(*positions_) && positions_->dim() == 1 && positions_->size(0) == tokens,
                  "positions must hold ", tokens, " int64 or int32 numbers on query's device");
      TORCH_CHECK(table_->device() == query.device() && table_->scalar_type() == at::kFloat && table_->dim() == 2 && table_->size(1) >= 2,
                  "cos_sin_cache must be float32 (positions, rotary_dim) on query's device; got ", table_->sizes(), " ", table_->scalar_type());
      table = table_->contiguous(), positions = positions_->contiguous();
    }
    for (const auto& [weight, to, name] : {std::make_tuple(&q_weight_, &q_weight, "q_weight"), std::make_tuple(&k_weight_, &k_weight, "k_weight")})
      if (weight->has_value()) {
        TORCH_CHECK((*weight)->device() == query.device() && (*weight)->scalar_type() == query.scalar_type() && (*weight)->dim() == 1 &&
                        (*weight)->size(0) == dim, name, " must hold ", dim, " numbers of query's type on its device");
        *to = (*weight)->contiguous();
      }
  }
  const void* data(const Tensor& t) const { return t.defined() ? t.const_data_ptr() : nullptr; }
};

int rotate(const Tensor& query, const Heads& q, const Heads& k, const Heads* v, const Rope& rope, double epsilon, bool is_neox, Tensor& q_out,
           Tensor* k_out, const sonar_kv_cache* keys, const sonar_kv_cache* values, const Tensor* cache, const Tensor* slots, int dtype) {
  const bool table = rope.table.defined();
  // (a table without rows has no address, and no position that would look at one)
  const void* rows = table && rope.table.size(0) == 0 ? rope.data(rope.positions) : rope.data(rope.table);
  return sonar_qk_norm_rope(
      q.t.const_data_ptr(), q.token_stride, q.head_stride, k.t.const_data_ptr(), k.token_stride, k.head_stride,
      v ? v->t.const_data_ptr() : nullptr, v ? v->token_stride : 0, v ? v->head_stride : 0, rope.data(rope.positions),
      table && rope.positions.scalar_type() == at::kLong, static_cast<const float*>(rows), table ? rope.table.size(0) : 0,
      table ? rope.table.size(1) : 0, is_neox ? 1 : 0, rope.data(rope.q_weight), rope.data(rope.k_weight), epsilon, q_out.mutable_data_ptr(),
      k_out ? k_out->mutable_data_ptr() : nullptr, keys, values, cache ? cache_code(*cache, dtype) : dtype, slots ? slots->const_data_ptr() : nullptr,
      slots && slots->scalar_type() == at::kLong, cache ? cache->size(0) : 0, cache ? cache->size(1) : 1, dtype, query.size(0), query.size(1),
      k.t.size(1), query.size(2), current_stream(query));
}

void check_query(const Tensor& query) {
  TORCH_CHECK(query.is_cuda(), "query is not on GPU");
  TORCH_CHECK(query.dim() == 3 && query.size(1) >= 1 && query.size(2) >= 1, "query must be (tokens, heads, head_dim); got ", query.sizes());
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& query, const Tensor& key, const OptTensor& positions, const OptTensor& cos_sin_cache,
                                        const OptTensor& q_weight, const OptTensor& k_weight, double epsilon, bool is_neox) {
  check_query(query);
  const int dtype = dtype_code(query, "query");
  check_heads(key, query, query.size(0), query.size(2), "key");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  const Rope rope(query, query.size(0), query.size(2), positions, cos_sin_cache, q_weight, k_weight);
  const Heads q(query, false), k(key, false);
  Tensor q_out = new_tensor(query, query.sizes(), query.scalar_type()), k_out = new_tensor(query, key.sizes(), query.scalar_type());
  raise_if_failed(rotate(query, q, k, nullptr, rope, epsilon, is_neox, q_out, &k_out, nullptr, nullptr, nullptr, nullptr, dtype));
  return {q_out, k_out};
}

Tensor qk_norm_rope_append(const Tensor& query, const Tensor& key, const Tensor& value, Tensor& key_cache, Tensor& value_cache,
                           const Tensor& slot_mapping, const OptTensor& positions, const OptTensor& cos_sin_cache, const OptTensor& q_weight,
                           const OptTensor& k_weight, double epsilon, bool is_neox, const OptTensor& k_scale, const OptTensor& v_scale) {
  check_query(query);
  const int dtype = dtype_code(query, "query");
  const int64_t tokens = query.size(0), dim = query.size(2);
  check_heads(key, query, tokens, dim, "key");
  check_heads(value, query, tokens, dim, "value");
  const int64_t kv_heads = key.size(1);
  TORCH_CHECK(value.size(1) == kv_heads, "value must have key's ", kv_heads, " heads; got ", value.sizes());
  const sonar_kv_cache keys = cache_of(key_cache, k_scale, query, kv_heads, dim, "key_cache", "k_scale");
  const sonar_kv_cache values = cache_of(value_cache, v_scale, query, kv_heads, dim, "value_cache", "v_scale");
  TORCH_CHECK(key_cache.sizes() == value_cache.sizes() && key_cache.scalar_type() == value_cache.scalar_type(),
              "key_cache and value_cache must have one shape and type");
  at::assert_no_internal_overlap(key_cache);
  at::assert_no_internal_overlap(value_cache);
  at::assert_no_overlap(key_cache, value_cache);
  TORCH_CHECK(slot_mapping.device() == query.device() && is_index(slot_mapping) && slot_mapping.dim() == 1 && slot_mapping.size(0) == tokens,
              "slot_mapping must hold ", tokens, " int64 or int32 numbers on query's device");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  const Rope rope(query, tokens, dim, positions, cos_sin_cache, q_weight, k_weight);
  const Heads q(query, false), k(key, false), v(value, false);
  const Tensor slots = slot_mapping.contiguous();
  Tensor q_out = new_tensor(query, query.sizes(), query.scalar_type());
  // a cache without pages takes nothing: the address is then one that no slot reaches
  sonar_kv_cache to_keys = keys, to_values = values;
  if (key_cache.numel() == 0) to_keys.data = to_values.data = q_out.mutable_data_ptr();
  raise_if_failed(rotate(query, q, k, &v, rope, epsilon, is_neox, q_out, nullptr, &to_keys, &to_values, &key_cache, &slots, dtype));
  return q_out;
}

// ---------------------------------------------------------------- attention
void attend(const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_table, const Tensor& seq_lens,
            const Tensor& query_start_loc, double scale, bool causal, int64_t window, double softcap, const OptTensor& alibi_slopes,
            const OptTensor& tree_mask, const OptTensor& k_scale, const OptTensor& v_scale, std::optional<int64_t> max_seq_len, Tensor& out,
            bool clear_rest) {
  const int dtype = dtype_code(query, "query");
  TORCH_CHECK(dtype != SONAR_DTYPE_F32, "query must be float16 or bfloat16");
  const int64_t tokens = query.size(0), heads = query.size(1), dim = query.size(2), seqs = seq_lens.numel();
  TORCH_CHECK(key_cache.dim() == 4, "key_cache must be (pages, page_size, kv_heads, head_dim); got ", key_cache.sizes());
  const int64_t kv_heads = key_cache.size(2), page_size = key_cache.size(1);
  TORCH_CHECK(kv_heads >= 1 && heads % kv_heads == 0, "query's ", heads, " heads are no multiple of the cache's ", kv_heads);
  const sonar_kv_cache keys = cache_of(key_cache, k_scale, query, kv_heads, dim, "key_cache", "k_scale");
  const sonar_kv_cache values = cache_of(value_cache, v_scale, query, kv_heads, dim, "value_cache", "v_scale");
  TORCH_CHECK(key_cache.sizes() == value_cache.sizes() && key_cache.scalar_type() == value_cache.scalar_type(),
              "key_cache and value_cache must have one shape and type");
  for (const auto& [t, count, name] : {std::make_tuple(&seq_lens, seqs, "seq_lens"), std::make_tuple(&query_start_loc, seqs + 1, "query_start_loc")})
    TORCH_CHECK(t->device() == query.device() && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == count, name, " must hold ", count,
                " int32 numbers on query's device");
  TORCH_CHECK(block_table.device() == query.device() && block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                  block_table.size(0) == seqs, "block_table must be int32 (", seqs, ", pages) on query's device; got ", block_table.sizes());
  if (alibi_slopes.has_value())
    TORCH_CHECK(alibi_slopes->device() == query.device() && alibi_slopes->scalar_type() == at::kFloat && alibi_slopes->numel() == heads,
                "alibi_slopes must hold ", heads, " float32 numbers on query's device");
  if (tree_mask.has_value())
    TORCH_CHECK(tree_mask->device() == query.device() && tree_mask->scalar_type() == at::kLong && tree_mask->dim() == 2 &&
                    tree_mask->size(0) == tokens && tree_mask->size(1) >= 1, "tree_mask must be int64 (", tokens, ", words) on query's device; got ",
                tree_mask->sizes());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
  const Heads q(query, true);
  const Tensor lens = seq_lens.contiguous(), starts = query_start_loc.contiguous();
  const bool rows = (block_table.size(1) <= 1 || block_table.stride(1) == 1) && (seqs <= 1 || block_table.stride(0) >= block_table.size(1));
  const Tensor table = rows ? block_table : block_table.clone(at::MemoryFormat::Contiguous);
  const Tensor slopes = alibi_slopes.has_value() ? alibi_slopes->contiguous() : Tensor();
  const Tensor tree = tree_mask.has_value() ? tree_mask->contiguous() : Tensor();
  const int64_t table_pages = table.size(1), table_stride = seqs > 1 ? table.stride(0) : table_pages;
  const int64_t longest = max_seq_len.has_value() ? *max_seq_len : table_pages * page_size;
  const size_t scratch_bytes = sonar_paged_attention_scratch_bytes(tokens, seqs, heads, kv_heads, dim, cache_code(key_cache, dtype), longest, window);
  Tensor scratch;
  if (scratch_bytes > 0) scratch = new_tensor(query, {(int64_t)scratch_bytes}, at::kByte);
  raise_if_failed(sonar_paged_attention(
      q.t.const_data_ptr(), q.token_stride, q.head_stride, &keys, &values, cache_code(key_cache, dtype), key_cache.size(0), page_size,
      static_cast<const int32_t*>(table.const_data_ptr()), table_stride, key_cache.size(0) > 0 ? table_pages : 0,
      static_cast<const int32_t*>(lens.const_data_ptr()), static_cast<const int32_t*>(starts.const_data_ptr()), out.mutable_data_ptr(),
      tokens > 1 ? out.stride(0) : heads * dim, heads > 1 ? out.stride(1) : dim, clear_rest ? 1 : 0, scale, softcap, window, causal ? 1 : 0,
      slopes.defined() ? static_cast<const float*>(slopes.const_data_ptr()) : nullptr,
      tree.defined() ? static_cast<const int64_t*>(tree.const_data_ptr()) : nullptr, tree.defined() ? tree.size(1) : 0,
      scratch_bytes > 0 ? scratch.mutable_data_ptr() : nullptr, scratch_bytes, dtype, tokens, seqs, heads, kv_heads, dim, longest,
      current_stream(query)));
}

Tensor paged_attention(const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_table, const Tensor& seq_lens,
                       const Tensor& query_start_loc, double scale, bool causal, int64_t window, double softcap, const OptTensor& alibi_slopes,
                       const OptTensor& tree_mask, const OptTensor& k_scale, const OptTensor& v_scale, std::optional<int64_t> max_seq_len) {
  check_query(query);
  Tensor out = new_tensor(query, query.sizes(), query.scalar_type());
  attend(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap, alibi_slopes, tree_mask, k_scale,
         v_scale, max_seq_len, out, true);
  return out;
}

void paged_attention_out(const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_table,
                         const Tensor& seq_lens, const Tensor& query_start_loc, double scale, bool causal, int64_t window, double softcap,
                         const OptTensor& alibi_slopes, const OptTensor& tree_mask, const OptTensor& k_scale, const OptTensor& v_scale,
                         std::optional<int64_t> max_seq_len, Tensor& out) {
  check_query(query);
  TORCH_CHECK(out.device() == query.device() && out.scalar_type() == query.scalar_type() && out.sizes() == query.sizes() &&
                  (out.size(2) <= 1 || out.stride(2) == 1), "out must have query's shape, type and device, the numbers of a head behind each other");
  at::assert_no_internal_overlap(out);
  for (const Tensor* t : {&query, &key_cache, &value_cache}) at::assert_no_overlap(out, *t);
  attend(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap, alibi_slopes, tree_mask, k_scale,
         v_scale, max_seq_len, out, false);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sonar_amd, m) {
  m.def(
      "qk_norm_rope(Tensor query, Tensor key, Tensor? positions, Tensor? cos_sin_cache, Tensor? q_weight, Tensor? k_weight, "
      "float epsilon, bool is_neox) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rope_append(Tensor query, Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slot_mapping, "
      "Tensor? positions, Tensor? cos_sin_cache, Tensor? q_weight, Tensor? k_weight, float epsilon, bool is_neox, Tensor? k_scale, "
      "Tensor? v_scale) -> Tensor");
  m.def(
      "paged_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, Tensor query_start_loc, "
      "float scale, bool causal, int window, float softcap, Tensor? alibi_slopes, Tensor? tree_mask, Tensor? k_scale, Tensor? v_scale, "
      "int? max_seq_len) -> Tensor");
  m.def(
      "paged_attention_out(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, Tensor query_start_loc, "
      "float scale, bool causal, int window, float softcap, Tensor? alibi_slopes, Tensor? tree_mask, Tensor? k_scale, Tensor? v_scale, "
      "int? max_seq_len, Tensor(a!) out) -> ()");
}
TORCH_LIBRARY_IMPL(sonar_amd, CUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_append", &qk_norm_rope_append);
  m.impl("paged_attention", &paged_attention);
  m.impl("paged_attention_out", &paged_attention_out);
}
