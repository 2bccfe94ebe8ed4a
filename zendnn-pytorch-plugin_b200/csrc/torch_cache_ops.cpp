// PyTorch boundary of the operators between a decoder layer's linears: rotary positions, the paged key/value cache and the
// attention that reads it.  The reference leaves them to its host framework, so the schemas are this library's own.  Like the
// linears' boundary (torch_ops.cpp) this only checks and marshals tensors into the C ABI on the current stream.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/record_function.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/util/SmallVector.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "torch_util.h"

namespace zentorch_b200 {

namespace {

int cache_code(c10::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return ZT_BF16;
    case at::kHalf: return ZT_F16;
    case at::kFloat: return ZT_F32;
    case at::kFloat8_e4m3fn: return ZT_E4M3;
    default: return -1;
  }
}

void check_index(const at::Tensor &t, const at::Tensor &input, const char *op, const char *name, int64_t numel) {
  check_on_device(t, input, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, op, ": ", name, " must be int32 or int64, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 1 && t.size(0) == numel, op, ": ", name, " must have shape [", numel, "], got ", t.sizes());
}
void check_lengths(const at::Tensor &t, const at::Tensor &input, const char *op, const char *name, int64_t dim) {
  check_on_device(t, input, op, name);
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must be ", dim, "D, got ", t.dim(), "D");
}

// Nothing is written twice, or while the same call still reads it.
void check_written(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK(at::has_internal_overlap(t) != at::MemOverlap::Yes, op, ": ", name, " is written and must not hold an element twice");
}
// The bytes of a tensor are its address plus sums of i * stride, 0 <= i < size.  Two tensors share one where their addresses differ by
// such a sum over the strides of both, i down to 1 - size for the other's: `from` is what the dimensions from `d` on, the widest
// first, have to add up to.  Strides of views are nested, which leaves one or two i each; `steps` bounds the search where they
// are not (nothing is found then).
struct Reach {
  int64_t stride, lo, hi;           // i from lo to hi
  int64_t rest_lo, rest_hi;         // what the dimensions behind this one add up to
};
using Reaches = c10::SmallVector<Reach, 12>;
bool adds_up(const Reaches &dims, size_t d, int64_t from, int &steps) {
  if (d == dims.size()) return from == 0;
  const Reach &r = dims[d];
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t lo = std::max(r.lo, -floor_div(r.rest_hi - from, r.stride)), hi = std::min(r.hi, floor_div(from - r.rest_lo, r.stride));
  for (int64_t i = lo; i <= hi && --steps >= 0; ++i)
    if (adds_up(dims, d + 1, from - i * r.stride, steps)) return true;
  return false;
}
int64_t bytes_spanned(const at::Tensor &t) {
  const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
  int64_t last = 0;
  for (size_t i = 0; i < sizes.size(); ++i) last += (sizes[i] - 1) * strides[i];
  return (last + 1) * (int64_t)t.element_size();
}
bool share_memory(const at::Tensor &a, const at::Tensor &b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(b.data_ptr()) - reinterpret_cast<uintptr_t>(a.data_ptr()));
  if (apart >= bytes_spanned(a) || -apart >= bytes_spanned(b)) return false;
  Reaches dims;                     // one per stride, the widest first
  auto dim = [&](int64_t stride, int64_t lo, int64_t hi) {
    if (stride == 0 || lo == hi) return;
    auto *at = std::find_if(dims.begin(), dims.end(), [&](const Reach &r) { return r.stride <= stride; });
    if (at != dims.end() && at->stride == stride) at->lo += lo, at->hi += hi;
    else dims.insert(at, Reach{stride, lo, hi, 0, 0});
  };
  for (const at::Tensor *t : {&a, &b}) {
    const at::IntArrayRef sizes = t->sizes(), strides = t->strides();
    const int64_t es = (int64_t)t->element_size(), sign = t == &a ? 1 : -1;
    dim(1, std::min<int64_t>(sign * (es - 1), 0), std::max<int64_t>(sign * (es - 1), 0));
    for (size_t i = 0; i < sizes.size(); ++i) {
      const int64_t far = sign * (sizes[i] - 1);
      dim(strides[i] * es, std::min<int64_t>(far, 0), std::max<int64_t>(far, 0));
    }
  }
  for (size_t d = dims.size(); d-- > 1;) {
    dims[d - 1].rest_lo = dims[d].rest_lo + dims[d].lo * dims[d].stride;
    dims[d - 1].rest_hi = dims[d].rest_hi + dims[d].hi * dims[d].stride;
  }
  int steps = 1000;
  return adds_up(dims, 0, apart, steps);
}
void check_apart(const at::Tensor &t, const at::Tensor &other, const char *op, const char *name, const char *other_name) {
  TORCH_CHECK(!share_memory(t, other), op, ": ", name, " is written and must not share memory with ", other_name);
}

// A pair of caches [pages, page_size, heads, head_dim] of one shape and type; for `input` of `head_dim`.
void check_caches(const at::Tensor &k, const at::Tensor &v, const at::Tensor &input, int64_t head_dim, const char *op) {
  check_on_device(k, input, op, "key_cache");
  check_on_device(v, input, op, "value_cache");
  TORCH_CHECK(k.dim() == 4, op, ": key_cache must be [pages, page_size, kv_heads, head_dim], got ", k.dim(), "D");
  TORCH_CHECK(v.sizes() == k.sizes(), op, ": value_cache must have the shape of key_cache ", k.sizes(), ", got ", v.sizes());
  TORCH_CHECK(k.scalar_type() == input.scalar_type() || k.scalar_type() == at::kFloat8_e4m3fn, op,
              ": the caches must be ", input.scalar_type(), " (as the input) or float8_e4m3fn, got ", k.scalar_type());
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), op, ": key_cache and value_cache must have one dtype");
  TORCH_CHECK(k.size(3) == head_dim, op, ": the caches have heads of ", k.size(3), " elements, the input of ", head_dim);
  TORCH_CHECK(k.size(1) >= 1, op, ": the page size must be positive");
  TORCH_CHECK(k.size(1) < (int64_t)1 << 31 && k.size(0) < (int64_t)1 << 31, op, ": pages of the cache out of range");
  TORCH_CHECK((k.size(3) == 1 || (k.stride(3) == 1 && v.stride(3) == 1)), op, ": the caches need unit stride along head_dim");
}
const float *cache_scale(const std::optional<at::Tensor> &t, const at::Tensor &cache, const at::Tensor &input, const char *op,
                         const char *name) {
  if (cache.scalar_type() != at::kFloat8_e4m3fn) {
    TORCH_CHECK(!t.has_value() || !t->defined(), op, ": ", name, " belongs to a float8_e4m3fn cache");
    return nullptr;
  }
  TORCH_CHECK(t.has_value() && t->defined(), op, ": a float8_e4m3fn cache needs ", name);
  check_on_device(*t, input, op, name);
  TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == cache.size(2) && t->is_contiguous(), op, ": ", name,
              " must be a contiguous float32 tensor with one value per kv head (", cache.size(2), ")");
  return t->data_ptr<float>();
}

// ---- rotary positions -------------------------------------------------------------------------------------
at::Tensor unit_inner(const at::Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }

void rope_fill(zt_rope_args_t &a, const at::Tensor &q, const at::Tensor &k, const at::Tensor &positions, const at::Tensor &inv_freq,
               bool interleaved, double factor, const char *op) {
  TORCH_CHECK(q.is_cuda(), op, " (CUDA): query must be a CUDA tensor");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3, op, ": query and key must be [tokens, heads, head_dim]");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat, op,
              ": query must be bfloat16, float16 or float32, got ", q.scalar_type());
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), op, ": key must have the dtype of the query");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2), op, ": query ", q.sizes(), " and key ", k.sizes(),
              " must agree in tokens and head_dim");
  check_on_device(k, q, op, "key");
  check_index(positions, q, op, "positions", q.size(0));
  check_on_device(inv_freq, q, op, "inv_freq");
  TORCH_CHECK(inv_freq.scalar_type() == at::kFloat && inv_freq.dim() == 1, op, ": inv_freq must be a 1D float32 tensor");
  TORCH_CHECK(2 * inv_freq.size(0) <= q.size(2), op, ": inv_freq rotates ", 2 * inv_freq.size(0), " elements of heads of ", q.size(2));
  a.q = q.data_ptr(), a.k = k.data_ptr();
  a.tokens = q.size(0);
  a.q_heads = (int32_t)q.size(1), a.kv_heads = (int32_t)k.size(1), a.head_dim = (int32_t)q.size(2);
  a.rot_dim = (int32_t)(2 * inv_freq.size(0));
  a.dtype = cache_code(q.scalar_type());
  for (int i = 0; i < 2; ++i) a.q_stride[i] = q.stride(i), a.k_stride[i] = k.stride(i);
  a.positions = positions.data_ptr(), a.positions_64 = positions.scalar_type() == at::kLong;
  a.inv_freq = inv_freq.data_ptr<float>();
  a.attention_factor = (float)factor;
  a.interleaved = interleaved;
}

std::tuple<at::Tensor, at::Tensor> rope(const at::Tensor &query, const at::Tensor &key, const at::Tensor &positions,
                                        const at::Tensor &inv_freq, bool interleaved, double attention_factor,
                                        std::string zentorch_op_name) {
  RECORD_FUNCTION(zentorch_op_name, std::vector<c10::IValue>({query, key}));
  const char *op = "zentorch_rope";
  zt_rope_args_t a{};
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3, op, ": query and key must be [tokens, heads, head_dim]");
  const at::Tensor q = unit_inner(query), k = unit_inner(key), pos = positions.contiguous(), freq = inv_freq.contiguous();
  rope_fill(a, q, k, pos, freq, interleaved, attention_factor, op);
  c10::cuda::CUDAGuard device_guard(q.device());
  at::Tensor q_out = at::empty(q.sizes(), q.options()), k_out = at::empty(k.sizes(), k.options());
  a.q_out = q_out.data_ptr(), a.k_out = k_out.data_ptr();
  for (int i = 0; i < 2; ++i) a.q_out_stride[i] = q_out.stride(i), a.k_out_stride[i] = k_out.stride(i);
  ZT_TORCH_CALL(zt_rope(&a, at::cuda::getCurrentCUDAStream()));
  return {q_out, k_out};
}

at::Tensor rope_cache(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const at::Tensor &positions,
                      const at::Tensor &inv_freq, at::Tensor &key_cache, at::Tensor &value_cache, const at::Tensor &slot_mapping,
                      const std::optional<at::Tensor> &k_scale, const std::optional<at::Tensor> &v_scale, bool interleaved,
                      double attention_factor, std::string zentorch_op_name) {
  RECORD_FUNCTION(zentorch_op_name, std::vector<c10::IValue>({query, key}));
  const char *op = "zentorch_rope_cache";
  zt_rope_args_t a{};
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3, op, ": query and key must be [tokens, heads, head_dim]");
  TORCH_CHECK(value.sizes() == key.sizes() && value.scalar_type() == key.scalar_type(), op,
              ": value must have the shape and dtype of the key");
  const at::Tensor q = unit_inner(query), k = unit_inner(key), v = unit_inner(value), pos = positions.contiguous(),
                   freq = inv_freq.contiguous(), slots = slot_mapping.contiguous();
  rope_fill(a, q, k, pos, freq, interleaved, attention_factor, op);
  check_on_device(v, q, op, "value");
  check_index(slots, q, op, "slot_mapping", q.size(0));
  check_caches(key_cache, value_cache, q, q.size(2), op);
  TORCH_CHECK(key_cache.size(2) == k.size(1), op, ": the caches have ", key_cache.size(2), " heads, the key ", k.size(1));
  check_written(key_cache, op, "key_cache"), check_written(value_cache, op, "value_cache");
  if (key_cache.data_ptr() != value_cache.data_ptr() || key_cache.strides() != value_cache.strides())      // (one tensor as both holds the values)
    check_apart(key_cache, value_cache, op, "key_cache", "value_cache");
  for (const auto &[name, cache] : {std::pair<const char *, const at::Tensor &>("key_cache", key_cache), {"value_cache", value_cache}}) {
    check_apart(cache, query, op, name, "query"), check_apart(cache, key, op, name, "key"), check_apart(cache, value, op, name, "value");
  }
  a.k_scale = cache_scale(k_scale, key_cache, q, op, "k_scale");
  a.v_scale = cache_scale(v_scale, value_cache, q, op, "v_scale");
  c10::cuda::CUDAGuard device_guard(q.device());
  at::Tensor q_out = at::empty(q.sizes(), q.options());
  a.v = v.data_ptr();
  a.q_out = q_out.data_ptr();
  for (int i = 0; i < 2; ++i) a.q_out_stride[i] = q_out.stride(i), a.v_stride[i] = v.stride(i);
  a.k_cache = key_cache.data_ptr(), a.v_cache = value_cache.data_ptr(), a.cache_dtype = cache_code(key_cache.scalar_type());
  for (int i = 0; i < 3; ++i) a.k_cache_stride[i] = key_cache.stride(i), a.v_cache_stride[i] = value_cache.stride(i);
  a.num_pages = key_cache.size(0), a.page_size = (int32_t)key_cache.size(1);
  a.slots = slots.data_ptr(), a.slots_64 = slots.scalar_type() == at::kLong;
  if (key_cache.numel() == 0) {   // no pages: every slot is past the cache; nothing can be stored
    TORCH_CHECK(q.size(0) == 0 || key_cache.size(0) > 0, op, ": the cache has no pages");
  }
  if (q.size(0) > 0) ZT_TORCH_CALL(zt_rope(&a, at::cuda::getCurrentCUDAStream()));
  return q_out;
}

// ---- pages ------------------------------------------------------------------------------------------------
// Whether the dimensions behind the first are one block without holes, in any order.
bool dense_pages(const at::Tensor &t) {
  c10::SmallVector<std::pair<int64_t, int64_t>, 8> dims;   // stride, size
  for (int64_t i = 1; i < t.dim(); ++i)
    if (t.size(i) != 1) dims.emplace_back(t.stride(i), t.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t expect = 1;
  for (auto &d : dims) {
    if (d.first != expect) return false;
    expect *= d.second;
  }
  return t.size(0) <= 1 || t.stride(0) >= expect;
}

void cache_copy_pages(at::TensorList caches, const at::Tensor &src, const at::Tensor &dst, std::string zentorch_op_name) {
  const char *op = "zentorch_cache_copy_pages";
  RECORD_FUNCTION(zentorch_op_name, std::vector<c10::IValue>({src, dst}));
  TORCH_CHECK(src.is_cuda(), op, " (CUDA): src must be a CUDA tensor");
  TORCH_CHECK(src.dim() == 1, op, ": src must be 1D");
  check_index(src, src, op, "src", src.size(0));
  check_index(dst, src, op, "dst", src.size(0));
  TORCH_CHECK(src.scalar_type() == dst.scalar_type(), op, ": src and dst must have one dtype");
  if (caches.empty()) return;
  c10::SmallVector<void *, 64> base;
  c10::SmallVector<int64_t, 64> stride, bytes;
  const at::Tensor &model = caches[0];      // the layers' caches are mostly alike
  for (const at::Tensor &t : caches) {
    check_on_device(t, src, op, "every cache");
    TORCH_CHECK(t.dim() >= 2, op, ": a cache must be [pages, ...], got ", t.dim(), "D");
    TORCH_CHECK(t.size(0) == model.size(0), op, ": the caches must have one number of pages");
    TORCH_CHECK(t.size(0) < (int64_t)1 << 31, op, ": pages of the cache out of range");
    if (t.numel() == 0) continue;
    const bool alike = !base.empty() && model.numel() > 0 && t.sizes() == model.sizes() && t.strides() == model.strides();
    TORCH_CHECK(alike || dense_pages(t), op, ": a page of a cache must be one block of memory; got strides ", t.strides(), " for ", t.sizes());
    const int64_t es = (int64_t)t.element_size();
    base.push_back(t.data_ptr());
    bytes.push_back(t.numel() / t.size(0) * es);
    stride.push_back(t.size(0) <= 1 ? bytes.back() : t.stride(0) * es);
  }
  if (base.empty() || src.size(0) == 0) return;
  c10::cuda::CUDAGuard device_guard(src.device());
  const at::Tensor s = src.contiguous(), d = dst.contiguous();
  zt_cache_copy_args_t a{};
  a.n_caches = (int32_t)base.size();
  a.caches = base.data(), a.page_stride_bytes = stride.data(), a.page_bytes = bytes.data();
  a.num_pages = (int32_t)model.size(0);
  a.n_pairs = s.size(0);
  a.src = s.data_ptr(), a.dst = d.data_ptr(), a.index_64 = s.scalar_type() == at::kLong;
  ZT_TORCH_CALL(zt_cache_copy_pages(&a, at::cuda::getCurrentCUDAStream()));
}

// ---- attention --------------------------------------------------------------------------------------------
void paged_attention_into(at::Tensor &out, const at::Tensor &query, const at::Tensor &key_cache, const at::Tensor &value_cache,
                          const at::Tensor &cu_seqlens_q, const at::Tensor &seq_lens, const at::Tensor &block_table,
                          std::optional<int64_t> max_query_len, std::optional<double> scale, bool causal, int64_t window,
                          const std::optional<at::Tensor> &k_scale, const std::optional<at::Tensor> &v_scale, bool zero_tail,
                          const std::string &op_name) {
  const char *op = "zentorch_paged_attention";
  RECORD_FUNCTION(op_name, std::vector<c10::IValue>({query, key_cache}));
  TORCH_CHECK(query.is_cuda(), op, " (CUDA): query must be a CUDA tensor");
  TORCH_CHECK(query.dim() == 3, op, ": query must be [tokens, q_heads, head_dim], got ", query.dim(), "D");
  TORCH_CHECK(query.scalar_type() == at::kBFloat16 || query.scalar_type() == at::kHalf, op,
              ": query must be bfloat16 or float16, got ", query.scalar_type());
  const int64_t T = query.size(0), hq = query.size(1), D = query.size(2);
  check_caches(key_cache, value_cache, query, D, op);
  TORCH_CHECK(key_cache.size(2) >= 1 && hq >= 1 && hq % key_cache.size(2) == 0, op, ": the query heads (", hq,
              ") must be a multiple of the caches' heads (", key_cache.size(2), ")");
  check_lengths(cu_seqlens_q, query, op, "cu_seqlens_q", 1);
  check_lengths(seq_lens, query, op, "seq_lens", 1);
  check_lengths(block_table, query, op, "block_table", 2);
  const int64_t B = seq_lens.size(0);
  TORCH_CHECK(cu_seqlens_q.size(0) == B + 1, op, ": cu_seqlens_q must have one entry more than seq_lens (", B, "), got ",
              cu_seqlens_q.size(0));
  TORCH_CHECK(block_table.size(0) == B, op, ": block_table must have a row per sequence (", B, "), got ", block_table.size(0));
  TORCH_CHECK(block_table.size(1) < (int64_t)1 << 31 && T < (int64_t)1 << 31 && B < (int64_t)1 << 31, op, ": sizes out of range");
  TORCH_CHECK(!max_query_len.has_value() || (*max_query_len >= 0 && *max_query_len < (int64_t)1 << 31), op,
              ": max_query_len must not be negative");
  TORCH_CHECK(window >= 0 && window < (int64_t)1 << 31, op, ": window must not be negative (0: none), got ", window);
  TORCH_CHECK(!scale.has_value() || (std::isfinite(*scale) && *scale > 0), op, ": scale must be positive and finite");
  check_on_device(out, query, op, "out");
  TORCH_CHECK(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type(), op,
              ": out must have the shape and dtype of the query");
  if (!zero_tail) {      // (else it was made for this call)
    check_written(out, op, "out");
    check_apart(out, query, op, "out", "query"), check_apart(out, key_cache, op, "out", "key_cache"), check_apart(out, value_cache, op, "out", "value_cache");
  }
  zt_paged_attention_args_t a{};
  a.k_scale = cache_scale(k_scale, key_cache, query, op, "k_scale");
  a.v_scale = cache_scale(v_scale, value_cache, query, op, "v_scale");
  if (T == 0) return;
  c10::cuda::CUDAGuard device_guard(query.device());
  auto wide_rows = [](const at::Tensor &t) {   // unit inner stride, rows on 16-byte boundaries
    return t.stride(2) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) | (uintptr_t)(t.stride(0) * 2) | (uintptr_t)(t.stride(1) * 2)) % 16 == 0;
  };
  const at::Tensor q = wide_rows(query) ? query : query.clone(at::MemoryFormat::Contiguous);
  const bool direct = wide_rows(out);
  at::Tensor y = direct ? out : (zero_tail ? at::empty(out.sizes(), out.options()) : out.clone(at::MemoryFormat::Contiguous));
  const at::Tensor cu = cu_seqlens_q.contiguous(), lens = seq_lens.contiguous();
  const at::Tensor table = block_table.size(1) <= 1 || block_table.stride(1) == 1 ? block_table : block_table.contiguous();
  a.q = q.data_ptr(), a.out = y.data_ptr();
  a.tokens = T, a.batch = (int32_t)B, a.q_heads = (int32_t)hq, a.kv_heads = (int32_t)key_cache.size(2), a.head_dim = (int32_t)D;
  a.dtype = cache_code(query.scalar_type()), a.cache_dtype = cache_code(key_cache.scalar_type());
  for (int i = 0; i < 2; ++i) a.q_stride[i] = q.stride(i), a.out_stride[i] = y.stride(i);
  a.k_cache = key_cache.data_ptr(), a.v_cache = value_cache.data_ptr();
  for (int i = 0; i < 3; ++i) a.k_cache_stride[i] = key_cache.stride(i), a.v_cache_stride[i] = value_cache.stride(i);
  a.num_pages = key_cache.size(0), a.page_size = (int32_t)key_cache.size(1);
  a.cu_seqlens_q = cu.data_ptr<int32_t>(), a.seq_lens = lens.data_ptr<int32_t>(), a.block_table = table.data_ptr<int32_t>();
  a.block_table_stride = table.stride(0), a.max_blocks = (int32_t)table.size(1);
  a.max_query_len = (int32_t)max_query_len.value_or(0);
  a.scale = (float)scale.value_or(1.0 / std::sqrt((double)D));
  a.causal = causal, a.window = (int32_t)window, a.zero_tail = zero_tail;
  const size_t bytes = zt_paged_attention_workspace_bytes(&a);
  at::Tensor ws;
  if (bytes > 0) {
    ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    a.workspace = ws.data_ptr(), a.workspace_bytes = bytes;
  }
  ZT_TORCH_CALL(zt_paged_attention(&a, at::cuda::getCurrentCUDAStream()));
  if (!direct) out.copy_(y);
}

at::Tensor paged_attention(const at::Tensor &query, const at::Tensor &key_cache, const at::Tensor &value_cache,
                           const at::Tensor &cu_seqlens_q, const at::Tensor &seq_lens, const at::Tensor &block_table,
                           std::optional<int64_t> max_query_len, std::optional<double> scale, bool causal, int64_t window,
                           const std::optional<at::Tensor> &k_scale, const std::optional<at::Tensor> &v_scale,
                           std::string zentorch_op_name) {
  at::Tensor out = at::empty(query.sizes(), query.options());
  paged_attention_into(out, query, key_cache, value_cache, cu_seqlens_q, seq_lens, block_table, max_query_len, scale, causal, window,
                       k_scale, v_scale, true, zentorch_op_name);
  return out;
}

void paged_attention_out(at::Tensor &out, const at::Tensor &query, const at::Tensor &key_cache, const at::Tensor &value_cache,
                         const at::Tensor &cu_seqlens_q, const at::Tensor &seq_lens, const at::Tensor &block_table,
                         std::optional<int64_t> max_query_len, std::optional<double> scale, bool causal, int64_t window,
                         const std::optional<at::Tensor> &k_scale, const std::optional<at::Tensor> &v_scale,
                         std::string zentorch_op_name) {
  paged_attention_into(out, query, key_cache, value_cache, cu_seqlens_q, seq_lens, block_table, max_query_len, scale, causal, window,
                       k_scale, v_scale, false, zentorch_op_name);
}

// ---- meta kernels -----------------------------------------------------------------------------------------
std::tuple<at::Tensor, at::Tensor> meta_rope(const at::Tensor &query, const at::Tensor &key, const at::Tensor &, const at::Tensor &,
                                             bool, double, std::string) {
  return {at::empty_symint(query.sym_sizes(), query.options()), at::empty_symint(key.sym_sizes(), key.options())};
}
at::Tensor meta_rope_cache(const at::Tensor &query, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                           at::Tensor &, at::Tensor &, const at::Tensor &, const std::optional<at::Tensor> &,
                           const std::optional<at::Tensor> &, bool, double, std::string) {
  return at::empty_symint(query.sym_sizes(), query.options());
}
void meta_cache_copy_pages(at::TensorList, const at::Tensor &, const at::Tensor &, std::string) {}
at::Tensor meta_paged_attention(const at::Tensor &query, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                const at::Tensor &, std::optional<int64_t>, std::optional<double>, bool, int64_t,
                                const std::optional<at::Tensor> &, const std::optional<at::Tensor> &, std::string) {
  return at::empty_symint(query.sym_sizes(), query.options());
}
void meta_paged_attention_out(at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                              const at::Tensor &, const at::Tensor &, std::optional<int64_t>, std::optional<double>, bool, int64_t,
                              const std::optional<at::Tensor> &, const std::optional<at::Tensor> &, std::string) {}

struct Registrar {
  std::vector<std::unique_ptr<torch::Library>> libs;
  Registrar() {
    auto frag = std::make_unique<torch::Library>(torch::Library::FRAGMENT, "zentorch", std::nullopt, __FILE__, __LINE__);
    frag->def(
        "zentorch_rope(Tensor query, Tensor key, Tensor positions, Tensor inv_freq, *, bool interleaved=False, "
        "float attention_factor=1.0, str zentorch_op_name='zentorch::zentorch_rope') -> (Tensor, Tensor)");
    frag->def(
        "zentorch_rope_cache(Tensor query, Tensor key, Tensor value, Tensor positions, Tensor inv_freq, Tensor(a!) key_cache, "
        "Tensor(b!) value_cache, Tensor slot_mapping, Tensor? k_scale=None, Tensor? v_scale=None, *, bool interleaved=False, "
        "float attention_factor=1.0, str zentorch_op_name='zentorch::zentorch_rope_cache') -> Tensor");
    frag->def(
        "zentorch_cache_copy_pages(Tensor(a!)[] caches, Tensor src, Tensor dst, *, "
        "str zentorch_op_name='zentorch::zentorch_cache_copy_pages') -> ()");
#define ZT_ATTENTION_ARGS                                                                                             \
  "Tensor query, Tensor key_cache, Tensor value_cache, Tensor cu_seqlens_q, Tensor seq_lens, Tensor block_table, "    \
  "int? max_query_len=None, *, float? scale=None, bool causal=True, int window=0, Tensor? k_scale=None, "             \
  "Tensor? v_scale=None, "
    frag->def("zentorch_paged_attention(" ZT_ATTENTION_ARGS
              "str zentorch_op_name='zentorch::zentorch_paged_attention') -> Tensor");
    frag->def("zentorch_paged_attention.out(Tensor(a!) out, " ZT_ATTENTION_ARGS
              "str zentorch_op_name='zentorch::zentorch_paged_attention.out') -> ()");
#undef ZT_ATTENTION_ARGS
    libs.push_back(std::move(frag));
    auto cuda = std::make_unique<torch::Library>(torch::Library::IMPL, "zentorch", c10::DispatchKey::CUDA, __FILE__, __LINE__);
    cuda->impl("zentorch_rope", rope);
    cuda->impl("zentorch_rope_cache", rope_cache);
    cuda->impl("zentorch_cache_copy_pages", cache_copy_pages);
    cuda->impl("zentorch_paged_attention", paged_attention);
    cuda->impl("zentorch_paged_attention.out", paged_attention_out);
    libs.push_back(std::move(cuda));
    auto meta = std::make_unique<torch::Library>(torch::Library::IMPL, "zentorch", c10::DispatchKey::Meta, __FILE__, __LINE__);
    meta->impl("zentorch_rope", meta_rope);
    meta->impl("zentorch_rope_cache", meta_rope_cache);
    meta->impl("zentorch_cache_copy_pages", meta_cache_copy_pages);
    meta->impl("zentorch_paged_attention", meta_paged_attention);
    meta->impl("zentorch_paged_attention.out", meta_paged_attention_out);
    libs.push_back(std::move(meta));
  }
};

Registrar g_cache_registrar;

}  // namespace

}  // namespace zentorch_b200
