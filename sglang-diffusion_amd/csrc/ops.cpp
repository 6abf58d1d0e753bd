// torch.ops.sgl_kernel for the operators around the paged 8-bit cache: arguments checked, outputs
// and workspace allocated, the C ABI of mi355_dit.h called.  They stand in C++ because a serving
// loop calls them one by one with a few microseconds of GPU work each, and the host's time is what
// such a call costs: 6.9 us for a block plan (13.2 with checks, arguments and foreign call in
// Python), 6.7 for a store (17.0), 14.6 for an attention of two launches (22.6).  The schemas are
// defined in sgl_kernel/_ops.py.
//
// The checks run on any device, so that a wrong call is refused with the same words everywhere;
// then tensors that are not on a HIP device are refused.  The library itself is loaded before this
// one, with its symbols visible: nothing here names its file.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "../../include/mi355_dit.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// The current stream of t's device.  The library keeps its state by the current device, so a
// tensor on another one is refused.
void* stream_of(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "mi355 kernels need tensors on a HIP device (got a CPU tensor)");
  const auto device = c10::hip::current_device();
  TORCH_CHECK(t.get_device() == device, "tensor on cuda:", (int)t.get_device(), " but the current device is cuda:",
              (int)device, ": wrap the call in torch.cuda.device(...)");
  return c10::hip::getCurrentHIPStream(device).stream();
}

void check_rc(int64_t rc, const char* what) {
  TORCH_CHECK(rc >= 0, what, " failed (code ", rc, "): ", mi355_last_error());
}

template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr(const OptTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

void check_device(const char* what, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.device() == like.device(), what, ": all tensors must be on ", like.device());
}
void check_ints(const char* what, const char* name, const Tensor& t, at::ScalarType dtype, const Tensor& like) {
  TORCH_CHECK(t.scalar_type() == dtype && t.dim() == 1 && t.is_contiguous(), what, ": ", name,
              " must be a contiguous 1-D ", dtype == at::kLong ? "int64" : "int32", " tensor");
  check_device(what, t, like);
}
void check_cache(const char* what, const char* name, const Tensor& cache, const OptTensor& scale, const Tensor& like) {
  TORCH_CHECK(cache.scalar_type() == at::kFloat8_e4m3fn && cache.dim() == 4 && cache.stride(3) == 1, what, ": ", name,
              "_cache must be [blocks, block_size, heads, head_size] float8_e4m3fn with a contiguous last dimension");
  TORCH_CHECK(scale && scale->scalar_type() == at::kFloat && scale->is_contiguous() && scale->dim() == 2 &&
                  scale->size(0) == cache.size(0) && scale->size(1) == cache.size(2),
              what, ": the scales of ", name, "_cache must be contiguous float32 [blocks, heads]");
  check_device(what, cache, like);
  check_device(what, *scale, like);
}
void check_table(const char* what, const char* name, const Tensor& table, int64_t rows, const Tensor& like) {
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == rows &&
                  (table.size(1) <= 1 || table.stride(1) == 1) && table.device() == like.device(),
              what, ": ", name, " must be int32 [sequences, blocks] with contiguous rows, on ", like.device());
}
void check_heads(const char* what, const char* name, const Tensor& x, int64_t tokens, const Tensor& like) {
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 && x.dim() == 3 && x.stride(2) == 1 && x.size(0) == tokens, what, ": ",
              name, " must be bfloat16 [tokens, heads, head_size] with a contiguous last dimension");
  check_device(what, x, like);
}
void check_inv_freq(const char* what, const Tensor& f, const Tensor& like) {
  TORCH_CHECK((f.scalar_type() == at::kDouble || f.scalar_type() == at::kFloat) && f.dim() == 1 && f.is_contiguous() &&
                  f.device() == like.device(),
              what, ": inv_freq must be a contiguous 1-D float64 or float32 tensor on ", like.device());
}

// ------------------------------------------------------------------------------------ plan --
void kv_block_plan(const Tensor& context_lens, const Tensor& new_lens, const Tensor& block_table,
                   const Tensor& free_blocks, const Tensor& free_begin, int64_t block_size, int64_t num_blocks,
                   const Tensor& slot_mapping, const Tensor& positions, const Tensor& cu_seqlens_q,
                   const Tensor& seq_lens, const Tensor& free_end, const Tensor& status) {
  constexpr const char* what = "kv_block_plan";
  check_ints(what, "context_lens", context_lens, at::kInt, slot_mapping);
  check_ints(what, "new_lens", new_lens, at::kInt, slot_mapping);
  check_ints(what, "free_blocks", free_blocks, at::kInt, slot_mapping);
  check_ints(what, "free_begin", free_begin, at::kInt, slot_mapping);
  check_ints(what, "cu_seqlens_q", cu_seqlens_q, at::kInt, slot_mapping);
  check_ints(what, "seq_lens", seq_lens, at::kInt, slot_mapping);
  check_ints(what, "free_end", free_end, at::kInt, slot_mapping);
  check_ints(what, "status", status, at::kInt, slot_mapping);
  check_ints(what, "slot_mapping", slot_mapping, at::kLong, slot_mapping);
  check_ints(what, "positions", positions, at::kLong, slot_mapping);
  const int64_t B = context_lens.numel();
  TORCH_CHECK(new_lens.numel() == B && seq_lens.numel() == B && cu_seqlens_q.numel() == B + 1, what,
              ": new_lens and seq_lens must have one entry for each request, cu_seqlens_q one more");
  check_table(what, "block_table", block_table, B, slot_mapping);
  TORCH_CHECK(positions.numel() == slot_mapping.numel(), what, ": positions and slot_mapping differ in length");
  TORCH_CHECK(free_begin.numel() == 1 && free_end.numel() == 1 && status.numel() == 3, what,
              ": free_begin and free_end must have 1 entry, status 3");
  void* stream = stream_of(slot_mapping);
  check_rc(mi355_kv_block_plan(ptr<int32_t>(context_lens), ptr<int32_t>(new_lens), B, ptr<int32_t>(block_table),
                               block_table.stride(0), block_table.size(1), ptr<int32_t>(free_blocks),
                               free_blocks.numel(), ptr<int32_t>(free_begin), block_size, num_blocks,
                               ptr<int64_t>(slot_mapping), ptr<int64_t>(positions), slot_mapping.numel(),
                               ptr<int32_t>(cu_seqlens_q), ptr<int32_t>(seq_lens), ptr<int32_t>(free_end),
                               ptr<int32_t>(status), stream),
           what);
}

// ------------------------------------------------------------------------------------ rope --
void rotary_embedding_scaled(const Tensor& positions, const Tensor& query, const OptTensor& key, const Tensor& inv_freq,
                             double attn_factor, bool is_neox, const Tensor& query_out, const OptTensor& key_out) {
  constexpr const char* what = "rotary_embedding_scaled";
  check_ints(what, "positions", positions, at::kLong, query);
  check_inv_freq(what, inv_freq, query);
  const int64_t T = positions.numel();
  check_heads(what, "query", query, T, query);
  check_heads(what, "query_out", query_out, T, query);
  TORCH_CHECK(query_out.sizes() == query.sizes(), what, ": query_out must have the shape of query");
  TORCH_CHECK(key.has_value() == key_out.has_value(), what, ": key and key_out come together");
  int64_t Hk = 0, ks[4] = {0, 0, 0, 0};
  if (key) {
    check_heads(what, "key", *key, T, query);
    check_heads(what, "key_out", *key_out, T, query);
    TORCH_CHECK(key_out->sizes() == key->sizes() && key->size(2) == query.size(2), what,
                ": key_out must have the shape of key, and both the head size of query");
    Hk = key->size(1);
    ks[0] = key->stride(0), ks[1] = key->stride(1), ks[2] = key_out->stride(0), ks[3] = key_out->stride(1);
  }
  void* stream = stream_of(query);
  check_rc(mi355_rope_scaled(ptr<int64_t>(positions), ptr<void>(query), ptr<void>(query_out), ptr<void>(key),
                             ptr<void>(key_out), T, query.size(1), Hk, query.size(2), 2 * inv_freq.numel(),
                             query.stride(0), query.stride(1), query_out.stride(0), query_out.stride(1), ks[0], ks[1],
                             ks[2], ks[3], ptr<void>(inv_freq), inv_freq.scalar_type() == at::kDouble,
                             (float)attn_factor, is_neox, stream),
           what);
}

// ----------------------------------------------------------------------------------- store --
void store_kv_cache_fp8(const Tensor& key, const Tensor& value, const Tensor& k_cache, const Tensor& v_cache,
                        const Tensor& k_scale, const Tensor& v_scale, const Tensor& slot_mapping,
                        const OptTensor& query, const OptTensor& positions, const OptTensor& inv_freq, double attn_factor, bool is_neox,
                        const OptTensor& query_out) {
  constexpr const char* what = "store_kv_cache_fp8";
  check_ints(what, "slot_mapping", slot_mapping, at::kLong, key);
  const int64_t T = slot_mapping.numel();
  check_heads(what, "key", key, T, key);
  check_heads(what, "value", value, T, key);
  check_cache(what, "k", k_cache, k_scale, key);
  check_cache(what, "v", v_cache, v_scale, key);
  TORCH_CHECK(value.sizes() == key.sizes() && v_cache.sizes() == k_cache.sizes() && k_cache.size(2) == key.size(1) &&
                  k_cache.size(3) == key.size(2),
              what, ": key and value must have one shape, the caches too, with the same heads");
  TORCH_CHECK(positions.has_value() == inv_freq.has_value(), what, ": positions and inv_freq come together");
  TORCH_CHECK(query.has_value() == query_out.has_value(), what, ": query and query_out come together");
  mi355_kv_store_args a = {};
  if (positions) {
    check_ints(what, "positions", *positions, at::kLong, key);
    check_inv_freq(what, *inv_freq, key);
    TORCH_CHECK(positions->numel() == T, what, ": positions and slot_mapping differ in length");
    a.positions = ptr<int64_t>(positions);
    a.inv_freq = ptr<void>(inv_freq);
    a.rot_dim = 2 * inv_freq->numel();
    a.inv_freq_is_f64 = inv_freq->scalar_type() == at::kDouble;
    a.is_neox = is_neox;
    a.attn_factor = (float)attn_factor;
  }
  if (query) {
    TORCH_CHECK(positions, what, ": a query is given to be rotated, and needs positions");
    check_heads(what, "query", *query, T, key);
    check_heads(what, "query_out", *query_out, T, key);
    TORCH_CHECK(query_out->sizes() == query->sizes() && query->size(2) == key.size(2), what,
                ": query_out must have the shape of query, with the head size of key");
    a.Hq = query->size(1);
    a.q = ptr<void>(query);
    a.q_out = ptr<void>(query_out);
    a.q_st = query->stride(0), a.q_sh = query->stride(1);
    a.qo_st = query_out->stride(0), a.qo_sh = query_out->stride(1);
  }
  void* stream = stream_of(key);
  a.k = ptr<void>(key);
  a.v = ptr<void>(value);
  a.k_st = key.stride(0), a.k_sh = key.stride(1);
  a.v_st = value.stride(0), a.v_sh = value.stride(1);
  a.k_cache = ptr<void>(k_cache);
  a.v_cache = ptr<void>(v_cache);
  a.kc_sb = k_cache.stride(0), a.kc_st = k_cache.stride(1), a.kc_sh = k_cache.stride(2);
  a.vc_sb = v_cache.stride(0), a.vc_st = v_cache.stride(1), a.vc_sh = v_cache.stride(2);
  a.k_scale = ptr<float>(k_scale);
  a.v_scale = ptr<float>(v_scale);
  a.slot_mapping = ptr<int64_t>(slot_mapping);
  a.tokens = T;
  a.Hk = key.size(1);
  a.D = key.size(2);
  a.block_size = k_cache.size(1);
  a.num_blocks = k_cache.size(0);
  check_rc(mi355_kv_store_fp8(&a, stream), what);
}

// ---------------------------------------------------------------------------------- attend --
void check_paged(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_descale,
                 const OptTensor& v_descale, const Tensor& page_table, const OptTensor& cache_seqlens,
                 const OptTensor& cu_seqlens_q, bool causal, int64_t window_left, int64_t window_right) {
  constexpr const char* what = "fwd";
  const bool packed = q.dim() == 3;
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && (packed || q.dim() == 4) && q.stride(-1) == 1,
              "fwd: q must be bfloat16 [T,H,d] or [B,S,H,d] with a contiguous last dimension");
  check_cache(what, "k", k_cache, k_descale, q);
  check_cache(what, "v", v_cache, v_descale, q);
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes() && k_cache.size(3) == q.size(-1),
              "fwd: k_cache and v_cache must have one shape, with the head size of q");
  TORCH_CHECK(cache_seqlens, "fwd: a paged cache needs the sequences' lengths (cache_seqlens)");
  const int64_t B = cache_seqlens->numel();
  check_table(what, "page_table", page_table, B, q);
  check_ints(what, "cache_seqlens", *cache_seqlens, at::kInt, q);
  if (packed) {
    TORCH_CHECK(cu_seqlens_q, "fwd: packed q needs cu_seqlens_q");
    check_ints(what, "cu_seqlens_q", *cu_seqlens_q, at::kInt, q);
    TORCH_CHECK(cu_seqlens_q->numel() == B + 1, "fwd: cu_seqlens_q and cache_seqlens disagree");
  } else {
    TORCH_CHECK(!cu_seqlens_q && q.size(0) == B,
                "fwd: batched q needs one sequence for each length and no cu_seqlens_q");
  }
  const int64_t H = q.size(-2), Hk = k_cache.size(2);
  TORCH_CHECK(Hk > 0 && H > 0 && H % Hk == 0, "fwd: the heads of q must be a multiple of the cache's");
  TORCH_CHECK((window_left < 0 && window_right < 0) || (causal && window_right >= -1 && window_right <= 0),
              "fwd: sliding windows need causal attention, and end at the token itself");
}

// lse: [H, T] or [B, H, S].  The workspace comes from the caching allocator: it belongs to the
// current stream, or to the graph that is being captured.
void run_paged(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_descale,
               const OptTensor& v_descale, const Tensor& page_table, const OptTensor& cache_seqlens,
               const OptTensor& cu_seqlens_q, std::optional<int64_t> max_seqlen_q, std::optional<double> softmax_scale,
               bool causal, int64_t window_left, const Tensor& out, const Tensor& lse) {
  const bool packed = q.dim() == 3;
  mi355_paged_attn_args a = {};
  a.B = page_table.size(0);
  if (q.numel() == 0 || a.B == 0) return;
  void* stream = stream_of(q);
  a.Sq = q.size(-3);
  a.H = q.size(-2);
  a.D = q.size(-1);
  a.Hk = k_cache.size(2);
  a.q = ptr<void>(q);
  a.out = ptr<void>(out);
  a.lse = ptr<float>(lse);
  a.k_cache = ptr<void>(k_cache);
  a.v_cache = ptr<void>(v_cache);
  a.k_scale = ptr<float>(k_descale);
  a.v_scale = ptr<float>(v_descale);
  a.cu_seqlens_q = ptr<int32_t>(cu_seqlens_q);
  a.cache_seqlens = ptr<int32_t>(cache_seqlens);
  a.page_table = ptr<int32_t>(page_table);
  a.max_seqlen_q = packed ? max_seqlen_q.value_or(a.Sq) : a.Sq;
  a.q_sb = packed ? 0 : q.stride(0), a.q_ss = q.stride(-3), a.q_sh = q.stride(-2);
  a.o_sb = packed ? 0 : out.stride(0), a.o_ss = out.stride(-3), a.o_sh = out.stride(-2);
  a.lse_sb = packed ? 0 : a.H * a.Sq, a.lse_sh = a.Sq;
  a.kc_sb = k_cache.stride(0), a.kc_st = k_cache.stride(1), a.kc_sh = k_cache.stride(2);
  a.vc_sb = v_cache.stride(0), a.vc_st = v_cache.stride(1), a.vc_sh = v_cache.stride(2);
  a.table_stride = page_table.stride(0);
  a.table_width = page_table.size(1);
  a.num_blocks = k_cache.size(0);
  a.block_size = k_cache.size(1);
  a.softmax_scale = (float)(softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)a.D));
  a.causal = causal;
  a.window_left = window_left;
  const int64_t need = mi355_paged_attn_workspace_bytes(&a);
  check_rc(need, "paged_attn_fp8");
  Tensor workspace;
  if (need) {
    workspace = at::empty({need}, q.options().dtype(at::kByte));
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = need;
  }
  check_rc(mi355_paged_attn_fp8(&a, stream), "paged_attn_fp8");
}

at::Tensor empty_lse(const Tensor& q) {
  const auto options = q.options().dtype(at::kFloat);
  if (q.dim() == 3) return at::empty({q.size(1), q.size(0)}, options);
  return at::empty({q.size(0), q.size(2), q.size(1)}, options);
}

std::tuple<Tensor, Tensor> fwd_paged_fp8(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                         const OptTensor& k_descale, const OptTensor& v_descale,
                                         const Tensor& page_table, const OptTensor& cache_seqlens,
                                         const OptTensor& cu_seqlens_q, std::optional<int64_t> max_seqlen_q,
                                         std::optional<double> softmax_scale, bool causal, int64_t window_left,
                                         int64_t window_right) {
  check_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, causal, window_left,
              window_right);
  const Tensor out = at::empty(q.sizes(), q.options()), lse = empty_lse(q);
  run_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q,
            softmax_scale, causal, window_left, out, lse);
  return {out, lse};
}

// the same into a given `out`; returns the log-sum-exp
Tensor fwd_paged_fp8_out(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const OptTensor& k_descale,
                         const OptTensor& v_descale, const Tensor& page_table, const OptTensor& cache_seqlens,
                         const OptTensor& cu_seqlens_q, std::optional<int64_t> max_seqlen_q,
                         std::optional<double> softmax_scale, bool causal, int64_t window_left, int64_t window_right,
                         const Tensor& out) {
  check_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, causal, window_left,
              window_right);
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.stride(-1) == 1 &&
                  out.device() == q.device(),
              "fwd: out must match q");
  const Tensor lse = empty_lse(q);
  run_paged(q, k_cache, v_cache, k_descale, v_descale, page_table, cache_seqlens, cu_seqlens_q, max_seqlen_q,
            softmax_scale, causal, window_left, out, lse);
  return lse;
}

void implement(torch::Library& m) {
  m.impl("kv_block_plan", kv_block_plan);
  m.impl("rotary_embedding_scaled", rotary_embedding_scaled);
  m.impl("store_kv_cache_fp8", store_kv_cache_fp8);
  m.impl("fwd_paged_fp8", fwd_paged_fp8);
  m.impl("fwd_paged_fp8_out", fwd_paged_fp8_out);
}

}  // namespace

TORCH_LIBRARY_IMPL(sgl_kernel, CUDA, m) { implement(m); }
TORCH_LIBRARY_IMPL(sgl_kernel, CPU, m) { implement(m); }
