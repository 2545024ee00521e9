// torch.ops.pageserve_b200.* — the hot-path operators registered with the
// PyTorch dispatcher (CUDA kernels + Meta shape functions for tracing), each a
// thin call into the plain extern "C" core (include/pageserve_b200.h,
// libpageserve_b200.so). No CPU kernels are registered: a CPU tensor raises
// the dispatcher's "no kernel for CPU" error (no CPU fallback).
//
// Operator names and arguments follow the reference's Python functions
// (engine/paged_attention.py, engine/quantization.py, engine/model.py); the
// batched forms take device-resident int32 metadata (graph-capturable).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "../../include/pageserve_b200.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PS_F32;
    case at::kBFloat16: return PS_BF16;
    case at::kHalf: return PS_F16;
    case at::kChar: return PS_I8;
    default: TORCH_CHECK(false, "pageserve_b200: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

ps_stream_t stream_of(const at::Tensor& t) {
  return reinterpret_cast<ps_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void check(int rc, const char* what) {
  if (rc == PS_OK) return;
  const char* msg = ps_last_error();
  TORCH_CHECK_INDEX(rc != PS_ERR_INDEX, what, ": ", msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != PS_ERR_UNSUPPORTED, what, ": ", msg);
  TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}

void* ptr(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

void need_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "pageserve_b200: ", name, " must be a CUDA tensor (no CPU fallback)");
  TORCH_CHECK(t.is_contiguous(), "pageserve_b200: ", name, " must be contiguous");
}

// ---------------------------------------------------------------- CUDA ----

void write_kv(at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& block_table, int64_t block_size,
              int64_t start_pos, const at::Tensor& k, const at::Tensor& v) {
  need_cuda(k_cache, "k_cache"); need_cuda(v_cache, "v_cache"); need_cuda(k, "k"); need_cuda(v, "v");
  need_cuda(block_table, "block_table");
  TORCH_CHECK(block_table.scalar_type() == at::kInt, "block_table must be int32");
  c10::cuda::CUDAGuard g(k_cache.device());
  check(ps_write_kv(k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr<int32_t>(), block_table.numel(),
                    k_cache.size(0), block_size, k_cache.size(2), k_cache.size(3), dtype_code(k), start_pos,
                    k.size(0), k.data_ptr(), v.data_ptr(), stream_of(k)),
        "write_kv");
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& block_tables, const at::Tensor& cu_q, const at::Tensor& start_pos,
                           int64_t max_q_len, int64_t max_ctx) {
  need_cuda(q, "q"); need_cuda(k_cache, "k_cache"); need_cuda(v_cache, "v_cache");
  need_cuda(block_tables, "block_tables"); need_cuda(cu_q, "cu_q"); need_cuda(start_pos, "start_pos");
  c10::cuda::CUDAGuard g(q.device());
  const int B = start_pos.numel(), Hq = q.size(1), D = q.size(2), Hkv = k_cache.size(2);
  at::Tensor out = at::empty_like(q);
  const size_t ws_bytes = ps_paged_attention_workspace_size(B, max_q_len, max_ctx, Hq, Hkv, D);
  at::Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 1)}, q.options().dtype(at::kByte));
  check(ps_paged_attention(out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                           block_tables.data_ptr<int32_t>(), block_tables.size(1), cu_q.data_ptr<int32_t>(),
                           start_pos.data_ptr<int32_t>(), B, q.size(0), max_q_len, max_ctx, k_cache.size(0),
                           k_cache.size(1), Hq, Hkv, D, dtype_code(q), ws.data_ptr(), ws_bytes, stream_of(q)),
        "paged_attention");
  return out;
}

std::tuple<at::Tensor, at::Tensor> quantize_per_channel(const at::Tensor& w) {
  need_cuda(w, "weight");
  c10::cuda::CUDAGuard g(w.device());
  at::Tensor q = at::empty({w.size(0), w.size(1)}, w.options().dtype(at::kChar));
  at::Tensor scale = at::empty({w.size(0), 1}, w.options().dtype(at::kFloat));
  check(ps_quantize_per_channel(q.data_ptr<int8_t>(), scale.data_ptr<float>(), w.data_ptr(), dtype_code(w),
                                w.size(0), w.size(1), stream_of(w)),
        "quantize_per_channel");
  return {q, scale};
}

at::Tensor tile_int8_weight(const at::Tensor& q) {
  need_cuda(q, "q");
  c10::cuda::CUDAGuard g(q.device());
  at::Tensor t = at::empty({static_cast<int64_t>(ps_tiled_int8_weight_bytes(q.size(0), q.size(1)))},
                           q.options().dtype(at::kChar));
  check(ps_tile_int8_weight(t.data_ptr<int8_t>(), q.data_ptr<int8_t>(), q.size(0), q.size(1), stream_of(q)),
        "tile_int8_weight");
  return t;
}

at::Tensor w8a16_linear(const at::Tensor& x, const at::Tensor& q_tiled, const at::Tensor& scale, int64_t N,
                        const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& residual) {
  need_cuda(x, "x"); need_cuda(q_tiled, "q_tiled"); need_cuda(scale, "scale");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t K = x.size(-1), M = x.numel() / K;
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  at::Tensor y = at::empty(sizes, x.options());
  const size_t ws_bytes = ps_w8a16_linear_tiled_workspace_size(M, N, K);
  at::Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 1)}, x.options().dtype(at::kByte));
  check(ps_w8a16_linear_tiled(y.data_ptr(), x.data_ptr(), q_tiled.data_ptr<int8_t>(), scale.data_ptr<float>(),
                              ptr(bias), ptr(residual), M, N, K, dtype_code(x), ws.data_ptr(), ws_bytes,
                              stream_of(x)),
        "w8a16_linear");
  return y;
}

at::Tensor linear16(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>& bias,
                    const c10::optional<at::Tensor>& residual) {
  need_cuda(x, "x"); need_cuda(w, "w");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t K = x.size(-1), M = x.numel() / K, N = w.size(0);
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  at::Tensor y = at::empty(sizes, x.options());
  const size_t ws_bytes = ps_w8a16_linear_tiled_workspace_size(M, N, K);
  at::Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 1)}, x.options().dtype(at::kByte));
  check(ps_linear(y.data_ptr(), x.data_ptr(), w.data_ptr(), ptr(bias), ptr(residual), M, N, K, dtype_code(x),
                  ws.data_ptr(), ws_bytes, stream_of(x)),
        "linear16");
  return y;
}

at::Tensor linear_swiglu(const at::Tensor& x, const at::Tensor& q_tiled, const at::Tensor& scale, int64_t N2) {
  need_cuda(x, "x"); need_cuda(q_tiled, "q_tiled"); need_cuda(scale, "scale");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t K = x.size(-1), M = x.numel() / K;
  auto sizes = x.sizes().vec();
  sizes.back() = N2 / 2;
  at::Tensor y = at::empty(sizes, x.options());
  check(ps_linear_swiglu(y.data_ptr(), x.data_ptr(), nullptr, PS_I8, q_tiled.data_ptr<int8_t>(),
                         scale.data_ptr<float>(), M, N2, K, dtype_code(x), stream_of(x)),
        "linear_swiglu");
  return y;
}

at::Tensor rms_norm(const at::Tensor& x, const at::Tensor& weight, double eps) {
  need_cuda(x, "x"); need_cuda(weight, "weight");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t H = x.size(-1);
  at::Tensor y = at::empty_like(x);
  at::Tensor w = weight.to(x.scalar_type()).contiguous();
  check(ps_rmsnorm(y.data_ptr(), nullptr, x.data_ptr(), nullptr, w.data_ptr(), static_cast<float>(eps),
                   x.numel() / H, H, dtype_code(x), stream_of(x)),
        "rms_norm");
  return y;
}

std::tuple<at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const at::Tensor& residual,
                                                const at::Tensor& weight, double eps) {
  need_cuda(x, "x"); need_cuda(residual, "residual"); need_cuda(weight, "weight");
  c10::cuda::CUDAGuard g(x.device());
  const int64_t H = x.size(-1);
  at::Tensor y = at::empty_like(x), sum = at::empty_like(x);
  at::Tensor w = weight.to(x.scalar_type()).contiguous();
  check(ps_rmsnorm(y.data_ptr(), sum.data_ptr(), x.data_ptr(), residual.data_ptr(), w.data_ptr(),
                   static_cast<float>(eps), x.numel() / H, H, dtype_code(x), stream_of(x)),
        "add_rms_norm");
  return {y, sum};
}

at::Tensor apply_rope(const at::Tensor& x, const at::Tensor& cos, const at::Tensor& sin) {
  need_cuda(x, "x"); need_cuda(cos, "cos"); need_cuda(sin, "sin");
  c10::cuda::CUDAGuard g(x.device());
  at::Tensor out = at::empty_like(x);
  at::Tensor c = cos.to(x.scalar_type()).contiguous(), s = sin.to(x.scalar_type()).contiguous();
  check(ps_apply_rope(out.data_ptr(), x.data_ptr(), c.data_ptr(), s.data_ptr(), x.size(0), x.size(1), x.size(2),
                      dtype_code(x), stream_of(x)),
        "apply_rope");
  return out;
}

at::Tensor embedding(const at::Tensor& ids, const at::Tensor& table) {
  need_cuda(ids, "ids"); need_cuda(table, "table");
  TORCH_CHECK(ids.scalar_type() == at::kLong, "ids must be int64");
  c10::cuda::CUDAGuard g(table.device());
  at::Tensor out = at::empty({ids.numel(), table.size(1)}, table.options());
  check(ps_embedding(out.data_ptr(), ids.data_ptr<int64_t>(), table.data_ptr(), ids.numel(), table.size(1),
                     table.size(0), dtype_code(table), stream_of(table)),
        "embedding");
  return out;
}

at::Tensor argmax(const at::Tensor& logits) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "argmax: 2-D CUDA logits rows");
  c10::cuda::CUDAGuard g(logits.device());
  at::Tensor out = at::empty({logits.size(0)}, logits.options().dtype(at::kInt));
  check(ps_argmax(out.data_ptr<int32_t>(), logits.data_ptr(), logits.size(0), logits.size(1), logits.stride(0),
                  dtype_code(logits), stream_of(logits)),
        "argmax");
  return out;
}

std::tuple<at::Tensor, at::Tensor> topk(const at::Tensor& logits, int64_t k) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "topk: 2-D CUDA logits rows");
  c10::cuda::CUDAGuard g(logits.device());
  at::Tensor vals = at::empty({logits.size(0), k}, logits.options().dtype(at::kFloat));
  at::Tensor idx = at::empty({logits.size(0), k}, logits.options().dtype(at::kInt));
  check(ps_topk(vals.data_ptr<float>(), idx.data_ptr<int32_t>(), logits.data_ptr(), logits.size(0), logits.size(1),
                logits.stride(0), k, dtype_code(logits), stream_of(logits)),
        "topk");
  return {vals, idx};
}

void copy_kv_blocks(at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& pairs) {
  need_cuda(k_cache, "k_cache"); need_cuda(v_cache, "v_cache"); need_cuda(pairs, "pairs");
  TORCH_CHECK(k_cache.dim() == 5 && pairs.scalar_type() == at::kInt, "copy_kv_blocks: (L, NB, bs, Hkv, D) caches, "
              "int32 (n, 2) pairs");
  c10::cuda::CUDAGuard g(k_cache.device());
  check(ps_copy_kv_blocks(k_cache.data_ptr(), v_cache.data_ptr(), pairs.data_ptr<int32_t>(), pairs.numel() / 2,
                          k_cache.size(0), k_cache.size(1), k_cache.size(2), k_cache.size(3), k_cache.size(4),
                          dtype_code(k_cache), stream_of(k_cache)),
        "copy_kv_blocks");
}

// ------------------------------------------------- trees of drafted tokens --
// The checks live here, with the Python exception types of _lib.check, so that
// pageserve_b200/speculative.py adds little to a call.

void check_v(int rc, const char* what) {
  TORCH_CHECK_VALUE(rc != PS_ERR_INVALID, what, ": ", ps_last_error());
  check(rc, what);
}

void on_device(const at::Tensor& t, const at::Device& dev, const char* what) {
  TORCH_CHECK(t.is_cuda(), "pageserve_b200 kernels run on CUDA tensors only (no CPU fallback); got a tensor on ",
              t.device());
  TORCH_CHECK_VALUE(t.device() == dev, what, ": tensors on different devices (", t.device(), ", ", dev, ")");
}

void metadata(const at::Tensor& t, const at::Device& dev, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt && t.is_contiguous(), what, ": metadata must be contiguous int32");
  on_device(t, dev, what);
}

void cache_like(const at::Tensor& k, const at::Tensor& v, const at::Device& dev, const char* what) {
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), what, ": K and V caches differ in shape");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), what, ": K and V caches differ in dtype");
  TORCH_CHECK_VALUE(k.is_contiguous() && v.is_contiguous(), what, ": the caches must be contiguous");
  on_device(k, dev, what);
  on_device(v, dev, what);
}

void mask_words(const at::Tensor& m, int64_t rows, int64_t max_q_len, const at::Device& dev, const char* what) {
  TORCH_CHECK_TYPE(m.scalar_type() == at::kLong && m.is_contiguous(), what, ": tree_mask must be contiguous int64");
  on_device(m, dev, what);
  const int64_t words = (max_q_len + 63) / 64;
  TORCH_CHECK_VALUE(m.dim() == 2 && m.size(0) >= rows && m.size(1) == words, what, ": tree_mask ", m.sizes(),
                    " does not hold ", rows, " rows of ", words, " words");
}

int int_arg(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= INT32_MIN && v <= INT32_MAX, what, ": ", v, " does not fit 32 bits");
  return static_cast<int>(v);
}

// An output of its own storage (operators' outputs must not alias, and a caller
// keeps some of them), without at::empty's dispatch: build_step_tables has seven.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, dev, c10::nullopt));
}

using StepOut = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

// `out` undefined: the tables are an output too.
StepOut step_tables_call(at::Tensor& out, const at::Tensor& seq_lens, const at::Tensor& q_lens,
                              const at::Tensor& block_tables, const at::Tensor& held, const at::Tensor& free_blocks,
                              int64_t num_blocks, int64_t block_size, int64_t total_tokens,
                              const c10::optional<at::Tensor>& parents, c10::optional<int64_t> max_q_len,
                              c10::optional<int64_t> max_ctx) {
  constexpr const char* what = "build_step_tables";
  const at::Device dev = seq_lens.device();
  metadata(seq_lens, dev, what);
  metadata(q_lens, dev, what);
  metadata(block_tables, dev, what);
  metadata(held, dev, what);
  metadata(free_blocks, dev, what);
  if (out.defined()) metadata(out, dev, what);
  const int64_t B = seq_lens.numel(), T = total_tokens;
  TORCH_CHECK_VALUE(B > 0, what, ": empty batch");
  TORCH_CHECK_VALUE(T >= 0, what, ": total_tokens below 0");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.size(0) == B && q_lens.numel() == B && held.numel() == B,
                    what, ": q_lens, held and block_tables need one entry per request");
  TORCH_CHECK_VALUE(!out.defined() || out.sizes() == block_tables.sizes(), what, ": out must have block_tables' shape");
  int64_t words = 0;
  if (parents.has_value()) {
    metadata(*parents, dev, what);
    TORCH_CHECK_VALUE(parents->numel() >= T, what, ": ", parents->numel(), " parents for ", T, " rows");
    TORCH_CHECK_VALUE(max_q_len.has_value(), what, ": max_q_len bounds the trees; pass it with parents");
    words = (std::max<int64_t>(*max_q_len, 0) + 63) / 64;
  }
  c10::cuda::CUDAGuard g(dev);
  at::Tensor mask = parents.has_value() ? fresh({T, words}, at::kLong, dev) : fresh({0}, at::kLong, dev);
  at::Tensor positions = fresh({T}, at::kInt, dev), slots = fresh({T}, at::kInt, dev);
  at::Tensor held_out = fresh({B}, at::kInt, dev), cu_q = fresh({B + 1}, at::kInt, dev);
  at::Tensor used = fresh({1}, at::kInt, dev);
  if (!out.defined()) out = fresh(block_tables.sizes(), at::kInt, dev);
  check_v(ps_build_step_tables_bounded(
              out.data_ptr<int32_t>(), held_out.data_ptr<int32_t>(), cu_q.data_ptr<int32_t>(),
              positions.data_ptr<int32_t>(), slots.data_ptr<int32_t>(),
              parents.has_value() ? mask.data_ptr<int64_t>() : nullptr, used.data_ptr<int32_t>(),
              block_tables.data_ptr<int32_t>(), held.data_ptr<int32_t>(), seq_lens.data_ptr<int32_t>(),
              q_lens.data_ptr<int32_t>(), free_blocks.data_ptr<int32_t>(),
              parents.has_value() ? parents->data_ptr<int32_t>() : nullptr, int_arg(B, what), int_arg(T, what),
              int_arg(max_q_len.value_or(0), what), int_arg(block_tables.size(1), what),
              int_arg(free_blocks.numel(), what), int_arg(num_blocks, what), int_arg(block_size, what),
              int_arg(max_ctx.value_or(INT32_MAX), what), stream_of(seq_lens)),
          what);
  return {held_out, cu_q, positions, slots, mask, used};
}

StepOut build_step_tables_out(at::Tensor out, const at::Tensor& seq_lens, const at::Tensor& q_lens,
                              const at::Tensor& block_tables, const at::Tensor& held, const at::Tensor& free_blocks,
                              int64_t num_blocks, int64_t block_size, int64_t total_tokens,
                              const c10::optional<at::Tensor>& parents, c10::optional<int64_t> max_q_len,
                              c10::optional<int64_t> max_ctx) {
  return step_tables_call(out, seq_lens, q_lens, block_tables, held, free_blocks, num_blocks, block_size, total_tokens,
                          parents, max_q_len, max_ctx);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> build_step_tables(
    const at::Tensor& seq_lens, const at::Tensor& q_lens, const at::Tensor& block_tables, const at::Tensor& held,
    const at::Tensor& free_blocks, int64_t num_blocks, int64_t block_size, int64_t total_tokens,
    const c10::optional<at::Tensor>& parents, c10::optional<int64_t> max_q_len, c10::optional<int64_t> max_ctx) {
  at::Tensor out;
  auto r = step_tables_call(out, seq_lens, q_lens, block_tables, held, free_blocks, num_blocks, block_size,
                                 total_tokens, parents, max_q_len, max_ctx);
  return {out, std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r), std::get<5>(r)};
}

void tree_attention_out(at::Tensor out, const at::Tensor& q_in, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& block_tables, const at::Tensor& cu_q, const at::Tensor& start_pos,
                        const at::Tensor& tree_mask, int64_t max_q_len, int64_t max_ctx,
                        const c10::optional<at::Tensor>& workspace) {
  constexpr const char* what = "tree_attention";
  TORCH_CHECK_VALUE(q_in.dim() == 3 && k_cache.dim() == 4 && block_tables.dim() == 2, what,
                    ": q (T, Hq, D), caches (NB, bs, Hkv, D), block_tables (B, max_blocks)");
  const at::Device dev = q_in.device();
  const int64_t T = q_in.size(0), Hq = q_in.size(1), D = q_in.size(2), B = start_pos.numel();
  TORCH_CHECK_VALUE(k_cache.size(3) == D, what, ": cache / query head_dim mismatch");
  TORCH_CHECK_TYPE(q_in.scalar_type() == k_cache.scalar_type(), what, ": q and cache dtypes differ");
  cache_like(k_cache, v_cache, dev, what);
  metadata(block_tables, dev, what);
  metadata(cu_q, dev, what);
  metadata(start_pos, dev, what);
  TORCH_CHECK_VALUE(block_tables.size(0) == B && cu_q.numel() == B + 1, what,
                    ": block_tables, cu_q and start_pos disagree on the batch");
  mask_words(tree_mask, T, max_q_len, dev, what);
  TORCH_CHECK_VALUE(out.sizes() == q_in.sizes() && out.is_contiguous() && out.device() == dev &&
                        out.scalar_type() == q_in.scalar_type(),
                    what, ": out must be contiguous, with q's shape, dtype and device");
  c10::cuda::CUDAGuard g(dev);
  const at::Tensor q = q_in.contiguous();
  const int nb = int_arg(k_cache.size(0), what), bs = int_arg(k_cache.size(1), what);
  const int hq = int_arg(Hq, what), hkv = int_arg(k_cache.size(2), what), d = int_arg(D, what);
  const int mq = int_arg(max_q_len, what), mc = int_arg(max_ctx, what), b = int_arg(B, what);
  const size_t bytes = ps_tree_attention_workspace_size(b, mq, mc, hq, hkv, d);
  at::Tensor ws;
  if (workspace.has_value()) {
    on_device(*workspace, dev, what);
    TORCH_CHECK_VALUE(workspace->is_contiguous(), what, ": the workspace must be contiguous");
    ws = *workspace;
  } else {
    ws = at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, q.options().dtype(at::kByte));
  }
  check_v(ps_tree_attention(out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                            block_tables.data_ptr<int32_t>(), int_arg(block_tables.size(1), what),
                            cu_q.data_ptr<int32_t>(), start_pos.data_ptr<int32_t>(), tree_mask.data_ptr<int64_t>(), b,
                            int_arg(T, what), mq, mc, nb, bs, hq, hkv, d, dtype_code(q), ws.data_ptr(), ws.nbytes(),
                            stream_of(q)),
          what);
}

at::Tensor tree_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                          const at::Tensor& block_tables, const at::Tensor& cu_q, const at::Tensor& start_pos,
                          const at::Tensor& tree_mask, int64_t max_q_len, int64_t max_ctx,
                          const c10::optional<at::Tensor>& workspace) {
  at::Tensor out = at::empty(q.sizes(), q.options());
  tree_attention_out(out, q, k_cache, v_cache, block_tables, cu_q, start_pos, tree_mask, max_q_len, max_ctx, workspace);
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> accept_trees(
    const at::Tensor& tokens, const at::Tensor& targets, const at::Tensor& tree_mask, const at::Tensor& cu_q,
    const at::Tensor& start_pos, int64_t max_q_len, const c10::optional<at::Tensor>& k_cache,
    const c10::optional<at::Tensor>& v_cache, const c10::optional<at::Tensor>& block_tables) {
  constexpr const char* what = "accept_trees";
  const at::Device dev = tokens.device();
  metadata(targets, dev, what);
  metadata(cu_q, dev, what);
  metadata(start_pos, dev, what);
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong && tokens.is_contiguous(), what,
                   ": tokens must be contiguous int64");
  const int64_t T = tokens.numel(), B = start_pos.numel();
  TORCH_CHECK_VALUE(targets.numel() == T && cu_q.numel() == B + 1, what,
                    ": one target per token and one start position per request are needed");
  TORCH_CHECK_VALUE(B > 0, what, ": empty batch");
  mask_words(tree_mask, T, max_q_len, dev, what);
  int L = 0, nb = 0, bs = 0, hkv = 0, d = 0, width = 0, code = 0;
  if (k_cache.has_value() || v_cache.has_value()) {
    TORCH_CHECK_VALUE(k_cache.has_value() && v_cache.has_value() && block_tables.has_value(), what,
                      ": the move needs both caches and block_tables");
    const at::Tensor& k = *k_cache;
    cache_like(k, *v_cache, dev, what);
    metadata(*block_tables, dev, what);
    TORCH_CHECK_VALUE(block_tables->dim() == 2 && block_tables->size(0) == B, what,
                      ": block_tables needs one row per request");
    TORCH_CHECK_VALUE(k.dim() == 4 || k.dim() == 5, what,
                      ": caches are (L, NB, bs, Hkv, D) or one layer's (NB, bs, Hkv, D)");
    L = k.dim() == 5 ? int_arg(k.size(0), what) : 1;
    nb = int_arg(k.size(-4), what);
    bs = int_arg(k.size(-3), what);
    hkv = int_arg(k.size(-2), what);
    d = int_arg(k.size(-1), what);
    width = int_arg(block_tables->size(1), what);
    code = dtype_code(k);
  }
  c10::cuda::CUDAGuard g(dev);
  const int64_t wide = std::max<int64_t>(max_q_len, 0);  // the C call refuses 0 and below
  at::Tensor num = fresh({B}, at::kInt, dev), start = fresh({B}, at::kInt, dev);
  at::Tensor nodes = fresh({B, wide}, at::kInt, dev), out = fresh({B, wide}, at::kInt, dev);
  check_v(ps_accept_trees(num.data_ptr<int32_t>(), nodes.data_ptr<int32_t>(), out.data_ptr<int32_t>(),
                          start.data_ptr<int32_t>(), tokens.data_ptr<int64_t>(), targets.data_ptr<int32_t>(),
                          tree_mask.data_ptr<int64_t>(), cu_q.data_ptr<int32_t>(), start_pos.data_ptr<int32_t>(),
                          int_arg(B, what), int_arg(T, what), int_arg(max_q_len, what), ptr(k_cache), ptr(v_cache),
                          k_cache.has_value() ? block_tables->data_ptr<int32_t>() : nullptr, width, L, nb, bs, hkv, d,
                          code, stream_of(tokens)),
          what);
  return {num, nodes, out, start};
}

// ---------------------------------------------------------------- Meta ----
// Output shapes only (torch.compile / fake-tensor tracing).

at::Tensor paged_attention_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                const at::Tensor&, const at::Tensor&, int64_t, int64_t) {
  return at::empty_like(q);
}
std::tuple<at::Tensor, at::Tensor> quantize_meta(const at::Tensor& w) {
  return {at::empty({w.size(0), w.size(1)}, w.options().dtype(at::kChar)),
          at::empty({w.size(0), 1}, w.options().dtype(at::kFloat))};
}
at::Tensor w8a16_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, int64_t N,
                      const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&) {
  auto s = x.sizes().vec();
  s.back() = N;
  return at::empty(s, x.options());
}
at::Tensor linear16_meta(const at::Tensor& x, const at::Tensor& w, const c10::optional<at::Tensor>&,
                         const c10::optional<at::Tensor>&) {
  auto s = x.sizes().vec();
  s.back() = w.size(0);
  return at::empty(s, x.options());
}
at::Tensor swiglu_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, int64_t N2) {
  auto s = x.sizes().vec();
  s.back() = N2 / 2;
  return at::empty(s, x.options());
}
at::Tensor rms_norm_meta(const at::Tensor& x, const at::Tensor&, double) { return at::empty_like(x); }
std::tuple<at::Tensor, at::Tensor> add_rms_norm_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&,
                                                     double) {
  return {at::empty_like(x), at::empty_like(x)};
}
at::Tensor apply_rope_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&) { return at::empty_like(x); }
at::Tensor argmax_meta(const at::Tensor& l) { return at::empty({l.size(0)}, l.options().dtype(at::kInt)); }
std::tuple<at::Tensor, at::Tensor> topk_meta(const at::Tensor& l, int64_t k) {
  return {at::empty({l.size(0), k}, l.options().dtype(at::kFloat)),
          at::empty({l.size(0), k}, l.options().dtype(at::kInt))};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> step_tables_meta(
    const at::Tensor& seq_lens, const at::Tensor&, const at::Tensor& block_tables, const at::Tensor&,
    const at::Tensor&, int64_t, int64_t, int64_t T, const c10::optional<at::Tensor>& parents,
    c10::optional<int64_t> max_q_len, c10::optional<int64_t>) {
  const auto i32 = seq_lens.options();
  const int64_t B = seq_lens.numel();
  auto mask = parents.has_value() ? at::empty({T, (max_q_len.value_or(0) + 63) / 64}, i32.dtype(at::kLong))
                                  : at::empty({0}, i32.dtype(at::kLong));
  return {at::empty(block_tables.sizes(), i32), at::empty({B}, i32), at::empty({B + 1}, i32), at::empty({T}, i32),
          at::empty({T}, i32), mask, at::empty({1}, i32)};
}
StepOut step_tables_out_meta(at::Tensor, const at::Tensor& seq_lens, const at::Tensor& q_lens,
                             const at::Tensor& block_tables, const at::Tensor& held, const at::Tensor& free_blocks,
                             int64_t num_blocks, int64_t block_size, int64_t T,
                             const c10::optional<at::Tensor>& parents, c10::optional<int64_t> max_q_len,
                             c10::optional<int64_t> max_ctx) {
  auto r = step_tables_meta(seq_lens, q_lens, block_tables, held, free_blocks, num_blocks, block_size, T, parents,
                            max_q_len, max_ctx);
  return {std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r), std::get<5>(r), std::get<6>(r)};
}
void tree_attention_out_meta(at::Tensor, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                             const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t,
                             const c10::optional<at::Tensor>&) {}
at::Tensor tree_attention_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                               const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t,
                               const c10::optional<at::Tensor>&) {
  return at::empty(q.sizes(), q.options());
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> accept_meta(
    const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor& start_pos,
    int64_t max_q_len, const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&,
    const c10::optional<at::Tensor>&) {
  const auto i32 = start_pos.options();
  const int64_t B = start_pos.numel();
  return {at::empty({B}, i32), at::empty({B, max_q_len}, i32), at::empty({B, max_q_len}, i32), at::empty({B}, i32)};
}

}  // namespace

TORCH_LIBRARY(pageserve_b200, m) {
  m.def("write_kv(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, int block_size, int start_pos, "
        "Tensor k, Tensor v) -> ()");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor cu_q, "
        "Tensor start_pos, int max_q_len, int max_ctx) -> Tensor");
  m.def("quantize_per_channel(Tensor weight) -> (Tensor, Tensor)");
  m.def("tile_int8_weight(Tensor q) -> Tensor");
  m.def("w8a16_linear(Tensor x, Tensor q_tiled, Tensor scale, int N, Tensor? bias=None, Tensor? residual=None) "
        "-> Tensor");
  m.def("linear16(Tensor x, Tensor w, Tensor? bias=None, Tensor? residual=None) -> Tensor");
  m.def("linear_swiglu(Tensor x, Tensor q_tiled, Tensor scale, int N2) -> Tensor");
  m.def("rms_norm(Tensor x, Tensor weight, float eps) -> Tensor");
  m.def("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor)");
  m.def("apply_rope(Tensor x, Tensor cos, Tensor sin) -> Tensor");
  m.def("embedding(Tensor ids, Tensor table) -> Tensor");
  m.def("argmax(Tensor logits) -> Tensor");
  m.def("topk(Tensor logits, int k) -> (Tensor, Tensor)");
  m.def("copy_kv_blocks(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor pairs) -> ()");
  m.def("build_step_tables(Tensor seq_lens, Tensor q_lens, Tensor block_tables, Tensor held, Tensor free_blocks, "
        "int num_blocks, int block_size, int total_tokens, Tensor? parents=None, int? max_q_len=None, "
        "int? max_ctx=None) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("build_step_tables_out(Tensor(a!) out, Tensor seq_lens, Tensor q_lens, Tensor block_tables, Tensor held, "
        "Tensor free_blocks, int num_blocks, int block_size, int total_tokens, Tensor? parents=None, "
        "int? max_q_len=None, int? max_ctx=None) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("tree_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor cu_q, Tensor start_pos, "
        "Tensor tree_mask, int max_q_len, int max_ctx, Tensor? workspace=None) -> Tensor");
  m.def("tree_attention_out(Tensor(a!) out, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, "
        "Tensor cu_q, Tensor start_pos, Tensor tree_mask, int max_q_len, int max_ctx, Tensor? workspace=None) -> ()");
  m.def("accept_trees(Tensor tokens, Tensor targets, Tensor tree_mask, Tensor cu_q, Tensor start_pos, int max_q_len, "
        "Tensor(a!)? k_cache=None, Tensor(b!)? v_cache=None, Tensor? block_tables=None) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(pageserve_b200, CUDA, m) {
  m.impl("write_kv", &write_kv);
  m.impl("paged_attention", &paged_attention);
  m.impl("quantize_per_channel", &quantize_per_channel);
  m.impl("tile_int8_weight", &tile_int8_weight);
  m.impl("w8a16_linear", &w8a16_linear);
  m.impl("linear16", &linear16);
  m.impl("linear_swiglu", &linear_swiglu);
  m.impl("rms_norm", &rms_norm);
  m.impl("add_rms_norm", &add_rms_norm);
  m.impl("apply_rope", &apply_rope);
  m.impl("embedding", &embedding);
  m.impl("argmax", &argmax);
  m.impl("topk", &topk);
  m.impl("copy_kv_blocks", &copy_kv_blocks);
  m.impl("build_step_tables", &build_step_tables);
  m.impl("build_step_tables_out", &build_step_tables_out);
  m.impl("tree_attention", &tree_attention);
  m.impl("tree_attention_out", &tree_attention_out);
  m.impl("accept_trees", &accept_trees);
}

TORCH_LIBRARY_IMPL(pageserve_b200, Meta, m) {
  m.impl("paged_attention", &paged_attention_meta);
  m.impl("quantize_per_channel", &quantize_meta);
  m.impl("w8a16_linear", &w8a16_meta);
  m.impl("linear16", &linear16_meta);
  m.impl("linear_swiglu", &swiglu_meta);
  m.impl("rms_norm", &rms_norm_meta);
  m.impl("add_rms_norm", &add_rms_norm_meta);
  m.impl("apply_rope", &apply_rope_meta);
  m.impl("argmax", &argmax_meta);
  m.impl("topk", &topk_meta);
  m.impl("build_step_tables", &step_tables_meta);
  m.impl("build_step_tables_out", &step_tables_out_meta);
  m.impl("tree_attention", &tree_attention_meta);
  m.impl("tree_attention_out", &tree_attention_out_meta);
  m.impl("accept_trees", &accept_meta);
}
