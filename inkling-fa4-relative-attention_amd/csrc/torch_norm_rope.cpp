// torch.ops.inkling_fa4.qk_norm_rope / .qk_norm_rope_bwd / .kv_append_paged: checks of
// tensors, allocation of the outputs, and the calls of the C ABI (include/ifa4.h) on the
// current stream of the tensors' GPU.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "torch_util.h"

namespace {

using ifa4_torch::check_no_tangent;
using ifa4_torch::check_status;
using ifa4_torch::dtype_code;
using ifa4_torch::empty_on;
using OptTensor = std::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_heads(const at::Tensor& x, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device(), "inkling_fa4.", op, ": ", name,
              " must be on k's GPU");
  TORCH_CHECK(x.dim() == 3 && x.size(0) == like.size(0) && x.size(2) == like.size(2),
              "inkling_fa4.", op, ": ", name, " must be [tokens, heads, head_dim] as k is");
  TORCH_CHECK(x.scalar_type() == like.scalar_type(), "inkling_fa4.", op, ": ", name,
              " must be of k's dtype");
  TORCH_CHECK(x.stride(2) == 1, "inkling_fa4.", op, ": the last dim of ", name,
              " must be contiguous");
}

void check_ints(const at::Tensor& x, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device() && x.scalar_type() == at::kInt &&
                  x.dim() == 1 && x.is_contiguous(),
              "inkling_fa4.", op, ": ", name, " must be int32, 1-D, contiguous, on k's GPU");
}

// The norm and rotation of q (may be absent) and k.
ifa4_norm_rope make_args(const char* op, const OptTensor& q, const at::Tensor& k,
                         const OptTensor& q_weight, const OptTensor& k_weight,
                         const OptTensor& cos, const OptTensor& sin, double eps,
                         bool interleaved) {
  TORCH_CHECK(k.is_cuda(), "inkling_fa4.", op, ": every tensor must be on the GPU");
  check_heads(k, k, op, "k");
  ifa4_norm_rope a{};
  a.struct_size = sizeof(ifa4_norm_rope);
  a.dtype = dtype_code(k.scalar_type());
  TORCH_CHECK(a.dtype == IFA4_BF16 || a.dtype == IFA4_FP16, "inkling_fa4.", op,
              ": q and k must be bf16 or fp16");
  a.total = k.size(0);
  a.kv_heads = static_cast<int32_t>(k.size(1));
  a.head_dim = static_cast<int32_t>(k.size(2));
  a.k = k.data_ptr();
  a.k_stride_t = k.stride(0);
  a.k_stride_h = k.stride(1);
  if (given(q)) {
    check_heads(*q, k, op, "q");
    a.n_heads = static_cast<int32_t>(q->size(1));
    a.q = q->data_ptr();
    a.q_stride_t = q->stride(0);
    a.q_stride_h = q->stride(1);
  }
  const at::ScalarType wt = given(q_weight)   ? q_weight->scalar_type()
                            : given(k_weight) ? k_weight->scalar_type()
                                              : at::kFloat;
  a.w_dtype = dtype_code(wt);
  TORCH_CHECK(a.w_dtype >= 0, "inkling_fa4.", op, ": weights must be bf16, fp16 or fp32");
  auto weight = [&](const OptTensor& w, const char* name) -> const void* {
    if (!given(w)) return nullptr;
    TORCH_CHECK(w->is_cuda() && w->device() == k.device() && w->dim() == 1 &&
                    w->size(0) == k.size(2) && w->is_contiguous() && w->scalar_type() == wt,
                "inkling_fa4.", op, ": ", name,
                " must be [head_dim], contiguous, on k's GPU, both weights of one dtype");
    return w->data_ptr();
  };
  a.q_weight = weight(q_weight, "q_weight");
  a.k_weight = weight(k_weight, "k_weight");
  TORCH_CHECK(given(cos) == given(sin), "inkling_fa4.", op, ": cos and sin come together");
  if (given(cos)) {
    TORCH_CHECK(cos->is_cuda() && cos->device() == k.device() && sin->is_cuda() &&
                    sin->device() == k.device() && cos->scalar_type() == at::kFloat &&
                    sin->scalar_type() == at::kFloat && cos->dim() == 2 &&
                    cos->sizes() == sin->sizes() && cos->stride(1) == 1 && sin->stride(1) == 1 &&
                    (cos->size(0) <= 1 || cos->stride(0) == sin->stride(0)),
                "inkling_fa4.", op,
                ": cos and sin must be fp32 [positions, rot_dim / 2] with contiguous rows, alike, "
                "on k's GPU");
    TORCH_CHECK(cos->size(0) >= 1 && cos->size(0) <= INT32_MAX && 2 * cos->size(1) <= k.size(2),
                "inkling_fa4.", op, ": cos and sin need a row, and at most head_dim / 2 columns");
    a.rot_dim = static_cast<int32_t>(2 * cos->size(1));
    a.max_position = static_cast<int32_t>(cos->size(0));
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    // the stride of a dimension of one row says nothing
    a.angle_stride = cos->size(0) > 1 ? cos->stride(0) : (cos->size(1) + 3) / 4 * 4;
  }
  a.eps = static_cast<float>(eps);
  a.interleaved = interleaved ? 1 : 0;
  return a;
}

void set_positions(ifa4_norm_rope& a, const char* op, const at::Tensor& k,
                   const OptTensor& positions) {
  if (a.rot_dim == 0) return;
  TORCH_CHECK(given(positions), "inkling_fa4.", op, ": the rotation needs positions");
  check_ints(*positions, k, op, "positions");
  TORCH_CHECK(positions->size(0) == k.size(0), "inkling_fa4.", op,
              ": positions needs one entry per token");
  a.positions = positions->data_ptr<int32_t>();
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k,
                                                const OptTensor& q_weight,
                                                const OptTensor& k_weight, const OptTensor& cos,
                                                const OptTensor& sin, const OptTensor& positions,
                                                double eps, bool interleaved) {
  constexpr const char* op = "qk_norm_rope";
  ifa4_norm_rope a = make_args(op, q, k, q_weight, k_weight, cos, sin, eps, interleaved);
  set_positions(a, op, k, positions);
  const c10::DeviceGuard guard(k.device());
  at::Tensor q_out = empty_on(q, q.sizes(), q.scalar_type());
  at::Tensor k_out = empty_on(k, k.sizes(), k.scalar_type());
  a.q_out = q_out.data_ptr();
  a.q_out_stride_t = q_out.stride(0);
  a.q_out_stride_h = q_out.stride(1);
  a.k_out = k_out.data_ptr();
  a.k_out_stride_t = k_out.stride(0);
  a.k_out_stride_h = k_out.stride(1);
  check_status(ifa4_qk_norm_rope_fwd(&a, stream_of(k)), op);
  return {q_out, k_out};
}

// Gradients of q, k, q_weight and k_weight; empty tensors where there is none (an output
// without a gradient, no weight).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd(
    const OptTensor& gq, const OptTensor& gk, const at::Tensor& q, const at::Tensor& k,
    const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& cos,
    const OptTensor& sin, const OptTensor& positions, double eps, bool interleaved) {
  constexpr const char* op = "qk_norm_rope_bwd";
  ifa4_norm_rope a = make_args(op, q, k, q_weight, k_weight, cos, sin, eps, interleaved);
  set_positions(a, op, k, positions);
  const c10::DeviceGuard guard(k.device());
  ifa4_norm_rope_grad g{};
  g.struct_size = sizeof(ifa4_norm_rope_grad);
  at::Tensor dq, dk, dqw, dkw;
  dq = dk = dqw = dkw = at::Tensor();
  auto none = [&] { return empty_on(k, {0}, k.scalar_type()); };
  if (given(gq)) {
    check_heads(*gq, k, op, "gq");
    TORCH_CHECK(gq->size(1) == q.size(1), "inkling_fa4.", op, ": gq must have q's shape");
    dq = empty_on(q, q.sizes(), q.scalar_type());
    g.gq = gq->data_ptr();
    g.gq_stride_t = gq->stride(0);
    g.gq_stride_h = gq->stride(1);
    g.dq = dq.data_ptr();
    g.dq_stride_t = dq.stride(0);
    g.dq_stride_h = dq.stride(1);
    if (given(q_weight)) dqw = empty_on(q, q_weight->sizes(), q_weight->scalar_type());
  }
  if (given(gk)) {
    check_heads(*gk, k, op, "gk");
    TORCH_CHECK(gk->size(1) == k.size(1), "inkling_fa4.", op, ": gk must have k's shape");
    dk = empty_on(k, k.sizes(), k.scalar_type());
    g.gk = gk->data_ptr();
    g.gk_stride_t = gk->stride(0);
    g.gk_stride_h = gk->stride(1);
    g.dk = dk.data_ptr();
    g.dk_stride_t = dk.stride(0);
    g.dk_stride_h = dk.stride(1);
    if (given(k_weight)) dkw = empty_on(k, k_weight->sizes(), k_weight->scalar_type());
  }
  if (a.total == 0) {  // no rows: the weights' gradients are zero
    if (dqw.defined()) dqw.zero_();
    if (dkw.defined()) dkw.zero_();
  } else {
    if (dqw.defined()) g.dq_weight = dqw.data_ptr();
    if (dkw.defined()) g.dk_weight = dkw.data_ptr();
  }
  const size_t ws_bytes = ifa4_qk_norm_rope_bwd_workspace_bytes(&a);
  // torch's allocations are aligned to 512 bytes
  const at::Tensor ws = ws_bytes > 0 ? empty_on(k, {(int64_t)ws_bytes}, at::kByte) : at::Tensor();
  check_status(ifa4_qk_norm_rope_bwd(&a, &g, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                                     stream_of(k)),
               op);
  return {dq.defined() ? dq : none(), dk.defined() ? dk : none(), dqw.defined() ? dqw : none(),
          dkw.defined() ? dkw : none()};
}

// The operators by name: calls that go on to the kernels, or to whatever a caller put before them.
template <typename F>
c10::TypedOperatorHandle<F> operator_named(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// A gradient as the kernels read it: contiguous last dim, 16-byte rows (an expanded, sliced or
// shifted one is copied).
OptTensor gradient_rows(const at::Tensor& g) {
  if (!g.defined()) return std::nullopt;
  const bool fine = g.stride(2) == 1 && g.stride(0) % 8 == 0 && g.stride(1) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0;
  return fine ? g : g.clone(at::MemoryFormat::Contiguous);
}

// qk_norm_rope in an autograd graph.  It keeps the inputs, nothing else; its gradients have
// no gradient of their own.
struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
      const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& cos,
      const OptTensor& sin, const OptTensor& positions, double eps, bool interleaved) {
    static const auto op = operator_named<decltype(qk_norm_rope)>("inkling_fa4::qk_norm_rope");
    const at::AutoDispatchBelowADInplaceOrView below;
    auto [q_out, k_out] =
        op.call(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
    auto kept = [](const OptTensor& t) { return given(t) ? *t : at::Tensor(); };
    ctx->save_for_backward(
        {q, k, kept(q_weight), kept(k_weight), kept(cos), kept(sin), kept(positions)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    return {q_out, k_out};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    static const auto op =
        operator_named<decltype(qk_norm_rope_bwd)>("inkling_fa4::qk_norm_rope_bwd");
    const torch::autograd::variable_list saved = ctx->get_saved_variables();
    bool needs[4];
    size_t edge = 0;  // only tensors that were given have an edge
    for (int i = 0; i < 4; ++i) needs[i] = saved[i].defined() && ctx->needs_input_grad(edge++);
    torch::autograd::variable_list out(9);
    const OptTensor gq = gradient_rows(needs[0] || needs[2] ? grads[0] : at::Tensor());
    const OptTensor gk = gradient_rows(needs[1] || needs[3] ? grads[1] : at::Tensor());
    if (!given(gq) && !given(gk)) return out;
    auto maybe = [&](int i) { return saved[i].defined() ? OptTensor(saved[i]) : std::nullopt; };
    std::optional<at::AutoDispatchBelowADInplaceOrView> below;
    if (!at::GradMode::is_enabled()) below.emplace();
    auto [dq, dk, dqw, dkw] =
        op.call(gq, gk, saved[0], saved[1], maybe(2), maybe(3), maybe(4), maybe(5), maybe(6),
                ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
    if (needs[0] && given(gq)) out[0] = dq;
    if (needs[1] && given(gk)) out[1] = dk;
    if (needs[2] && given(gq)) out[2] = dqw;
    if (needs[3] && given(gk)) out[3] = dkw;
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_autograd(
    const at::Tensor& q, const at::Tensor& k, const OptTensor& q_weight, const OptTensor& k_weight,
    const OptTensor& cos, const OptTensor& sin, const OptTensor& positions, double eps,
    bool interleaved) {
  auto wants = [](const OptTensor& t) { return given(t) && t->requires_grad(); };
  check_no_tangent("qk_norm_rope", q, k, q_weight, k_weight, cos, sin);
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK_VALUE(!wants(cos) && !wants(sin),
                      "inkling_fa4.qk_norm_rope: cos and sin have no gradient");
    if (wants(q) || wants(k) || wants(q_weight) || wants(k_weight)) {
      auto out = QkNormRope::apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
      return {out[0], out[1]};
    }
  }
  static const auto op = operator_named<decltype(qk_norm_rope)>("inkling_fa4::qk_norm_rope");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved);
}

at::Tensor kv_append_paged(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                           const at::Tensor& v_cache, const at::Tensor& cu_seqlens,
                           const at::Tensor& seqused_k, const at::Tensor& block_table,
                           const OptTensor& q, const OptTensor& q_weight,
                           const OptTensor& k_weight, const OptTensor& cos, const OptTensor& sin,
                           double eps, bool interleaved, double k_scale, double v_scale) {
  constexpr const char* op = "kv_append_paged";
  ifa4_norm_rope a = make_args(op, q, k, q_weight, k_weight, cos, sin, eps, interleaved);
  TORCH_CHECK(given(q) || !given(q_weight), "inkling_fa4.", op, ": q_weight without q");
  check_heads(v, k, op, "v");
  TORCH_CHECK(v.size(1) == k.size(1), "inkling_fa4.", op, ": k and v shapes differ");
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_cache.device() == k.device() &&
                  v_cache.device() == k.device(),
              "inkling_fa4.", op, ": k_cache / v_cache must be on k's GPU");
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() &&
                  k_cache.size(2) == k.size(1) && k_cache.size(3) == k.size(2) &&
                  k_cache.stride(3) == 1 && v_cache.stride(3) == 1,
              "inkling_fa4.", op,
              ": k_cache / v_cache must be [num_blocks, block_size, kv_heads, head_dim] with k's "
              "heads and a contiguous last dim");
  const bool fp8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(k_cache.scalar_type() == v_cache.scalar_type() &&
                  (fp8 || k_cache.scalar_type() == k.scalar_type()),
              "inkling_fa4.", op, ": k_cache / v_cache must be of k's dtype or float8_e4m3fn");
  TORCH_CHECK(k_cache.size(0) <= INT32_MAX && k_cache.size(1) <= INT32_MAX, "inkling_fa4.", op,
              ": pool too large");
  check_ints(cu_seqlens, k, op, "cu_seqlens_q");
  check_ints(seqused_k, k, op, "seqused_k");
  TORCH_CHECK(block_table.is_cuda() && block_table.device() == k.device() &&
                  block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
                  block_table.stride(1) == 1,
              "inkling_fa4.", op, ": block_table must be int32, 2-D with contiguous rows, on k's GPU");
  TORCH_CHECK(cu_seqlens.numel() >= 1 && seqused_k.numel() == cu_seqlens.numel() - 1 &&
                  block_table.size(0) == seqused_k.numel(),
              "inkling_fa4.", op, ": cu_seqlens_q needs batch + 1 entries, seqused_k / block_table "
                                  "one row per sequence");
  const c10::DeviceGuard guard(k.device());
  at::Tensor q_out;
  if (given(q)) {
    q_out = empty_on(k, q->sizes(), q->scalar_type());
    a.q_out = q_out.data_ptr();
    a.q_out_stride_t = q_out.stride(0);
    a.q_out_stride_h = q_out.stride(1);
  } else {
    q_out = empty_on(k, {0}, k.scalar_type());
  }
  ifa4_kv_append ap{};
  ap.struct_size = sizeof(ifa4_kv_append);
  ap.kv_dtype = fp8 ? (int32_t)IFA4_FP8_E4M3 : a.dtype;
  ap.v = v.data_ptr();
  ap.v_stride_t = v.stride(0);
  ap.v_stride_h = v.stride(1);
  ap.k_cache = k_cache.data_ptr();
  ap.v_cache = v_cache.data_ptr();
  ap.k_cache_stride_t = k_cache.stride(1);
  ap.k_cache_stride_h = k_cache.stride(2);
  ap.v_cache_stride_t = v_cache.stride(1);
  ap.v_cache_stride_h = v_cache.stride(2);
  ap.cu_seqlens = cu_seqlens.data_ptr<int32_t>();
  ap.batch = static_cast<int32_t>(seqused_k.numel());
  ap.k_scale = static_cast<float>(k_scale);
  ap.v_scale = static_cast<float>(v_scale);
  ifa4_paged_kv kv{};
  kv.struct_size = sizeof(ifa4_paged_kv);
  kv.block_size = static_cast<int32_t>(k_cache.size(1));
  kv.block_table = block_table.data_ptr<int32_t>();
  kv.seqused_k = seqused_k.data_ptr<int32_t>();
  kv.block_table_stride = block_table.stride(0);
  kv.k_stride_block = k_cache.stride(0);
  kv.v_stride_block = v_cache.stride(0);
  kv.num_blocks = static_cast<int32_t>(k_cache.size(0));
  kv.max_blocks_per_seq = static_cast<int32_t>(block_table.size(1));
  check_status(ifa4_kv_append_paged(&a, &ap, &kv, stream_of(k)), op);
  return q_out;
}

// The append as a change in place: a graph that has saved a cache finds it changed.
at::Tensor kv_append_paged_in_place(
    const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
    const at::Tensor& cu_seqlens, const at::Tensor& seqused_k, const at::Tensor& block_table,
    const OptTensor& q, const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& cos,
    const OptTensor& sin, double eps, bool interleaved, double k_scale, double v_scale) {
  static const auto op = operator_named<decltype(kv_append_paged)>("inkling_fa4::kv_append_paged");
  at::Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(k, v, k_cache, v_cache, cu_seqlens, seqused_k, block_table, q, q_weight, k_weight,
                  cos, sin, eps, interleaved, k_scale, v_scale);
  }
  for (const at::Tensor* cache : {&k_cache, &v_cache})
    if (!cache->is_inference()) cache->unsafeGetTensorImpl()->bump_version();
  return out;
}

// The append has no gradient: whatever its inputs ask for, its output never requires one.  A
// tangent is refused, and so is a cache that requires a gradient, which would go on as if it had
// not been written.
at::Tensor kv_append_paged_autograd(
    const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
    const at::Tensor& cu_seqlens, const at::Tensor& seqused_k, const at::Tensor& block_table,
    const OptTensor& q, const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& cos,
    const OptTensor& sin, double eps, bool interleaved, double k_scale, double v_scale) {
  check_no_tangent("kv_append_paged", k, v, k_cache, v_cache, q, q_weight, k_weight, cos, sin);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(k_cache.requires_grad() || v_cache.requires_grad()),
              "inkling_fa4.kv_append_paged: a cache that requires a gradient is written in place");
  return kv_append_paged_in_place(k, v, k_cache, v_cache, cu_seqlens, seqused_k, block_table, q,
                                  q_weight, k_weight, cos, sin, eps, interleaved, k_scale, v_scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(inkling_fa4, m) {
  m.def(
      "qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, "
      "Tensor? sin, Tensor? positions, float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rope_bwd(Tensor? gq, Tensor? gk, Tensor q, Tensor k, Tensor? q_weight, "
      "Tensor? k_weight, Tensor? cos, Tensor? sin, Tensor? positions, float eps, "
      "bool interleaved) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "kv_append_paged(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, "
      "Tensor cu_seqlens_q, Tensor seqused_k, Tensor block_table, Tensor? q, Tensor? q_weight, "
      "Tensor? k_weight, Tensor? cos, Tensor? sin, float eps, bool interleaved, float k_scale, "
      "float v_scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(inkling_fa4, CUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_bwd", &qk_norm_rope_bwd);
  m.impl("kv_append_paged", &kv_append_paged);
}

// where there is no autograd above it (inference mode)
TORCH_LIBRARY_IMPL(inkling_fa4, ADInplaceOrView, m) {
  m.impl("kv_append_paged", &kv_append_paged_in_place);
}

TORCH_LIBRARY_IMPL(inkling_fa4, Autograd, m) {
  m.impl("qk_norm_rope", &qk_norm_rope_autograd);
  m.impl("qk_norm_rope_bwd", torch::autograd::autogradNotImplementedFallback());
  m.impl("kv_append_paged", &kv_append_paged_autograd);
}
