// Torch binding of the key bounds and the block choice over the C ABI (include/ifa4.h):
// torch.ops.inkling_fa4.key_bounds_paged / .select_blocks_paged.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "torch_util.h"

namespace {

using ifa4_torch::check_no_tangent;
using ifa4_torch::check_status;
using ifa4_torch::dtype_code;
using ifa4_torch::empty_on;

int32_t kv_code(const at::Tensor& x) {
  return x.scalar_type() == at::kFloat8_e4m3fn ? (int32_t)IFA4_FP8_E4M3 : dtype_code(x.scalar_type());
}

// bounds [num_blocks, kv_heads, 2, head_dim]
void check_bounds(const at::Tensor& bounds, const at::Tensor& on, const char* op) {
  TORCH_CHECK(bounds.is_cuda() && bounds.device() == on.device(), "inkling_fa4.", op,
              ": every tensor must be on one GPU");
  TORCH_CHECK(bounds.dim() == 4 && bounds.size(2) == 2 && bounds.stride(3) == 1 &&
                  bounds.stride(2) == bounds.size(3),
              "inkling_fa4.", op,
              ": bounds must be [num_blocks, kv_heads, 2, head_dim] with the last two dims contiguous");
  TORCH_CHECK(bounds.size(0) <= INT32_MAX, "inkling_fa4.", op, ": pool too large");
  TORCH_CHECK_INDEX(bounds.size(0) > 0, "inkling_fa4.", op, ": the pool has no blocks");
}

// The table's part of an ifa4_paged_kv, its tensors checked.
ifa4_paged_kv table_of(const at::Tensor& cu_q, const at::Tensor& seqused_k,
                       const at::Tensor& block_table, int64_t block_size, int64_t num_blocks,
                       const at::Tensor& on, const char* op) {
  for (const at::Tensor* x : {&cu_q, &seqused_k, &block_table})
    TORCH_CHECK(x->is_cuda() && x->device() == on.device() && x->scalar_type() == at::kInt,
                "inkling_fa4.", op, ": cu_seqlens_q, seqused_k and block_table must be int32 on the "
                "cache's GPU");
  TORCH_CHECK(cu_q.dim() == 1 && cu_q.is_contiguous() && seqused_k.dim() == 1 &&
                  seqused_k.is_contiguous() && block_table.dim() == 2 && block_table.stride(1) == 1,
              "inkling_fa4.", op, ": cu_seqlens_q and seqused_k must be 1-D contiguous, block_table "
              "2-D with contiguous rows");
  TORCH_CHECK(cu_q.numel() >= 1 && seqused_k.numel() == cu_q.numel() - 1 &&
                  block_table.size(0) == seqused_k.numel(),
              "inkling_fa4.", op, ": cu_seqlens_q needs batch + 1 entries, seqused_k / block_table "
              "one row per sequence");
  TORCH_CHECK(block_size > 0 && block_size <= 65536, "inkling_fa4.", op, ": bad block_size");
  ifa4_paged_kv kv{};
  kv.struct_size = sizeof(ifa4_paged_kv);
  kv.block_size = static_cast<int32_t>(block_size);
  kv.block_table = block_table.data_ptr<int32_t>();
  kv.seqused_k = seqused_k.data_ptr<int32_t>();
  kv.block_table_stride = block_table.stride(0);
  kv.num_blocks = static_cast<int32_t>(num_blocks);
  kv.max_blocks_per_seq = static_cast<int32_t>(block_table.size(1));
  return kv;
}

int32_t length(int64_t n, const char* op) {
  TORCH_CHECK(n >= 0 && n <= INT32_MAX, "inkling_fa4.", op, ": length out of range");
  return static_cast<int32_t>(n);
}

hipStream_t stream_of(const at::Tensor& x) {
  return c10::hip::getCurrentHIPStream(x.device().index()).stream();
}

void key_bounds_paged(const at::Tensor& k_cache, const at::Tensor& bounds, const at::Tensor& cu_q,
                      const at::Tensor& seqused_k, const at::Tensor& block_table, int64_t max_q) {
  constexpr const char* op = "key_bounds_paged";
  TORCH_CHECK(k_cache.is_cuda() && k_cache.dim() == 4 && k_cache.stride(3) == 1, "inkling_fa4.", op,
              ": k_cache must be [num_blocks, block_size, kv_heads, head_dim] on a GPU, its last dim "
              "contiguous");
  check_bounds(bounds, k_cache, op);
  TORCH_CHECK(bounds.scalar_type() == k_cache.scalar_type() && bounds.size(0) == k_cache.size(0) &&
                  bounds.size(1) == k_cache.size(2) && bounds.size(3) == k_cache.size(3),
              "inkling_fa4.", op, ": bounds must have k_cache's dtype, blocks, heads and head_dim");
  ifa4_paged_kv kv = table_of(cu_q, seqused_k, block_table, k_cache.size(1), k_cache.size(0), k_cache, op);
  kv.k_stride_block = k_cache.stride(0);
  ifa4_key_bounds a{};
  a.struct_size = sizeof(ifa4_key_bounds);
  a.kv_dtype = kv_code(k_cache);
  a.head_dim = length(k_cache.size(3), op);
  a.kv_heads = length(k_cache.size(2), op);
  a.batch = length(seqused_k.numel(), op);
  a.max_seqlen_q = length(max_q, op);
  a.k_cache = k_cache.data_ptr();
  a.k_stride_t = k_cache.stride(1);
  a.k_stride_h = k_cache.stride(2);
  a.bounds = bounds.data_ptr();
  a.bounds_stride_block = bounds.stride(0);
  a.bounds_stride_h = bounds.stride(1);
  a.cu_seqlens = cu_q.data_ptr<int32_t>();
  const c10::DeviceGuard guard(k_cache.device());
  check_status(ifa4_key_bounds_paged(&a, &kv, stream_of(k_cache)), op);
}

at::Tensor select_blocks_paged(const at::Tensor& q, const at::Tensor& bounds, const at::Tensor& cu_q,
                               const at::Tensor& seqused_k, const at::Tensor& block_table,
                               int64_t block_size, int64_t max_q, int64_t max_k, int64_t n_select,
                               int64_t sink, int64_t recent) {
  constexpr const char* op = "select_blocks_paged";
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.stride(2) == 1, "inkling_fa4.", op,
              ": q must be [tokens, heads, head_dim] on a GPU, its last dim contiguous");
  check_bounds(bounds, q, op);
  TORCH_CHECK(bounds.size(3) == q.size(2) && bounds.size(1) > 0 && q.size(1) % bounds.size(1) == 0,
              "inkling_fa4.", op, ": bounds must have q's head_dim and a divisor of its heads");
  TORCH_CHECK(bounds.scalar_type() == q.scalar_type() || bounds.scalar_type() == at::kFloat8_e4m3fn,
              "inkling_fa4.", op, ": bounds must be of q's dtype or float8_e4m3fn");
  const ifa4_paged_kv kv = table_of(cu_q, seqused_k, block_table, block_size, bounds.size(0), q, op);
  ifa4_block_select a{};
  a.struct_size = sizeof(ifa4_block_select);
  a.dtype = dtype_code(q.scalar_type());
  a.kv_dtype = kv_code(bounds);
  a.head_dim = length(q.size(2), op);
  a.n_heads = length(q.size(1), op);
  a.kv_heads = length(bounds.size(1), op);
  a.batch = length(seqused_k.numel(), op);
  a.max_seqlen_q = length(max_q, op);
  a.max_seqlen_k = length(max_k, op);
  a.n_select = length(n_select, op);
  a.sink_blocks = length(sink, op);
  a.recent_blocks = length(recent, op);
  a.total_q = q.size(0);
  a.q = q.data_ptr();
  a.q_stride_t = q.stride(0);
  a.q_stride_h = q.stride(1);
  a.bounds = bounds.data_ptr();
  a.bounds_stride_block = bounds.stride(0);
  a.bounds_stride_h = bounds.stride(1);
  a.cu_seqlens = cu_q.data_ptr<int32_t>();
  const c10::DeviceGuard guard(q.device());
  const at::Tensor blocks = empty_on(q, {q.size(0), bounds.size(1), n_select}, at::kInt);
  a.blocks = blocks.data_ptr<int32_t>();
  // 0 bytes: no list leaves a block out, or invalid arguments, which the call reports
  const size_t ws_bytes = ifa4_select_blocks_workspace_bytes(&a, &kv);
  const at::Tensor ws = ws_bytes > 0 ? empty_on(q, {(int64_t)ws_bytes}, at::kByte) : at::Tensor();
  check_status(ifa4_select_blocks_paged(&a, &kv, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                                        stream_of(q)),
               op);
  return blocks;
}

// The bounds as a change in place: a graph that has saved them finds them changed.
void key_bounds_in_place(const at::Tensor& k_cache, const at::Tensor& bounds, const at::Tensor& cu_q,
                         const at::Tensor& seqused_k, const at::Tensor& block_table, int64_t max_q) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("inkling_fa4::key_bounds_paged", "")
                             .typed<decltype(key_bounds_paged)>();
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    op.call(k_cache, bounds, cu_q, seqused_k, block_table, max_q);
  }
  if (!bounds.is_inference()) bounds.unsafeGetTensorImpl()->bump_version();
}

// There is no derivative: a tangent is refused, and so are bounds that require a gradient, which
// would go on as if they had not been written.
void key_bounds_autograd(const at::Tensor& k_cache, const at::Tensor& bounds, const at::Tensor& cu_q,
                         const at::Tensor& seqused_k, const at::Tensor& block_table, int64_t max_q) {
  check_no_tangent("key_bounds_paged", k_cache, bounds);
  TORCH_CHECK(!at::GradMode::is_enabled() || !bounds.requires_grad(),
              "inkling_fa4.key_bounds_paged: bounds that require a gradient are written in place");
  key_bounds_in_place(k_cache, bounds, cu_q, seqused_k, block_table, max_q);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(inkling_fa4, m) {
  m.def(
      "key_bounds_paged(Tensor k_cache, Tensor(a!) bounds, Tensor cu_seqlens_q, Tensor seqused_k, "
      "Tensor block_table, int max_seqlen_q) -> ()");
  m.def(
      "select_blocks_paged(Tensor q, Tensor bounds, Tensor cu_seqlens_q, Tensor seqused_k, "
      "Tensor block_table, int block_size, int max_seqlen_q, int max_seqlen_k, int n_select, "
      "int sink_blocks, int recent_blocks) -> Tensor");
}

TORCH_LIBRARY_IMPL(inkling_fa4, CUDA, m) {
  m.impl("key_bounds_paged", &key_bounds_paged);
  m.impl("select_blocks_paged", &select_blocks_paged);
}

// where there is no autograd above it (inference mode)
TORCH_LIBRARY_IMPL(inkling_fa4, ADInplaceOrView, m) {
  m.impl("key_bounds_paged", &key_bounds_in_place);
}

TORCH_LIBRARY_IMPL(inkling_fa4, Autograd, m) {
  m.impl("key_bounds_paged", &key_bounds_autograd);
}
