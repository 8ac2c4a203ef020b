// C ABI of the head norm and rotation and of the paged cache append: argument checks
// and dispatch (include/ifa4.h, kernels in norm_rope.hip).
#include "ifa4.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "ifa4_kernels.h"

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// 16-byte rows of `heads` heads; written rows must not overlap.  The stride of a dimension of one
// is never stepped along: it says nothing.
int32_t check_rows(const void* p, int64_t total, int64_t heads, int64_t st, int64_t sh, int d,
                   bool written) {
  if (st < 0 || sh < 0) return IFA4_EINVAL;
  if (total == 0 || heads == 0) return IFA4_OK;
  if (p == nullptr) return IFA4_EINVAL;
  if (!aligned(p, 16) || ((total > 1 ? st : 0) | (heads > 1 ? sh : 0)) % 8 != 0)
    return IFA4_EUNSUPPORTED;
  if (written && ((heads > 1 && sh < d) || (total > 1 && st < d))) return IFA4_EUNSUPPORTED;
  return IFA4_OK;
}

// What forward, backward and append share; outputs and positions are checked by each.
int32_t check_norm_rope(const ifa4_norm_rope* a) {
  if (a == nullptr || a->struct_size != sizeof(ifa4_norm_rope)) return IFA4_EINVAL;
  if (a->n_heads < 0 || a->kv_heads < 0 || a->head_dim < 1) return IFA4_EINVAL;
  if (a->total < 0 || a->rot_dim < 0 || a->rot_dim > a->head_dim) return IFA4_EINVAL;
  if (a->interleaved != 0 && a->interleaved != 1) return IFA4_EINVAL;
  if (a->dtype < IFA4_BF16 || a->dtype > IFA4_FP32) return IFA4_EINVAL;
  if (!std::isfinite(a->eps) || a->eps < 0.f) return IFA4_EINVAL;
  if (a->head_dim != 64 && a->head_dim != 128) return IFA4_EUNSUPPORTED;
  if (a->dtype == IFA4_FP32 || a->rot_dim % 16 != 0) return IFA4_EUNSUPPORTED;
  if (a->total > INT32_MAX) return IFA4_EUNSUPPORTED;
  if ((int64_t)a->n_heads + 2 * (int64_t)a->kv_heads > (1 << 20)) return IFA4_EUNSUPPORTED;
  if (a->q_weight != nullptr || a->k_weight != nullptr) {
    if (a->w_dtype < IFA4_BF16 || a->w_dtype > IFA4_FP32) return IFA4_EINVAL;
    const uintptr_t esize = a->w_dtype == IFA4_FP32 ? 4 : 2;
    if (!aligned(a->q_weight, esize) || !aligned(a->k_weight, esize)) return IFA4_EINVAL;
  }
  if (a->rot_dim > 0) {
    if (a->cos == nullptr || a->sin == nullptr || a->max_position < 1) return IFA4_EINVAL;
    if (a->angle_stride < a->rot_dim / 2) return IFA4_EINVAL;
    if (!aligned(a->cos, 16) || !aligned(a->sin, 16) || a->angle_stride % 4 != 0)
      return IFA4_EUNSUPPORTED;
  }
  int32_t st = check_rows(a->q, a->total, a->n_heads, a->q_stride_t, a->q_stride_h, a->head_dim, false);
  if (st != IFA4_OK) return st;
  return check_rows(a->k, a->total, a->kv_heads, a->k_stride_t, a->k_stride_h, a->head_dim, false);
}

int32_t check_positions(const ifa4_norm_rope* a) {
  if (a->rot_dim == 0 || a->total == 0) return IFA4_OK;
  return a->positions != nullptr && aligned(a->positions, 4) ? IFA4_OK : IFA4_EINVAL;
}

ifa4::NormRopeParams make_params(const ifa4_norm_rope* a) {
  ifa4::NormRopeParams p{};
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.q_st = a->q_stride_t;
  p.q_sh = a->q_stride_h;
  p.k_st = a->k_stride_t;
  p.k_sh = a->k_stride_h;
  p.qo_st = a->q_out_stride_t;
  p.qo_sh = a->q_out_stride_h;
  p.ko_st = a->k_out_stride_t;
  p.ko_sh = a->k_out_stride_h;
  p.q_weight = a->q_weight;
  p.k_weight = a->k_weight;
  p.cos = a->cos;
  p.sin = a->sin;
  p.positions = a->rot_dim > 0 ? a->positions : nullptr;
  p.angle_stride = a->angle_stride;
  p.total = a->total;
  p.n_heads = a->n_heads;
  p.kv_heads = a->kv_heads;
  p.w_dtype = a->w_dtype;
  p.rot = a->rot_dim;
  p.pairs = a->interleaved;
  p.max_position = a->max_position;
  p.eps = a->eps;
  return p;
}

// Paged cache of kv_heads x head_dim rows of esize bytes that the call writes.
int32_t check_cache(const ifa4_norm_rope* a, const ifa4_kv_append* ap, const ifa4_paged_kv* kv) {
  if (ap->batch < 0) return IFA4_EINVAL;
  const bool fp8 = ap->kv_dtype == IFA4_FP8_E4M3;
  if (!fp8 && ap->kv_dtype != a->dtype) return IFA4_EUNSUPPORTED;
  if (fp8 && (!std::isfinite(ap->k_scale) || !std::isfinite(ap->v_scale) || !(ap->k_scale > 0.f) ||
              !(ap->v_scale > 0.f) || !std::isfinite(1.f / ap->k_scale) ||
              !std::isfinite(1.f / ap->v_scale)))
    return IFA4_EINVAL;
  const int32_t bs = kv->block_size;
  if (bs < 8 || bs > 65536 || (bs & (bs - 1)) != 0) return IFA4_EINVAL;
  if (kv->block_table_stride < 0 || kv->k_stride_block < 0 || kv->v_stride_block < 0 ||
      kv->num_blocks < 0 || kv->max_blocks_per_seq < 0)
    return IFA4_EINVAL;
  if (ap->k_cache_stride_t < 0 || ap->k_cache_stride_h < 0 || ap->v_cache_stride_t < 0 ||
      ap->v_cache_stride_h < 0)
    return IFA4_EINVAL;
  const int32_t st = check_rows(ap->v, a->total, a->kv_heads, ap->v_stride_t, ap->v_stride_h,
                                a->head_dim, false);
  if (st != IFA4_OK || ap->batch == 0 || a->total == 0) return st;
  if (ap->cu_seqlens == nullptr || kv->block_table == nullptr || kv->seqused_k == nullptr ||
      ap->k_cache == nullptr || ap->v_cache == nullptr || !aligned(ap->cu_seqlens, 4) ||
      !aligned(kv->block_table, 4) || !aligned(kv->seqused_k, 4))
    return IFA4_EINVAL;
  if (kv->num_blocks < 1 || kv->max_blocks_per_seq < 1) return IFA4_EINVAL;
  if ((int64_t)kv->max_blocks_per_seq * bs > (int64_t(1) << 30)) return IFA4_EUNSUPPORTED;
  const int64_t unit = fp8 ? 16 : 8;
  int64_t steps = ap->k_cache_stride_t | ap->v_cache_stride_t;
  if (a->kv_heads > 1) steps |= ap->k_cache_stride_h | ap->v_cache_stride_h;
  if (kv->num_blocks > 1) steps |= kv->k_stride_block | kv->v_stride_block;
  if (steps % unit != 0 || !aligned(ap->k_cache, 16) || !aligned(ap->v_cache, 16))
    return IFA4_EUNSUPPORTED;
  // rows of the cache must not overlap
  const int64_t d = a->head_dim;
  if (ap->k_cache_stride_t < d || ap->v_cache_stride_t < d ||
      (a->kv_heads > 1 && (ap->k_cache_stride_h < d || ap->v_cache_stride_h < d)) ||
      (kv->num_blocks > 1 && (kv->k_stride_block < d || kv->v_stride_block < d)))
    return IFA4_EUNSUPPORTED;
  return IFA4_OK;
}

int32_t status_of(hipError_t e) { return e == hipSuccess ? IFA4_OK : IFA4_ELAUNCH; }

}  // namespace

extern "C" {

int32_t ifa4_qk_norm_rope_fwd(const ifa4_norm_rope* a, void* stream) {
  int32_t st = check_norm_rope(a);
  if (st != IFA4_OK) return st;
  if (a->n_heads < 1 || a->kv_heads < 1) return IFA4_EINVAL;
  if ((st = check_positions(a)) != IFA4_OK) return st;
  st = check_rows(a->q_out, a->total, a->n_heads, a->q_out_stride_t, a->q_out_stride_h, a->head_dim, true);
  if (st != IFA4_OK) return st;
  st = check_rows(a->k_out, a->total, a->kv_heads, a->k_out_stride_t, a->k_out_stride_h, a->head_dim, true);
  if (st != IFA4_OK || a->total == 0) return st;
  return status_of(ifa4::launch_norm_rope(make_params(a), ifa4::AppendParams{}, 0, a->head_dim,
                                          a->dtype, static_cast<hipStream_t>(stream)));
}

size_t ifa4_qk_norm_rope_bwd_workspace_bytes(const ifa4_norm_rope* a) {
  if (check_norm_rope(a) != IFA4_OK || a->total == 0 || a->n_heads < 1 || a->kv_heads < 1 ||
      (a->q_weight == nullptr && a->k_weight == nullptr))
    return 0;
  const ifa4::NormRopeBwdGrid grid =
      ifa4::norm_rope_bwd_grid(a->total, a->n_heads + a->kv_heads, a->head_dim);
  return (size_t)grid.x * grid.y * 2 * a->head_dim * sizeof(float);
}

int32_t ifa4_qk_norm_rope_bwd(const ifa4_norm_rope* a, const ifa4_norm_rope_grad* gr,
                              void* workspace, size_t workspace_bytes, void* stream) {
  int32_t st = check_norm_rope(a);
  if (st != IFA4_OK) return st;
  if (gr == nullptr || gr->struct_size != sizeof(ifa4_norm_rope_grad)) return IFA4_EINVAL;
  if (a->n_heads < 1 || a->kv_heads < 1) return IFA4_EINVAL;
  if ((st = check_positions(a)) != IFA4_OK) return st;
  if (a->total == 0 || (gr->gq == nullptr && gr->gk == nullptr)) {
    // nothing to sum: a weight's gradient would be zero, which the caller sets
    return gr->dq_weight == nullptr && gr->dk_weight == nullptr ? IFA4_OK : IFA4_EINVAL;
  }
  if ((gr->dq_weight != nullptr) != (gr->gq != nullptr && a->q_weight != nullptr) ||
      (gr->dk_weight != nullptr) != (gr->gk != nullptr && a->k_weight != nullptr))
    return IFA4_EINVAL;
  if (gr->gq != nullptr) {
    st = check_rows(gr->gq, a->total, a->n_heads, gr->gq_stride_t, gr->gq_stride_h, a->head_dim, false);
    if (st != IFA4_OK) return st;
    st = check_rows(gr->dq, a->total, a->n_heads, gr->dq_stride_t, gr->dq_stride_h, a->head_dim, true);
    if (st != IFA4_OK) return st;
  }
  if (gr->gk != nullptr) {
    st = check_rows(gr->gk, a->total, a->kv_heads, gr->gk_stride_t, gr->gk_stride_h, a->head_dim, false);
    if (st != IFA4_OK) return st;
    st = check_rows(gr->dk, a->total, a->kv_heads, gr->dk_stride_t, gr->dk_stride_h, a->head_dim, true);
    if (st != IFA4_OK) return st;
  }
  const uintptr_t esize = a->w_dtype == IFA4_FP32 ? 4 : 2;
  if (!aligned(gr->dq_weight, esize) || !aligned(gr->dk_weight, esize)) return IFA4_EINVAL;
  ifa4::NormRopeGrad g{};
  g.gq = gr->gq;
  g.gk = gr->gk;
  g.dq = gr->dq;
  g.dk = gr->dk;
  g.gq_st = gr->gq_stride_t;
  g.gq_sh = gr->gq_stride_h;
  g.gk_st = gr->gk_stride_t;
  g.gk_sh = gr->gk_stride_h;
  g.dq_st = gr->dq_stride_t;
  g.dq_sh = gr->dq_stride_h;
  g.dk_st = gr->dk_stride_t;
  g.dk_sh = gr->dk_stride_h;
  g.dq_weight = gr->dq_weight;
  g.dk_weight = gr->dk_weight;
  if (gr->dq_weight != nullptr || gr->dk_weight != nullptr) {
    if (workspace == nullptr || !aligned(workspace, 256) ||
        workspace_bytes < ifa4_qk_norm_rope_bwd_workspace_bytes(a))
      return IFA4_EWORKSPACE;
    g.partial = static_cast<float*>(workspace);
  }
  return status_of(ifa4::launch_norm_rope_bwd(make_params(a), g, a->head_dim, a->dtype,
                                              static_cast<hipStream_t>(stream)));
}

int32_t ifa4_kv_append_paged(const ifa4_norm_rope* a, const ifa4_kv_append* ap,
                             const ifa4_paged_kv* kv, void* stream) {
  int32_t st = check_norm_rope(a);
  if (st != IFA4_OK) return st;
  if (ap == nullptr || ap->struct_size != sizeof(ifa4_kv_append)) return IFA4_EINVAL;
  if (kv == nullptr || kv->struct_size != sizeof(ifa4_paged_kv)) return IFA4_EINVAL;
  if (a->kv_heads < 1) return IFA4_EINVAL;
  st = check_rows(a->q_out, a->total, a->n_heads, a->q_out_stride_t, a->q_out_stride_h, a->head_dim, true);
  if (st != IFA4_OK) return st;
  if ((st = check_cache(a, ap, kv)) != IFA4_OK) return st;
  if (a->total == 0 || ap->batch == 0) return IFA4_OK;
  ifa4::AppendParams p{};
  p.v = ap->v;
  p.k_cache = ap->k_cache;
  p.v_cache = ap->v_cache;
  p.cu = ap->cu_seqlens;
  p.seqused_k = kv->seqused_k;
  p.block_table = kv->block_table;
  p.v_st = ap->v_stride_t;
  p.v_sh = ap->v_stride_h;
  p.kc_st = ap->k_cache_stride_t;
  p.kc_sh = ap->k_cache_stride_h;
  p.kc_sblk = kv->k_stride_block;
  p.vc_st = ap->v_cache_stride_t;
  p.vc_sh = ap->v_cache_stride_h;
  p.vc_sblk = kv->v_stride_block;
  p.bt_stride = kv->block_table_stride;
  p.batch = ap->batch;
  p.block_shift = __builtin_ctz((unsigned)kv->block_size);
  p.num_blocks = kv->num_blocks;
  p.max_blocks = kv->max_blocks_per_seq;
  p.k_scale = ap->k_scale;
  p.v_scale = ap->v_scale;
  p.inv_k_scale = 1.f / ap->k_scale;
  p.inv_v_scale = 1.f / ap->v_scale;
  return status_of(ifa4::launch_norm_rope(make_params(a), p, ap->kv_dtype == IFA4_FP8_E4M3 ? 2 : 1,
                                          a->head_dim, a->dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
