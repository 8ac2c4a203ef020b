// C ABI of the key bounds and the block choice: argument checks and dispatch (include/ifa4.h,
// kernels in block_select.hip).
#include "ifa4.h"

#include <hip/hip_runtime.h>

#include <cstdint>

#include "ifa4_kernels.h"

namespace {

// Workgroups of 256 threads in a grid of less than 2^32 threads.
constexpr int64_t kMostGroups = int64_t(1) << 24;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Block tables, lengths and the new tokens' offsets of `batch` sequences.
int32_t check_table(const ifa4_paged_kv* kv, const int32_t* cu, int32_t batch) {
  const int32_t bs = kv->block_size;
  if (bs < 8 || bs > 65536 || (bs & (bs - 1)) != 0) return IFA4_EINVAL;
  if (kv->block_table_stride < 0 || kv->num_blocks < 0 || kv->max_blocks_per_seq < 0 || batch < 0)
    return IFA4_EINVAL;
  if (batch == 0) return IFA4_OK;
  if (cu == nullptr || kv->block_table == nullptr || kv->seqused_k == nullptr || !aligned(cu, 4) ||
      !aligned(kv->block_table, 4) || !aligned(kv->seqused_k, 4))
    return IFA4_EINVAL;
  if (kv->num_blocks < 1 || kv->max_blocks_per_seq < 1) return IFA4_EINVAL;
  // positions stay in 31 bits; a grid's second dimension holds the sequences
  if ((int64_t)kv->max_blocks_per_seq * bs > (int64_t(1) << 30) || batch > 65535)
    return IFA4_EUNSUPPORTED;
  return IFA4_OK;
}

// Bounds [num_blocks, kv_heads, 2, head_dim]; written ones must not overlap.
int32_t check_bounds(const void* bounds, int64_t sblk, int64_t sh, const ifa4_paged_kv* kv,
                     int kv_heads, int d, int esize, bool written) {
  if (sblk < 0 || sh < 0 || bounds == nullptr) return IFA4_EINVAL;
  const int64_t steps = (kv_heads > 1 ? sh : 0) | (kv->num_blocks > 1 ? sblk : 0);
  if (!aligned(bounds, 16) || steps % (16 / esize) != 0) return IFA4_EUNSUPPORTED;
  if (written && ((kv_heads > 1 && sh < 2 * d) || (kv->num_blocks > 1 && sblk < 2 * d)))
    return IFA4_EUNSUPPORTED;
  return IFA4_OK;
}

int32_t check_key_bounds(const ifa4_key_bounds* a, const ifa4_paged_kv* kv) {
  if (a == nullptr || a->struct_size != sizeof(ifa4_key_bounds)) return IFA4_EINVAL;
  if (kv == nullptr || kv->struct_size != sizeof(ifa4_paged_kv)) return IFA4_EINVAL;
  if (a->kv_heads < 1 || a->head_dim < 1 || a->max_seqlen_q < 0) return IFA4_EINVAL;
  if (a->kv_dtype != IFA4_BF16 && a->kv_dtype != IFA4_FP16 && a->kv_dtype != IFA4_FP8_E4M3)
    return IFA4_EUNSUPPORTED;
  if ((a->head_dim != 64 && a->head_dim != 128) || a->kv_heads > (1 << 16)) return IFA4_EUNSUPPORTED;
  int32_t st = check_table(kv, a->cu_seqlens, a->batch);
  if (st != IFA4_OK || a->batch == 0) return st;
  const int esize = a->kv_dtype == IFA4_FP8_E4M3 ? 1 : 2;
  if (a->k_cache == nullptr || a->k_stride_t < 0 || a->k_stride_h < 0 || kv->k_stride_block < 0)
    return IFA4_EINVAL;
  const int64_t steps = a->k_stride_t | (a->kv_heads > 1 ? a->k_stride_h : 0) |
                        (kv->num_blocks > 1 ? kv->k_stride_block : 0);
  if (!aligned(a->k_cache, 16) || steps % (16 / esize) != 0) return IFA4_EUNSUPPORTED;
  return check_bounds(a->bounds, a->bounds_stride_block, a->bounds_stride_h, kv, a->kv_heads,
                      a->head_dim, esize, true);
}

int32_t check_select(const ifa4_block_select* a, const ifa4_paged_kv* kv) {
  if (a == nullptr || a->struct_size != sizeof(ifa4_block_select)) return IFA4_EINVAL;
  if (kv == nullptr || kv->struct_size != sizeof(ifa4_paged_kv)) return IFA4_EINVAL;
  if (a->n_heads < 1 || a->kv_heads < 1 || a->n_heads % a->kv_heads != 0 || a->head_dim < 1 ||
      a->max_seqlen_q < 0 || a->max_seqlen_k < 0 || a->total_q < 0)
    return IFA4_EINVAL;
  if (a->n_select < 1 || a->sink_blocks < 0 || a->recent_blocks < 1 ||
      (int64_t)a->sink_blocks + a->recent_blocks > a->n_select)
    return IFA4_EINVAL;
  if ((a->dtype != IFA4_BF16 && a->dtype != IFA4_FP16) ||
      (a->kv_dtype != a->dtype && a->kv_dtype != IFA4_FP8_E4M3))
    return IFA4_EUNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return IFA4_EUNSUPPORTED;
  int32_t st = check_table(kv, a->cu_seqlens, a->batch);
  if (st != IFA4_OK || a->total_q == 0) return st;
  if (a->blocks == nullptr || !aligned(a->blocks, 4)) return IFA4_EINVAL;
  // a workgroup for each list, of at most 2^32 threads in all
  if (a->total_q * a->kv_heads >= kMostGroups) return IFA4_EUNSUPPORTED;
  if (a->batch == 0) return IFA4_OK;
  if ((int64_t)kv->max_blocks_per_seq * kv->block_size < a->max_seqlen_k) return IFA4_EINVAL;
  if (a->q == nullptr || a->q_stride_t < 0 || a->q_stride_h < 0) return IFA4_EINVAL;
  if (!aligned(a->q, 16) || ((a->total_q > 1 ? a->q_stride_t : 0) | (a->n_heads > 1 ? a->q_stride_h : 0)) % 8 != 0)
    return IFA4_EUNSUPPORTED;
  // workgroups that score: a few tokens against 256 blocks each, 16 tokens against any number
  const int64_t q_tiles = ((int64_t)a->max_seqlen_q + 15) / 16;
  const int64_t spans = (int64_t)a->max_seqlen_k / kv->block_size / 256 + 2;
  if (q_tiles * a->kv_heads > (int64_t(1) << 20) || spans * a->kv_heads * 3 >= kMostGroups)
    return IFA4_EUNSUPPORTED;
  return check_bounds(a->bounds, a->bounds_stride_block, a->bounds_stride_h, kv, a->kv_heads,
                      a->head_dim, a->kv_dtype == IFA4_FP8_E4M3 ? 1 : 2, false);
}

// Blocks of the longest sequence; 0 where no sequence has a token.
int32_t select_cols(const ifa4_block_select* a, const ifa4_paged_kv* kv) {
  if (a->batch == 0 || a->max_seqlen_q == 0) return 0;
  return (int32_t)(((int64_t)a->max_seqlen_k + kv->block_size - 1) / kv->block_size);
}

// Scores of all tokens, where a list can leave a block out.
size_t select_bytes(const ifa4_block_select* a, const ifa4_paged_kv* kv) {
  const int64_t cols = select_cols(a, kv);
  if (a->total_q == 0 || cols <= a->n_select) return 0;
  return (size_t)((a->total_q * a->kv_heads * cols * 8 + 255) / 256 * 256);
}

int32_t status_of(hipError_t e) { return e == hipSuccess ? IFA4_OK : IFA4_ELAUNCH; }

}  // namespace

extern "C" {

int32_t ifa4_key_bounds_paged(const ifa4_key_bounds* a, const ifa4_paged_kv* kv, void* stream) {
  const int32_t st = check_key_bounds(a, kv);
  if (st != IFA4_OK || a->batch == 0 || a->max_seqlen_q == 0) return st;
  ifa4::KeyBoundsParams p{};
  p.k = a->k_cache;
  p.bounds = a->bounds;
  p.cu_q = a->cu_seqlens;
  p.seqused_k = kv->seqused_k;
  p.block_table = kv->block_table;
  p.k_st = a->k_stride_t;
  p.k_sh = a->k_stride_h;
  p.k_sblk = kv->k_stride_block;
  p.b_sh = a->bounds_stride_h;
  p.b_sblk = a->bounds_stride_block;
  p.bt_stride = kv->block_table_stride;
  p.batch = a->batch;
  p.kv_heads = a->kv_heads;
  p.block_shift = __builtin_ctz((unsigned)kv->block_size);
  p.num_blocks = kv->num_blocks;
  p.max_blocks = kv->max_blocks_per_seq;
  // n keys in a row meet at most this many blocks
  const int64_t slots = ((int64_t)a->max_seqlen_q + kv->block_size - 2) / kv->block_size + 1;
  p.slots = (int32_t)(slots < p.max_blocks ? slots : p.max_blocks);
  if ((int64_t)p.slots * a->kv_heads >= kMostGroups) return IFA4_EUNSUPPORTED;
  return status_of(ifa4::launch_key_bounds(p, a->head_dim, a->kv_dtype, a->kv_dtype == IFA4_FP8_E4M3,
                                           static_cast<hipStream_t>(stream)));
}

size_t ifa4_select_blocks_workspace_bytes(const ifa4_block_select* a, const ifa4_paged_kv* kv) {
  return check_select(a, kv) == IFA4_OK ? select_bytes(a, kv) : 0;
}

int32_t ifa4_select_blocks_paged(const ifa4_block_select* a, const ifa4_paged_kv* kv,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  const int32_t st = check_select(a, kv);
  if (st != IFA4_OK || a->total_q == 0) return st;
  const size_t need = select_bytes(a, kv);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
    return IFA4_EWORKSPACE;
  ifa4::SelectParams p{};
  p.q = a->q;
  p.bounds = a->bounds;
  p.cu_q = a->cu_seqlens;
  p.seqused_k = kv->seqused_k;
  p.block_table = kv->block_table;
  p.out = a->blocks;
  p.scores = need > 0 ? static_cast<uint64_t*>(workspace) : nullptr;
  p.q_st = a->q_stride_t;
  p.q_sh = a->q_stride_h;
  p.b_sh = a->bounds_stride_h;
  p.b_sblk = a->bounds_stride_block;
  p.bt_stride = kv->block_table_stride;
  p.total_q = (int32_t)a->total_q;
  p.max_q = a->max_seqlen_q;
  p.batch = a->batch;
  p.kv_heads = a->kv_heads;
  p.group = a->n_heads / a->kv_heads;
  p.block_shift = __builtin_ctz((unsigned)kv->block_size);
  p.num_blocks = kv->num_blocks;
  p.max_blocks = kv->max_blocks_per_seq;
  p.cols = select_cols(a, kv);
  p.n_select = a->n_select;
  p.sink = a->sink_blocks;
  p.recent = a->recent_blocks;
  return status_of(ifa4::launch_select_blocks(p, a->head_dim, a->dtype, a->kv_dtype == IFA4_FP8_E4M3,
                                              static_cast<hipStream_t>(stream)));
}

}  // extern "C"
