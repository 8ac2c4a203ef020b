// Internal interface between the C ABI layer (ifa4_api.cpp) and the HIP
// kernels.  Not installed; the public interface is include/ifa4.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "workgroup_order.h"

struct ifa4_args;

namespace ifa4 {

struct PrefillParams {
  const void* q;
  const void* k;
  const void* v;
  const void* rel;
  void* out;
  float* lse;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, rel_st, rel_sh, o_st, o_sh, lse_sh;
  int32_t total_q;      // rows of q / out (cu_seqlens_q is clamped to it)
  int32_t total_k;      // rows of k / v (cu_seqlens_k is clamped to it)
  int32_t batch;
  int32_t n_heads;
  int32_t group;        // n_heads / kv_heads
  int32_t rel_extent;
  int32_t rel_width;    // last dim of rel (>= rel_extent)
  int32_t window_left;  // -1: none
  int32_t causal;
  int32_t bottom_right; // 1: query i sits at key position i + (lk - lq) (IFA4_FLAG_BOTTOM_RIGHT)
  int32_t no_prune;
  int32_t rel_dtype;    // 0 bf16, 1 fp16, 2 fp32
  int32_t n_qtiles;     // ceil(max_seqlen_q / block_q)
  int32_t ragged;       // rows a sixteenth (1) or a quarter (2) below batch * longest, or 0
  WorkgroupOrder order; // set by launch_prefill
  float scale_log2;     // softmax_scale * log2(e)
  // Split KV (chunk_tiles > 0): each q tile's KV tile range is cut into chunks
  // of chunk_tiles tiles, one workgroup each (n_chunks chunk slots per q tile in
  // the grid); a tile with more than one chunk writes normalised partials
  // part_o [n_chunks][n_heads][total_q][head_dim] fp32 and their LSE (log2
  // units) part_lse [n_chunks][n_heads][total_q], merged by a second pass.
  int32_t chunk_tiles;
  int32_t n_chunks;
  int32_t seen_chunks;  // slots that pruned query tiles can use (the merge's form)
  // A query tile is q_step queries x `pack` query heads of one kv head (packed
  // rows, pack > 1: row r of the tile is query (r * pack_magic) >> 16); tile_heads
  // = n_heads / pack tiles side by side, tile_group of them per kv head.
  int32_t pack, q_step, pack_magic, tile_heads, tile_group;
  int32_t max_q;        // max_seqlen_q
  float* part_o;
  float* part_lse;
  // Fused relative-logit projection (wt != nullptr): rel / rel_st / rel_sh /
  // rel_dtype describe r [Tq, Hq, 16]; wt is W^T [rel_width, 16] fp32, rows
  // contiguous; bias(i, dist) = sum_c r[i, c] * wt[dist, c].
  const float* wt;
  // Paged KV cache (block_table != nullptr): k/v are block pools, as in DecodeParams; k_st,
  // k_sh, k_sblk (and v's) count elements of the cache's type.
  const int32_t* block_table;
  const int32_t* seqused_k;
  int64_t bt_stride, k_sblk, v_sblk;
  int32_t block_shift, num_blocks, max_blocks;
  float v_scale;  // of an e4m3 cache: multiplies the output (the K scale is in scale_log2)
};

struct DecodeParams {
  const void* q;
  const void* k;
  const void* v;
  const void* rel;
  void* out;
  float* lse;
  const int32_t* cu_q;
  const int32_t* cu_k;
  float* ws_o;        // [batch * kv_heads + n_waves][group][head_dim] partials
  float* ws_lse;      // [batch * kv_heads + n_waves][group] (log2 domain)
  int32_t* ws_meta;   // [batch * kv_heads][2]: first and last wave of a segment
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, rel_st, rel_sh, o_st, o_sh, lse_sh;
  int32_t total_q;   // rows of q / out (cu_seqlens_q is clamped to it)
  int32_t total_k;   // rows of k / v (cu_seqlens_k is clamped to it; unused when paged)
  int32_t batch;
  int32_t n_heads;
  int32_t kv_heads;
  int32_t group;
  int32_t rel_extent;
  int32_t causal;
  int32_t bottom_right;  // see PrefillParams
  int32_t window_left;   // -1: none (only matters with bottom_right: top-left decode never masks)
  int32_t rel_dtype;
  int32_t n_waves;   // persistent waves of pass 1 (0: nothing to stream)
  int32_t whole;     // 1: one launch, a workgroup per (sequence, kv head); no workspace
  int32_t kv_fp8;    // 1: K and V are fp8 (OCP e4m3), K scale folded into scale_log2
  // 1: each kv head of these params is a pair of adjacent fp8 kv heads (k_sh,
  // v_sh = 2 * head_dim, group = both heads' query heads), streamed as whole rows
  int32_t kv_pair;
  float scale_log2;
  float v_scale;     // multiplies the output (1 for 16-bit V)
  // Paged KV cache (block_table != nullptr): k/v are block pools, key j of
  // sequence b is row j & (2^block_shift - 1) of block
  // block_table[b * bt_stride + (j >> block_shift)]; lengths from seqused_k.
  const int32_t* block_table;
  const int32_t* seqused_k;
  int64_t bt_stride, k_sblk, v_sblk;
  int32_t block_shift;
  int32_t num_blocks;
  int32_t max_blocks;  // table entries per sequence
};

// Head norm and rotation (norm_rope.hip).  q and k rows in, q_out and k_out rows out.
struct NormRopeParams {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  const void* q_weight;      // [head_dim] or NULL: not normed
  const void* k_weight;
  const float* cos;          // [max_position, rot / 2], rows angle_stride apart
  const float* sin;
  const int32_t* positions;  // [total] (rot > 0; a cache append has its own)
  int64_t angle_stride;
  int64_t total;             // tokens
  int64_t first_token;       // of this launch (set by the launch)
  int32_t n_heads, kv_heads;
  int32_t w_dtype;           // 0 bf16, 1 fp16, 2 fp32
  int32_t rot;               // leading elements of a head that turn
  int32_t pairs;             // 1: neighbours turn together, 0: elements rot / 2 apart
  int32_t max_position;
  int32_t heads_per;         // heads of a token that one lane group walks over (set by the launch)
  float eps;
};

// Where the keys and values of new tokens go (paged cache, as in DecodeParams).
struct AppendParams {
  const void* v;
  void* k_cache;
  void* v_cache;
  const int32_t* cu;         // [batch + 1] new tokens of each sequence
  const int32_t* seqused_k;  // keys of each sequence, the new ones included
  const int32_t* block_table;
  int64_t v_st, v_sh, kc_st, kc_sh, kc_sblk, vc_st, vc_sh, vc_sblk, bt_stride;
  int32_t batch, block_shift, num_blocks, max_blocks;
  float k_scale, v_scale, inv_k_scale, inv_v_scale;
};

// Gradients of the norm and rotation; gq or gk NULL: that output has none.
struct NormRopeGrad {
  const void* gq;
  const void* gk;
  void* dq;
  void* dk;
  int64_t gq_st, gq_sh, gk_st, gk_sh, dq_st, dq_sh, dk_st, dk_sh;
  void* dq_weight;
  void* dk_weight;
  float* partial;  // [workgroups of the backward pass][2][head_dim], or NULL without weights
};

// n / d for 32-bit n by a multiplication: magic = floor(2^32 / d) gives the quotient or one less.
struct FastDiv {
  uint32_t magic, d;
  static FastDiv of(int64_t d) {
    const uint64_t m = (uint64_t(1) << 32) / (uint64_t)d;
    return FastDiv{m > 0xffffffffu ? 0xffffffffu : (uint32_t)m, (uint32_t)d};
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    const uint32_t q = (uint32_t)(((uint64_t)n * magic) >> 32);
    return q + (n - q * d >= d ? 1u : 0u);
  }
};

// Paged decode behind a prefix that the whole batch shares (decode_shared.hip).
struct SharedParams {
  const void* q;
  const void* k;
  const void* v;
  const void* rel;
  void* out;
  float* lse;
  const int32_t* cu_q;
  const int32_t* seqused_k;
  const int32_t* block_table;
  const int32_t* prefix_table;
  float* part_o;    // [prefix_chunks + own_chunks][batch][n_heads][head_dim]
  float2* part_ml;  // [prefix_chunks + own_chunks][batch][n_heads]: maximum (natural units), sum
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, rel_st, rel_sh, o_st, o_sh, lse_sh;
  int64_t k_sblk, v_sblk, bt_stride;
  int64_t rel_span;        // elements of the bias, first to last
  int32_t total_q, batch, n_heads, kv_heads, group;
  int32_t rel_extent, rel_dtype, window_left;
  int32_t block_shift, num_blocks, max_blocks;
  int32_t prefix_entries;  // of prefix_table that may be read
  int32_t prefix_keys;     // keys of the prefix that are computed once for all, whole tiles
  int32_t chunk_keys;      // of a prefix workgroup
  int32_t prefix_chunks;
  int32_t row_tiles;       // prefix workgroups side by side over batch * group rows
  int32_t prefix_blocks;   // workgroups of the prefix, all XCDs' shares alike
  int32_t own_chunks;      // pieces of a (sequence, kv head)'s own keys
  int32_t own_first;       // of them for a workgroup without a prefix piece, ahead of the others
  int32_t own_pieces;      // batch * kv_heads * own_chunks
  int32_t kv_fp8;
  FastDiv by_tiles, by_kv, by_batch, by_group, by_heads, by_chunk;  // divisions by row_tiles,
                           // kv_heads, batch, group, n_heads, chunk_keys
  float scale;             // softmax_scale (times the K scale of an e4m3 cache)
  float v_scale;
};
constexpr int kSharedTile = 64, kSharedRows = 128, kSharedOwnRound = 128;
constexpr int kSharedSlots = 512;  // resident workgroups, two a CU
hipError_t launch_decode_shared(const SharedParams& p, int head_dim, int qkv_dtype,
                                hipStream_t stream);

// Bounds of the keys of a paged cache's blocks (block_select.hip).
struct KeyBoundsParams {
  const void* k;
  void* bounds;              // [blocks][kv_heads][2][head_dim], of the cache's type
  const int32_t* cu_q;
  const int32_t* seqused_k;
  const int32_t* block_table;
  int64_t k_st, k_sh, k_sblk, b_sh, b_sblk, bt_stride;
  int32_t batch, kv_heads, block_shift, num_blocks, max_blocks;
  int32_t slots;             // blocks of a sequence that new tokens can have changed
};
hipError_t launch_key_bounds(const KeyBoundsParams& p, int head_dim, int dtype, bool fp8,
                             hipStream_t stream);

// The blocks that each token and kv head reads, by those bounds.
struct SelectParams {
  const void* q;
  const void* bounds;
  const int32_t* cu_q;
  const int32_t* seqused_k;
  const int32_t* block_table;
  int32_t* out;              // [total_q][kv_heads][n_select]
  uint64_t* scores;          // [total_q][kv_heads][cols] keys of the scores
  int64_t q_st, q_sh, b_sh, b_sblk, bt_stride;
  int32_t total_q, max_q, batch, kv_heads, group, block_shift, num_blocks, max_blocks;
  int32_t cols;              // blocks of the longest sequence
  int32_t n_select, sink, recent;
  int32_t score_parts;       // workgroups that share the blocks of 16 tokens (set by the launch)
};
hipError_t launch_select_blocks(const SelectParams& p, int head_dim, int dtype, bool fp8,
                                hipStream_t stream);

// Attention of each token and kv head over the blocks its list names (sparse_fwd.hip).
struct SparseParams {
  const void* q;
  const void* k;
  const void* v;
  const void* rel;
  void* out;
  float* lse;
  const int32_t* cu_q;
  const int32_t* seqused_k;
  const int32_t* block_table;
  const int32_t* blocks;     // lists, ls_st elements between tokens, ls_sh between kv heads
  float* part_o;             // [splits][total_q][n_heads][head_dim], splits > 1
  float2* part_ml;           // [splits][total_q][n_heads]: maximum (log2 units), sum
  int64_t q_st, q_sh, k_st, k_sh, k_sblk, v_st, v_sh, v_sblk, rel_st, rel_sh, o_st, o_sh, lse_sh;
  int64_t bt_stride, ls_st, ls_sh;
  int32_t total_q, batch, n_heads, kv_heads, group;
  int32_t rel_extent, rel_dtype, window_left;
  int32_t block_shift, num_blocks, max_blocks;
  int32_t n_select;
  int32_t waves, splits;     // waves of a workgroup, workgroups that share a list
  int32_t steps;             // of a list
  int32_t once;              // one token a sequence at most: rows are read once
  int32_t groups, per_xcd;   // workgroups, those of an XCD
  FastDiv by_splits, by_total;  // divisions by splits, total_q
  int32_t kv_fp8;
  float scale_log2;          // with the K scale of an e4m3 cache
  float v_scale;
};
constexpr int kSparseStep = 32;
// Waves that share a list of `rows` rows, for `items` (token, kv head) pairs: enough of them in all
// to fill the chip, each with two steps at least; up to 8 in a workgroup, the rest as workgroups
// whose partials a second pass joins.  A call in us with 2048 / 4096 waves: 64 sequences x 128 blocks
// of 16 30.4 / 34.1, of e4m3 21.1 / 23.6, 512 tokens x 128 blocks 55.1 / 57.6, x 100 blocks of e4m3
// 38.8 / 37.7, 4 sequences x 16 blocks of 64 9.9 / 9.8.
constexpr int kSparseWaves = 2048;
// A workgroup takes in about 53 KB a us, the second pass takes 3.5 us: shares pay where they take more
// than this many bytes of K and V off a workgroup.  A call in us, one workgroup a list / shares:
// lists of 256 KiB (16 blocks of 64, d 64; 4 sequences, 2 shares) 9.3 / 11.9, of 512 KiB (128 of 16, e4m3;
// 4 sequences, 4 shares) 15.6 / 13.0, of 1 MiB (the same, bf16) 24.8 / 15.6.
constexpr int64_t kSparseSplitBytes = 192 << 10;
struct SparsePlan {
  int32_t waves, splits;
};
inline SparsePlan sparse_plan(int64_t items, int64_t rows, int64_t row_bytes) {
  const int64_t steps = (rows + kSparseStep - 1) / kSparseStep;
  int64_t want = items > 0 ? (kSparseWaves + items - 1) / items : 1;
  if (want > steps / 2) want = steps / 2;
  SparsePlan pl{1, 1};
  while (pl.waves < 8 && 2 * pl.waves <= want) pl.waves *= 2;
  int64_t s = want / pl.waves;
  if (s > 1 && rows * row_bytes / s * (s - 1) <= kSparseSplitBytes) s = 1;
  pl.splits = (int32_t)(s < 1 ? 1 : s);
  return pl;
}
hipError_t launch_sparse(const SparseParams& p, int head_dim, int qkv_dtype, hipStream_t stream);

// Workgroups of the backward pass, over tokens (x) and chunks of heads_per heads (y), each with a
// row of partial weight gradients.
struct NormRopeBwdGrid {
  unsigned x, y;
  int heads_per;
};
NormRopeBwdGrid norm_rope_bwd_grid(int64_t total, int heads, int head_dim);
// cache: 0 none, 1 of the inputs' type, 2 e4m3
hipError_t launch_norm_rope(const NormRopeParams& p, const AppendParams& a, int cache, int head_dim,
                            int dtype, hipStream_t stream);
hipError_t launch_norm_rope_bwd(const NormRopeParams& p, const NormRopeGrad& g, int head_dim,
                                int dtype, hipStream_t stream);

int prefill_block_q();
int prefill_proj_block_q();  // query rows per workgroup of the fused-projection kernel
int prefill_block_k();
bool prefill_tab(const PrefillParams& p);  // the shared bias table is staged in LDS
bool prefill_tab_packs(int rel_extent, int pack);  // ... and holds the tables of `pack` heads
int prefill_waves();
hipError_t launch_prefill(const PrefillParams& p, int head_dim, int qkv_dtype, hipStream_t stream);
hipError_t launch_prefill_paged(const PrefillParams& p, int head_dim, int qkv_dtype,
                                hipStream_t stream);
hipError_t launch_prefill_paged_fp8(const PrefillParams& p, int head_dim, int qkv_dtype,
                                    hipStream_t stream);

int decode_max_group();
int decode_fp8_max_group();
hipError_t launch_decode(const DecodeParams& p, int head_dim, int qkv_dtype, hipStream_t stream);

// Common body of the contiguous 16-bit decode entry points (ifa4_api.cpp): the
// host checks with the workspace bytes the call needs, and the call itself on
// a caller-provided workspace.
int32_t decode_workspace_need(const ifa4_args* args, size_t* bytes);
int32_t decode_run(const ifa4_args* args, void* workspace, size_t workspace_bytes, void* stream);

}  // namespace ifa4
