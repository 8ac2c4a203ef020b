// Which blocks of a paged cache a token's attention reads, for gfx950 (MI355X): bounds of the
// keys of every block, scores of the blocks by them, and the choice.  The reference has none.
//
//   lo, hi[blk, h, d] = least and greatest key element of the block's rows (the type holds them
//     exactly; NaN where a key is NaN)
//   score[t, h, b] = sum over the query heads g of kv head h and d of max(q_gd lo_d, q_gd hi_d)
//                  = sum_d qn_d lo_d + qp_d hi_d,  qn = sum_g min(q_g, 0), qp = sum_g max(q_g, 0):
//     no key of the block has a greater sum of its group's dot products.  (An infinite bound meets
//     a qn or qp of 0 as NaN: the block counts as the best, which it may be.)
//   list[t, h] = the first `sink` blocks, the last `recent` ones up to the token's own, and the
//     best by score of those between (a score of NaN as infinity, equal ones the lower block
//     first), ascending; all blocks where there are no more than the list holds.
//
// The choice is whole numbers, so it should not hang on the order of a sum: scores are summed in
// 64 bits, where the products are exact to 2^-53 (in 32 bits about one list in a few hundred of
// 2000 blocks changed with the summation order).  The chip multiplies 64-bit floats at 74 TFLOP/s
// on the matrix cores and converts and adds 17e12 elements a second on the vector unit, so a
// decode step is bound by the bounds' bytes all the same.
#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

typedef double f64x4_t __attribute__((ext_vector_type(4)));

// Elements of a cache: 16 bytes of them as fp32.
template <typename Tag, int Eb>
__device__ __forceinline__ void unpack16(u32x4_t w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Eb == 2) {
      f[2 * i] = Elem<Tag>::lo(w[i]);
      f[2 * i + 1] = Elem<Tag>::hi(w[i]);
    } else {
      typedef float f32x2_t __attribute__((ext_vector_type(2)));
      const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
      const f32x2_t b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      f[4 * i] = a[0];
      f[4 * i + 1] = a[1];
      f[4 * i + 2] = b[0];
      f[4 * i + 3] = b[1];
    }
  }
}
template <typename Tag, int Eb>
__device__ __forceinline__ u32x4_t pack16(const float* f) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Eb == 2) {
      w[i] = Elem<Tag>::pack2(f[2 * i], f[2 * i + 1]);
    } else {  // exact: the values are e4m3 values
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], x, true);
    }
  }
  return w;
}

__device__ __forceinline__ float lower(float x, float m) { return x < m || x != x ? x : m; }
__device__ __forceinline__ float higher(float x, float m) { return x > m || x != x ? x : m; }

// ---- bounds ----------------------------------------------------------------------------------
// A wave takes one (block, kv head) whose rows new tokens changed: D * Eb / 16 lanes a row, as
// many rows at a time as fit, then the row groups meet by lane exchange.  Blocks of 64 rows and
// more: the four waves of the workgroup share one.
constexpr int kBoundWaves = 4;
template <int D, typename Tag, int Eb>
__global__ __launch_bounds__(64 * kBoundWaves) void key_bounds_kernel(KeyBoundsParams p) {
  constexpr int kLpr = D * Eb / 16, kRpi = 64 / kLpr, kEpl = 16 / Eb;
  __shared__ float part[kBoundWaves][2][D];
  const int seq = blockIdx.y;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int bs = 1 << p.block_shift;
  const int team = bs >= 64 ? kBoundWaves : 1;  // waves a block
  const int item = (int)blockIdx.x * (kBoundWaves / team) + (team > 1 ? 0 : wave);
  const int slot = item / p.kv_heads, h = item - slot * p.kv_heads;
  const int64_t cap = (int64_t)p.max_blocks << p.block_shift;
  const int64_t used = min(max((int64_t)p.seqused_k[seq], (int64_t)0), cap);
  const int64_t n = min(max((int64_t)p.cu_q[seq + 1] - p.cu_q[seq], (int64_t)0), used);
  const int64_t blk = ((used - n) >> p.block_shift) + slot;
  const bool on = n > 0 && slot < p.slots && (blk << p.block_shift) < used;  // team: uniform
  const int ent = on ? p.block_table[seq * p.bt_stride + blk] : -1;
  const bool good = (uint32_t)ent < (uint32_t)p.num_blocks;
  if (team == 1 && !good) return;
  const int rows = good ? (int)min(used - (blk << p.block_shift), (int64_t)bs) : 0;
  const int r = lane / kLpr, c = lane % kLpr;
  const char* const base = static_cast<const char*>(p.k) +
                           ((int64_t)(good ? ent : 0) * p.k_sblk + (int64_t)h * p.k_sh) * Eb + 16 * c;
  float lo[kEpl], hi[kEpl];
#pragma unroll
  for (int e = 0; e < kEpl; ++e) {
    lo[e] = INFINITY;
    hi[e] = -INFINITY;
  }
  const int first = team > 1 ? wave * kRpi : 0, step = team * kRpi;
#pragma unroll 4
  for (int row = first + r; row < rows; row += step) {
    float f[kEpl];
    unpack16<Tag, Eb>(ld_global_16(base + (int64_t)row * p.k_st * Eb), f);
#pragma unroll
    for (int e = 0; e < kEpl; ++e) {
      lo[e] = lower(f[e], lo[e]);
      hi[e] = higher(f[e], hi[e]);
    }
  }
#pragma unroll
  for (int off = kLpr; off < 64; off <<= 1) {
#pragma unroll
    for (int e = 0; e < kEpl; ++e) {
      lo[e] = lower(__shfl_xor(lo[e], off), lo[e]);
      hi[e] = higher(__shfl_xor(hi[e], off), hi[e]);
    }
  }
  if (team > 1) {
    if (r == 0) {
#pragma unroll
      for (int e = 0; e < kEpl; ++e) {
        part[wave][0][kEpl * c + e] = lo[e];
        part[wave][1][kEpl * c + e] = hi[e];
      }
    }
    __syncthreads();
    if (wave != 0 || !good) return;
#pragma unroll
    for (int w = 1; w < kBoundWaves; ++w) {
#pragma unroll
      for (int e = 0; e < kEpl; ++e) {
        lo[e] = lower(part[w][0][kEpl * c + e], lo[e]);
        hi[e] = higher(part[w][1][kEpl * c + e], hi[e]);
      }
    }
  }
  if (r > 1) return;
  char* const dst = static_cast<char*>(p.bounds) +
                    ((int64_t)ent * p.b_sblk + (int64_t)h * p.b_sh) * Eb + 16 * c;
  // row group 0 writes the lower bounds, row group 1 the upper (a wave holds two rows at least)
  *reinterpret_cast<u32x4_t*>(dst + r * D * Eb) = pack16<Tag, Eb>(r == 0 ? lo : hi);
}

// ---- scores ----------------------------------------------------------------------------------
// Keys that order as the scores do: greater score, greater key; NaN as the greatest of all with
// infinity's key (+0 and -0 alike).
__device__ __forceinline__ uint64_t score_key(double x) {
  x = x != x ? (double)INFINITY : x + 0.0;
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return b >> 63 ? ~b : b | (uint64_t(1) << 63);
}

// Blocks that token t of sequence seq may read: those up to its own.
struct TokenSpan {
  int start, len;  // tokens of the sequence
  int past;        // keys before its first token
};
__device__ __forceinline__ TokenSpan token_span(const SelectParams& p, int seq) {
  const SeqBounds b = seq_bounds(p.cu_q, seq, p.total_q);
  const int lk = min(max(p.seqused_k[seq], 0), p.max_blocks << p.block_shift);
  return TokenSpan{b.start, b.len, lk - b.len};
}
__device__ __forceinline__ int token_blocks(const SelectParams& p, const TokenSpan& s, int i) {
  const int pos = s.past + i;
  return pos < 0 ? 0 : min((pos >> p.block_shift) + 1, p.cols);
}

// 16 tokens of a sequence against 16 blocks a step, on v_mfma_f64_16x16x4: A = bounds (lane l:
// block l % 16, elements of the chunks l / 16 modulo 4), B = qn, qp of the same elements (token
// l % 16), held in registers over the blocks; C (lane l, register r) = block 4 r + l / 16, token
// l % 16.
constexpr int kScoreWaves = 4;
constexpr int kHeadsAtOnce = 4;  // query heads whose loads are in flight together
// Workgroups of the tile kernel in all: one resident round (512 tokens over 1900 blocks of e4m3, us a
// call with 256 / 512 / 768 / 1024: 43.5 / 41.6 / 47.3 / 44.7).
constexpr int kScoreGroups = 512;
// Tokens of a sequence up to which the vector unit takes them one by one (16 sequences over 1900
// blocks, vector / matrix: 2 tokens 20.6 / 26.3, 4 tokens 27.1 / 26.8).
constexpr int kStepTokens = 3;
template <int D, typename Tag, int Eb>
__global__ __launch_bounds__(64 * kScoreWaves) void score_tile_kernel(SelectParams p) {
  constexpr int kEpc = 16 / Eb;                // elements of a 16-byte chunk
  constexpr int kChunks = 2 * D / kEpc / 4;    // chunks a lane holds of a block's bounds
  const int seq = blockIdx.y;
  const int part0 = blockIdx.x % p.score_parts, rest = blockIdx.x / p.score_parts;
  const int h = rest % p.kv_heads, i0 = rest / p.kv_heads * 16;
  const TokenSpan s = token_span(p, seq);
  if (i0 >= s.len) return;
  const int most = token_blocks(p, s, min(i0 + 16, s.len) - 1);  // of the tile's last token
  const int lane = threadIdx.x & 63, wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, g = lane >> 4;
  // a list that takes every block needs no scores; nor do the sink and recent blocks
  if (most <= p.n_select) return;
  const int last = most - p.recent;  // blocks [sink, last) compete for the tile's last token
  int tile = (p.sink >> 4) + part0 * kScoreWaves + wave;
  if ((tile - wave) * 16 >= last) return;

  // qn and qp of the 16 tokens, summed over the heads by the four waves together (8 elements of
  // a lane each, in units of 8)
  constexpr int kUnits = D / 32;
  __shared__ __align__(16) double q_lds[2 * kUnits][64][8];
  const int64_t tok = s.start + min(i0 + m, s.len - 1);
  const char* const q_row = static_cast<const char*>(p.q) +
                            (tok * p.q_st + (int64_t)h * p.group * p.q_sh) * 2;
  const int32_t* const table = p.block_table + seq * p.bt_stride;
  auto load = [&](int t, u32x4_t* w) {
    const int blk = min(16 * t + m, most - 1);
    const int ent = table[blk];
    const bool good = (uint32_t)ent < (uint32_t)p.num_blocks;
    const char* src = static_cast<const char*>(p.bounds) +
                      ((int64_t)(good ? ent : 0) * p.b_sblk + (int64_t)h * p.b_sh) * Eb + 16 * g;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      w[i] = ld_global_16(src + 64 * i);
      if (!good) w[i] = u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  u32x4_t w[kChunks], next[kChunks];
  load(tile, w);  // (a tile past the last is read as the last block)
  if (wave < kUnits) {
    const int d = kEpc * (4 * (wave / (kEpc / 8)) + g) + 8 * (wave % (kEpc / 8));
    double neg[8], up[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) neg[e] = up[e] = 0.0;
    for (int head = 0; head < p.group; head += kHeadsAtOnce) {
      u32x4_t x[kHeadsAtOnce];
#pragma unroll
      for (int i = 0; i < kHeadsAtOnce; ++i)
        x[i] = ld_global_16(q_row + (min(head + i, p.group - 1) * p.q_sh + d) * 2);
#pragma unroll
      for (int i = 0; i < kHeadsAtOnce; ++i) {
        if (head + i < p.group) {
          float f[8];
          unpack16<Tag, 2>(x[i], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            neg[e] += (double)(f[e] > 0.f ? 0.f : f[e]);  // a NaN in both
            up[e] += (double)(f[e] < 0.f ? 0.f : f[e]);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q_lds[wave][lane][e] = neg[e];
      q_lds[kUnits + wave][lane][e] = up[e];
    }
  }
  __syncthreads();
  if (tile * 16 >= last) return;
  double q[kChunks][kEpc];
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int e = 0; e < kEpc; ++e) q[i][e] = q_lds[i * (kEpc / 8) + e / 8][lane][e % 8];

  const int step = p.score_parts * kScoreWaves;
  for (; tile * 16 < last; tile += step) {
    if ((tile + step) * 16 < last) load(tile + step, next);
    f64x4_t acc = {0.0, 0.0, 0.0, 0.0}, acc1 = acc;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float f[kEpc];
      unpack16<Tag, Eb>(w[i], f);
#pragma unroll
      for (int e = 0; e < kEpc; e += 2) {
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f[e], q[i][e], acc, 0, 0, 0);
        acc1 = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f[e + 1], q[i][e + 1], acc1, 0, 0, 0);
      }
    }
    acc += acc1;
    if (i0 + m < s.len) {
      uint64_t* const dst = p.scores + ((tok * p.kv_heads + h) * (int64_t)p.cols + 16 * tile + g);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * tile + g + 4 * r < p.cols) dst[4 * r] = score_key(acc[r]);
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) w[i] = next[i];
  }
}

// One token of a sequence against its blocks, on the vector unit: a lane group of 8 takes a block
// (lane `sub`: the chunks sub modulo 8), qn and qp of a lane's elements stay in registers, a wave
// walks over 64 blocks (one load of their table entries), the next 8 blocks' bounds in flight
// while 8 are summed (24 or 32 in flight cost a wave per SIMD: 39 us instead of 30).
constexpr int kStepBlocks = 64;  // of a wave
template <int Ctrl>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)b, Ctrl, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(b >> 32), Ctrl, 0xf, 0xf, true);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int D, typename Tag, int Eb>
__global__ __launch_bounds__(64 * kScoreWaves) void score_step_kernel(SelectParams p) {
  constexpr int kEpc = 16 / Eb;              // elements of a 16-byte chunk
  constexpr int kHalf = D / kEpc;            // chunks of lo, and of hi
  constexpr int kChunks = 2 * kHalf / 8;     // of a lane
  const int lane = threadIdx.x & 63, wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seq = blockIdx.y;
  // kv heads side by side: their bounds of a block are neighbours in memory (64 sequences over
  // 2000..32700 keys in blocks of 16, a call: 29.2 -> 27.0 us; over 32000 each 38.9 -> 38.7)
  const int h = blockIdx.x % p.kv_heads, rest = blockIdx.x / p.kv_heads;
  const int part0 = rest % p.score_parts, i0 = rest / p.score_parts;
  const TokenSpan s = token_span(p, seq);
  if (i0 >= s.len) return;
  const int nb = token_blocks(p, s, i0);
  if (nb <= p.n_select) return;
  const int last = nb - p.recent;
  const int first = p.sink + (part0 * kScoreWaves + wave) * kStepBlocks;
  if (first >= last) return;
  const int sub = lane & 7, row = lane >> 3;
  const int ent_mine = p.block_table[seq * p.bt_stride + min(first + lane, nb - 1)];

  const int64_t tok = s.start + i0;
  const char* const q_row = static_cast<const char*>(p.q) +
                            (tok * p.q_st + (int64_t)h * p.group * p.q_sh) * 2;
  double q[kChunks][kEpc];
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int e = 0; e < kEpc; ++e) q[i][e] = 0.0;
  // chunk c: elements d = kEpc (c % kHalf) .., of lo for c < kHalf, else of hi
  for (int head = 0; head < p.group; head += 2) {
    u32x4_t x[2][kChunks][kEpc / 8];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int part = 0; part < kEpc / 8; ++part)
          x[k][i][part] = ld_global_16(
              q_row + (min(head + k, p.group - 1) * p.q_sh +
                       kEpc * ((sub + 8 * i) & (kHalf - 1)) + 8 * part) * 2);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (head + k < p.group) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
          const bool up = sub + 8 * i >= kHalf;
#pragma unroll
          for (int part = 0; part < kEpc / 8; ++part) {
            float f[8];
            unpack16<Tag, 2>(x[k][i][part], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = up ? f[e] : -f[e];
              q[i][8 * part + e] += (double)(y < 0.f ? 0.f : f[e]);  // a NaN in both
            }
          }
        }
      }
    }
  }

  const char* const bounds = static_cast<const char*>(p.bounds) + (int64_t)h * p.b_sh * Eb + 16 * sub;
  auto load = [&](int it, u32x4_t* w) {
    const int ent = __shfl(ent_mine, 8 * it + row);
    const bool good = (uint32_t)ent < (uint32_t)p.num_blocks;
    const char* src = bounds + (int64_t)(good ? ent : 0) * p.b_sblk * Eb;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      w[i] = ld_global_16(src + 128 * i);
      if (!good) w[i] = u32x4_t{0u, 0u, 0u, 0u};
    }
  };
  uint64_t* const dst = p.scores + ((tok * p.kv_heads + h) * (int64_t)p.cols + first);
  auto sum = [&](int it, const u32x4_t* w) {
    double acc[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      float f[kEpc];
      unpack16<Tag, Eb>(w[i], f);
#pragma unroll
      for (int e = 0; e < kEpc; ++e) acc[e & 1] = fma((double)f[e], q[i][e], acc[e & 1]);
    }
    double x = acc[0] + acc[1];
    x = dpp_add<0xb1>(x);   // lane ^ 1
    x = dpp_add<0x4e>(x);   // lane ^ 2
    x = dpp_add<0x141>(x);  // the other four of eight
    if (sub == 0 && first + 8 * it + row < last) dst[8 * it + row] = score_key(x);
  };
  const int its = min(kStepBlocks / 8, (last - first + 7) / 8);
  u32x4_t a[kChunks], b[kChunks];
  load(0, a);
  for (int it = 0; it < its; it += 2) {
    if (it + 1 < its) load(it + 1, b);
    sum(it, a);
    if (it + 1 >= its) break;
    if (it + 2 < its) load(it + 2, a);
    sum(it + 1, b);
  }
}

// ---- choice ----------------------------------------------------------------------------------
// One workgroup per (token, kv head).  The border of the n_free best competing blocks is found by
// halving the keys' range by 1024 at a time, from least to greatest: count the keys of each of
// 1024 equal parts, keep the part that holds the border, until all its keys are taken, they are
// few enough to rank one against another, or they are all equal.  Scores spread over a range, so
// one count mostly leaves a handful.  Then the list in ascending order by a prefix sum over the
// blocks: a thread holds kPer consecutive ones, a workgroup kRound (kOne: they stay in registers
// from pass to pass; longer rows are read again).
constexpr int kPickThreads = 256, kPer = 8, kRound = kPickThreads * kPer, kBins = 1024;
constexpr int kRankMost = 64;
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int off) {
  return (uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), off) << 32 | (uint32_t)__shfl_xor((int)x, off);
}
template <bool kOne>
__global__ __launch_bounds__(kPickThreads) void pick_blocks_kernel(SelectParams p) {
  constexpr int kPickWaves = kPickThreads / 64;
  __shared__ int hist[kBins];
  __shared__ uint64_t ends[2][kPickWaves];
  __shared__ int sums[kPickWaves];
  __shared__ int border[2];
  __shared__ uint64_t few_key[kRankMost];
  __shared__ int few_at[kRankMost];
  __shared__ int few_n;
  __shared__ uint64_t top_key;
  __shared__ int top_equal;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int t = (int)(row / p.kv_heads);
  int32_t* const list = p.out + row * p.n_select;
  const int first = p.sink;  // competing blocks [first, first + n)
  const uint64_t* const keys = p.scores + row * (int64_t)p.cols + first;
  uint64_t mine[kPer];
  auto load = [&](int r0, int end) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = r0 + tid * kPer + i;
      mine[i] = b < end ? keys[b] : 0;
    }
  };
  // before n is known, and with it which of them were written
  if constexpr (kOne) load(0, p.scores != nullptr ? p.cols - first : 0);

  // the token's sequence: the first whose tokens end past it
  int nb = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int b = b0 + lane;
    const uint64_t past = __builtin_amdgcn_ballot_w64(b < p.batch && p.cu_q[min(b, p.batch - 1) + 1] > t);
    if (past != 0) {
      const TokenSpan s = token_span(p, b0 + __builtin_ctzll(past));
      if (t >= s.start && t < s.start + s.len) nb = token_blocks(p, s, t - s.start);
      break;
    }
  }
  if (nb <= p.n_select) {
    for (int i = tid; i < p.n_select; i += kPickThreads) list[i] = i < nb ? i : -1;
    return;
  }
  for (int i = tid; i < p.sink; i += kPickThreads) list[i] = i;
  for (int i = tid; i < p.recent; i += kPickThreads)
    list[p.n_select - p.recent + i] = nb - p.recent + i;
  const int n = nb - p.recent - p.sink;  // > 0
  int need = p.n_select - p.sink - p.recent;
  if (need == 0) return;
  const int rounds = kOne ? 1 : (n + kRound - 1) / kRound;
  // every key of the row, in any order
  auto each = [&](auto&& f) {
    for (int r = 0; r < rounds; ++r) {
      if constexpr (!kOne) load(r * kRound, n);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (r * kRound + tid * kPer + i < n) f(mine[i], r * kRound + tid * kPer + i);
    }
  };

  uint64_t lo = ~uint64_t(0), hi = 0;
  each([&](uint64_t k, int) {
    lo = k < lo ? k : lo;
    hi = k > hi ? k : hi;
  });
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t a = shfl_xor64(lo, off), b = shfl_xor64(hi, off);
    lo = a < lo ? a : lo;
    hi = b > hi ? b : hi;
  }
  if (lane == 0) {
    ends[0][wave] = lo;
    ends[1][wave] = hi;
  }
  if (tid == 0) few_n = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPickWaves; ++w) {
    lo = ends[0][w] < lo ? ends[0][w] : lo;
    hi = ends[1][w] > hi ? ends[1][w] : hi;
  }

  uint64_t top;   // keys above it are taken,
  int equal;      // and so many of those equal to it, the lower blocks
  while (true) {
    if (lo == hi) {
      top = lo;
      equal = need;
      break;
    }
    const int bits = 64 - __builtin_clzll(hi - lo);
    const int shift = bits > 10 ? bits - 10 : 0;
#pragma unroll
    for (int i = 0; i < kBins / kPickThreads; ++i) hist[tid + i * kPickThreads] = 0;
    __syncthreads();
    each([&](uint64_t k, int) {
      if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> shift)], 1);
    });
    __syncthreads();
    // thread t holds the bins kBins - 4 t - 4 .. + 3: counts from the top
    constexpr int kMine = kBins / kPickThreads;
    int c[kMine], total = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      c[i] = hist[kBins - 1 - tid * kMine - i];
      total += c[i];
    }
    int incl = total;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int up = __shfl_up(incl, off);
      if (lane >= off) incl += up;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w)
      if (w < wave) incl += sums[w];
    int above = incl - total;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (above < need && above + c[i] >= need) {
        border[0] = kBins - 1 - tid * kMine - i;
        border[1] = above;
      }
      above += c[i];
    }
    __syncthreads();
    const int bin = border[0];
    const int held = hist[bin];
    need -= border[1];
    lo += (uint64_t)bin << shift;
    const uint64_t span = (uint64_t(1) << shift) - 1;  // lo + span may lie past 64 bits
    hi = hi - lo < span ? hi : lo + span;
    if (held == need) {  // all of them: keys >= lo
      top = lo - 1;      // (lo > 0: some key lies below the border's part, or lo is the least key)
      equal = 0;
      if (lo == 0) {
        top = 0;
        equal = need;
      }
      break;
    }
    if (held <= kRankMost) {
      each([&](uint64_t k, int b) {
        if (k >= lo && k <= hi) {
          const int i = atomicAdd(&few_n, 1);
          few_key[i] = k;
          few_at[i] = b;
        }
      });
      __syncthreads();
      if (wave == 0) {
        const uint64_t k = lane < held ? few_key[lane] : 0;
        const int at = lane < held ? few_at[lane] : 0;
        int rank = 0, same = 0;  // keys before mine, and of them those equal to it
        for (int i = 0; i < held; ++i) {
          const uint64_t o = few_key[i];
          const bool before = o == k && few_at[i] < at;
          same += before;
          rank += before || o > k;
        }
        if (lane < held && rank == need - 1) {
          top_key = k;
          top_equal = same + 1;
        }
      }
      __syncthreads();
      top = top_key;
      equal = top_equal;
      break;
    }
    __syncthreads();  // hist is cleared again
  }

  // the list: blocks with keys above `top`, and the first `equal` of those equal to it
  int at = p.sink, met = 0;  // places filled, keys equal to top met
  for (int r = 0; r < rounds; ++r) {
    if constexpr (!kOne) load(r * kRound, n);
    int a = 0, e = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = r * kRound + tid * kPer + i < n;
      a += in && mine[i] > top;
      e += in && mine[i] == top;
    }
    int incl = a | e << 16;  // at most kRound of either
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int up = __shfl_up(incl, off);
      if (lane >= off) incl += up;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w) {
      if (w < wave) incl += sums[w];
      all += sums[w];
    }
    int ab = (incl & 0xffff) - a, eb = met + (incl >> 16) - e;  // before this thread's
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = r * kRound + tid * kPer + i;
      if (b < n) {
        const bool above = mine[i] > top, same = mine[i] == top;
        if (above || (same && eb < equal))
          list[at + ab + min(eb, equal) - min(met, equal)] = first + b;
        ab += above;
        eb += same;
      }
    }
    at += (all & 0xffff) + min(met + (all >> 16), equal) - min(met, equal);
    met += all >> 16;
  }
}

template <int D, typename Tag, int Eb>
hipError_t launch_select_t(const SelectParams& p_in, hipStream_t stream) {
  SelectParams p = p_in;
  if (p.cols > p.n_select) {
    hipError_t e;
    if (p.max_q <= kStepTokens) {
      p.score_parts = (p.cols + kStepBlocks * kScoreWaves - 1) / (kStepBlocks * kScoreWaves);
      hipLaunchKernelGGL((score_step_kernel<D, Tag, Eb>),
                         dim3((unsigned)((int64_t)p.score_parts * p.max_q * p.kv_heads), p.batch),
                         dim3(64 * kScoreWaves), 0, stream, p);
    } else {
      const int tiles = (p.cols + 15) / 16, q_tiles = (p.max_q + 15) / 16;
      // workgroups for every tile of blocks, or kScoreGroups of them where there are many tokens:
      // each begins with the sums over its query heads.  (Counted by the longest sequence: beside
      // one chunk, single tokens get a workgroup each.  512 tokens over 30000 keys and 63 single
      // ones over 2K..32K 390 us in one call, 44 and 27 in two.)
      const int per = (tiles + kScoreWaves - 1) / kScoreWaves;
      const int64_t others = (int64_t)q_tiles * p.kv_heads * p.batch;
      p.score_parts = (int)max(int64_t(1), min((int64_t)per, kScoreGroups / max(int64_t(1), others)));
      hipLaunchKernelGGL((score_tile_kernel<D, Tag, Eb>),
                         dim3((unsigned)((int64_t)p.score_parts * q_tiles * p.kv_heads), p.batch),
                         dim3(64 * kScoreWaves), 0, stream, p);
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)((int64_t)p.total_q * p.kv_heads));
  if (p.cols <= kRound)
    hipLaunchKernelGGL(pick_blocks_kernel<true>, grid, dim3(kPickThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(pick_blocks_kernel<false>, grid, dim3(kPickThreads), 0, stream, p);
  return hipGetLastError();
}

template <int D, typename Tag>
hipError_t launch_select_d(const SelectParams& p, bool fp8, hipStream_t stream) {
  return fp8 ? launch_select_t<D, Tag, 1>(p, stream) : launch_select_t<D, Tag, 2>(p, stream);
}

template <int D, typename Tag, int Eb>
hipError_t launch_bounds_t(const KeyBoundsParams& p, hipStream_t stream) {
  const int per = (1 << p.block_shift) >= 64 ? 1 : kBoundWaves;
  const int64_t items = (int64_t)p.slots * p.kv_heads;
  hipLaunchKernelGGL((key_bounds_kernel<D, Tag, Eb>), dim3((unsigned)((items + per - 1) / per), p.batch),
                     dim3(64 * kBoundWaves), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_key_bounds(const KeyBoundsParams& p, int head_dim, int dtype, bool fp8,
                             hipStream_t stream) {
  if (fp8)
    return head_dim == 128 ? launch_bounds_t<128, Bf16Tag, 1>(p, stream)
                           : launch_bounds_t<64, Bf16Tag, 1>(p, stream);
  if (head_dim == 128)
    return dtype == 0 ? launch_bounds_t<128, Bf16Tag, 2>(p, stream)
                      : launch_bounds_t<128, F16Tag, 2>(p, stream);
  return dtype == 0 ? launch_bounds_t<64, Bf16Tag, 2>(p, stream)
                    : launch_bounds_t<64, F16Tag, 2>(p, stream);
}

hipError_t launch_select_blocks(const SelectParams& p, int head_dim, int dtype, bool fp8,
                                hipStream_t stream) {
  if (head_dim == 128)
    return dtype == 0 ? launch_select_d<128, Bf16Tag>(p, fp8, stream)
                      : launch_select_d<128, F16Tag>(p, fp8, stream);
  return dtype == 0 ? launch_select_d<64, Bf16Tag>(p, fp8, stream)
                    : launch_select_d<64, F16Tag>(p, fp8, stream);
}

}  // namespace ifa4
