// Attention over listed blocks of a paged cache for gfx950 (MI355X): each token and kv head
// attends to the blocks that its own list names.  The reference has none.
//
//   x_j = scale q . k_j + bias[pos - j]  (0 <= pos - j < rel_extent) over the keys j <= pos,
//   j >= pos - window of the listed blocks, pos the token's position (bottom-right);
//   out = softmax(x) V, lse = log sum exp(x), as in the paged decode.
//
// Work decomposition.  A workgroup of four waves takes one (token, kv head) or, for few of them,
// one of `splits` shares of its list.  The listed rows laid end to end are cut into steps of 32
// keys and every wave takes an equal run of steps, with a softmax of its own; the four meet in
// LDS, the shares in a second pass.  A step is four runs of eight keys; each run lies in one block
// (blocks hold eight rows or more), so what is known per run - its block in the pool, its position,
// which of its keys are visible - is the lane's that holds the run's keys.
//
// Products (16x16x32 MFMA, the group's query heads as the 16 columns, zero padded).  S^T = K Q^T:
// row 4g + j of key block blk is key 8g + 4 blk + j, so lane (n, g) = (l % 16, l / 16) ends up with
// the eight keys of run g, and its P are the k-slots 8g .. 8g+7 of O^T += V^T P^T as they stand.
// A = K rows straight from memory (16 bytes a lane; e4m3: 16 bytes are the operands of two
// products, Q taken in the same order), A = V^T through a swizzled LDS tile by transposing reads.
// A list is read once and its blocks lie anywhere: what bounds a decode step is the bytes of
// the listed rows, what bounds a chunk is the same rows from L2 for every token.
#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

constexpr int kWaves = kSparseWaves, kStep = kSparseStep;
typedef int i32x4_t __attribute__((ext_vector_type(4)));

template <int D, int Eb>
struct SparseShape {
  static constexpr int kLpr = D * Eb / 16;    // lanes per V row
  static constexpr int kRpi = 64 / kLpr;      // V rows per load
  static constexpr int kVLoads = kStep / kRpi;
  static constexpr int kKLoads = D * Eb / 64; // 16-byte loads per lane and key block of 16
  static constexpr int kKSteps = D / 32;      // products per key block
  static constexpr int kDBlocks = D / 16;
  static constexpr int kVBytes = kStep * D * Eb;
  static constexpr int kLdsBytes = kVBytes > 16 * D * 4 ? kVBytes : 16 * D * 4;  // a wave's tile
};

// 16-byte chunk of V row `row` in LDS: chunk c sits at c ^ vswz(row).  A transposing read of 16
// bits covers rows 8g + 4r .. + 3 of two groups g at one chunk pair, one of 8 bits rows 8g .. 8g + 7
// at one chunk: the swizzle gives these rows distinct banks.
template <int D, int Eb>
__device__ __forceinline__ int vswz(int row) {
  if constexpr (Eb == 2 && D == 128) return 2 * ((row & 3) | ((row >> 3) & 1) << 2);
  if constexpr (Eb == 2 && D == 64) return 2 * (((row >> 1) & 1) | ((row >> 3) & 1) << 1);
  if constexpr (Eb == 1 && D == 128) return (row >> 1) & 7;
  return (row >> 2) & 3;
}

template <typename E>
__device__ __forceinline__ u32x4_t fp8x8_operand(uint32_t lo, uint32_t hi) {
  return u32x4_t{E::template fp8x2<false>(lo), E::template fp8x2<true>(lo),
                 E::template fp8x2<false>(hi), E::template fp8x2<true>(hi)};
}

__device__ __forceinline__ float rel_value(const SparseParams& p, int64_t off) {
  if (p.rel_dtype == 2) return static_cast<const float*>(p.rel)[off];
  const uint16_t x = static_cast<const uint16_t*>(p.rel)[off];
  return p.rel_dtype == 0 ? __uint_as_float((uint32_t)x << 16) : (float)__builtin_bit_cast(_Float16, x);
}

template <int D, typename Tag, int Eb>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2))) void
sparse_fwd_kernel(SparseParams p) {
  using E = Elem<Tag>;
  using S = SparseShape<D, Eb>;
  __shared__ __align__(16) uint8_t tiles[kWaves][S::kLdsBytes];
  __shared__ float part_m[kWaves][16], part_l[kWaves][16];
  const int lane = threadIdx.x & 63;
  const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;

  // workgroup -> (share, token, kv head); tokens side by side on one XCD (workgroup i runs on XCD
  // i % 8), whose L2 then serves blocks that neighbours both list
  const uint32_t items = (uint32_t)p.total_q * (uint32_t)p.kv_heads * (uint32_t)p.splits;
  const uint32_t per_xcd = (items + 7) / 8;
  const uint32_t at = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (at >= items) return;
  const int split = (int)(at % (uint32_t)p.splits);
  const uint32_t item = at / (uint32_t)p.splits;
  const int kvh = (int)(item / (uint32_t)p.total_q), t = (int)(item - (uint32_t)kvh * (uint32_t)p.total_q);
  const int head0 = kvh * p.group;

  // the token's sequence: the first whose tokens end past it
  int seq = -1;
  for (int b0 = 0; b0 < p.batch && seq < 0; b0 += 64) {
    const int b = b0 + lane;
    const uint64_t past =
        __builtin_amdgcn_ballot_w64(b < p.batch && p.cu_q[min(b, p.batch - 1) + 1] > t);
    if (past != 0) seq = b0 + (int)__builtin_ctzll(past);
  }
  if (seq < 0) return;
  const SeqBounds bq = seq_bounds(p.cu_q, seq, p.total_q);
  if (t < bq.start || t >= bq.start + bq.len) return;
  const int lk = min(max(p.seqused_k[seq], 0), p.max_blocks << p.block_shift);
  const int pos = lk - bq.len + (t - bq.start);
  const int kmin = p.window_left >= 0 ? max(0, pos - p.window_left) : 0;  // visible: kmin .. pos

  // ---- this wave's steps --------------------------------------------------------------------
  const int64_t rows = (int64_t)p.n_select << p.block_shift;
  const int steps = pos < 0 ? 0 :  // no key at all: out 0, lse -inf
                        (int)((rows + kStep - 1) / kStep);
  const int parts = p.splits * kWaves, mine = split * kWaves + wave;
  const int s_beg = (int)((int64_t)steps * mine / parts), s_end = (int)((int64_t)steps * (mine + 1) / parts);
  const int bmask = (1 << p.block_shift) - 1;
  const int32_t* const list = p.blocks + (int64_t)t * p.ls_st + (int64_t)kvh * p.ls_sh;
  const int32_t* const table = p.block_table + (int64_t)seq * p.bt_stride;

  // Lane l holds list entry win + l: the position of the block's first row and its place in the
  // pool (-1: no entry, no block, or none of its keys visible).
  int win = -1, ent_pos = 0, ent_blk = -1;
  auto load_window = [&](int first) {
    win = first;
    const int e = first + lane;
    const int blk = e < p.n_select ? list[e] : -1;
    const bool named = (uint32_t)blk < (uint32_t)p.max_blocks &&
                       (blk << p.block_shift) <= pos && ((blk + 1) << p.block_shift) > kmin;
    const int phys = table[named ? blk : 0];
    ent_pos = blk << p.block_shift;
    ent_blk = named && (uint32_t)phys < (uint32_t)p.num_blocks ? phys : -1;
  };
  // The runs of a step: run r's block (-1: nothing to read) and the position of its first key,
  // wave-uniform.
  struct Step {
    i32x4_t blk, pos;
  };
  auto find = [&](int s) -> Step {
    const int first = s * kStep;
    const int e0 = first >> p.block_shift, e3 = (first + kStep - 8) >> p.block_shift;
    if (win < 0 || e0 < win || e3 >= win + 64) load_window(e0);
    // a run past the token, or left of its window, is not read
    auto run_pos = [&](int r) {
      const int v = first + 8 * r;
      return (int)__builtin_amdgcn_readlane(ent_pos, (v >> p.block_shift) - win) + (v & bmask);
    };
    auto run_blk = [&](int r, int at) {
      const int blk = __builtin_amdgcn_readlane(ent_blk, ((first + 8 * r) >> p.block_shift) - win);
      return at <= pos && at + 7 >= kmin ? blk : -1;
    };
    const i32x4_t at = {run_pos(0), run_pos(1), run_pos(2), run_pos(3)};
    return Step{i32x4_t{run_blk(0, at[0]), run_blk(1, at[1]), run_blk(2, at[2]), run_blk(3, at[3])}, at};
  };
  auto reads = [](const Step& st) {
    return max(max(st.blk[0], st.blk[1]), max(st.blk[2], st.blk[3])) >= 0;
  };
  const int vr = lane / S::kLpr, vc = lane % S::kLpr;  // row layout of the V loads
  auto load = [&](const Step& st, u32x4_t* kr, u32x4_t* vv) {
    // K: lane (n, g) reads row n of each key block, key 8 (n / 4) + 4 blk + n % 4, a row of an
    // absent run from the pool's first row (its scores are masked)
    const int run = n >> 2;
    const int kb = run == 0 ? st.blk[0] : run == 1 ? st.blk[1] : run == 2 ? st.blk[2] : st.blk[3];
    const int kp = run == 0 ? st.pos[0] : run == 1 ? st.pos[1] : run == 2 ? st.pos[2] : st.pos[3];
    const int64_t row = kb >= 0 ? (kp & bmask) + (n & 3) : 0;
    const char* const src = static_cast<const char*>(p.k) +
                            ((kb >= 0 ? (int64_t)kb : 0) * p.k_sblk + (int64_t)kvh * p.k_sh +
                             row * p.k_st) * Eb + 16 * g;
    const int64_t next = kb >= 0 ? 4 * p.k_st * Eb : 0;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int i = 0; i < S::kKLoads; ++i) kr[blk * S::kKLoads + i] = ld_global_16(src + blk * next + 64 * i);
    // V: rows through one resource a run (e4m3, d 64: a load's 16 rows lie in one block), rows
    // that no query sees read as zero
#pragma unroll
    for (int i = 0; i < S::kVLoads; ++i) {
      const int r = S::kRpi * i / 8, off = S::kRpi * i % 8;  // run, first row in it
      const int first = st.pos[r] + off;
      // a load of 16 rows covers two runs of one block
      const int vblk = S::kRpi > 8 ? max(st.blk[r], st.blk[r + (S::kRpi > 8 ? 1 : 0)]) : st.blk[r];
      const bool on = vblk >= 0;
      const int left = pos + 1 - first;
      const char* const base = static_cast<const char*>(p.v) +
                               ((on ? (int64_t)vblk : 0) * p.v_sblk + (int64_t)kvh * p.v_sh +
                                (on ? (int64_t)(first & bmask) : 0) * p.v_st) * Eb;
      const rsrc_t rv = make_rsrc_uniform(
          base, on && left > 0 ? (uint32_t)(((int64_t)(min(left, S::kRpi) - 1) * p.v_st + D) * Eb) : 0u);
      vv[i] = buf_load_16(rv, first + vr >= kmin ? (uint32_t)(vr * (int)p.v_st * Eb + 16 * vc) : kOutOfRange);
    }
  };

  // ---- Q: column n = query head n of the kv head ------------------------------------------------
  u32x4_t qf[S::kKSteps];
  {
    const uint16_t* const src = static_cast<const uint16_t*>(p.q) + (int64_t)t * p.q_st +
                                (int64_t)(head0 + min(n, p.group - 1)) * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < S::kKSteps; ++kk) {
      const int d = Eb == 2 ? 32 * kk + 8 * g : 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
      qf[kk] = ld_global_16(src + d);
      if (n >= p.group) qf[kk] = u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  const int64_t rel_row = (int64_t)t * p.rel_st + (int64_t)(head0 + min(n, p.group - 1)) * p.rel_sh;

  const float c2 = p.scale_log2;
  float m_run = -INFINITY, l_run = 0.f;  // of head n (same over g; the sum over this lane's keys)
  f32x4_t o[S::kDBlocks];
#pragma unroll
  for (int db = 0; db < S::kDBlocks; ++db) o[db] = f32x4_t{};
  uint8_t* const tile = tiles[wave];

  auto compute = [&](const Step& st, const u32x4_t* kr, const u32x4_t* vv) {
#pragma unroll
    for (int i = 0; i < S::kVLoads; ++i) {
      const int row = S::kRpi * i + vr;
      *reinterpret_cast<u32x4_t*>(tile + row * D * Eb + 16 * (vc ^ vswz<D, Eb>(row))) = vv[i];
    }
    f32x4_t acc[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      acc[blk] = f32x4_t{};
#pragma unroll
      for (int kk = 0; kk < S::kKSteps; ++kk) {
        u32x4_t a;
        if constexpr (Eb == 2) {
          a = kr[blk * S::kKLoads + kk];
        } else {
          const u32x4_t w = kr[blk * S::kKLoads + (kk >> 1)];
          a = (kk & 1) ? fp8x8_operand<E>(w[2], w[3]) : fp8x8_operand<E>(w[0], w[1]);
        }
        acc[blk] = E::mfma16(a, qf[kk], acc[blk]);
      }
    }
    // lane (n, g): keys kp .. kp + 7 of run g
    const int kb = g == 0 ? st.blk[0] : g == 1 ? st.blk[1] : g == 2 ? st.blk[2] : st.blk[3];
    const int kp = g == 0 ? st.pos[0] : g == 1 ? st.pos[1] : g == 2 ? st.pos[2] : st.pos[3];
    const int hi = kb >= 0 ? min(7, pos - kp) : -1, lo = max(0, kmin - kp);
    const bool masked = wave_any(hi < 7 || lo > 0);
    const bool near = kb >= 0 && n < p.group && pos - kp - 7 < p.rel_extent;
    const bool bias = p.rel_extent > 0 && wave_any(near);
    float mx = -INFINITY;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * blk + j;
        float x = acc[blk][j] * c2;
        if (bias) {
          const int dist = pos - kp - e;
          if (near && (uint32_t)dist < (uint32_t)p.rel_extent)
            x = fmaf(rel_value(p, rel_row + dist), kLog2e, x);
        }
        if (masked) x = e >= lo && e <= hi ? x : -INFINITY;
        acc[blk][j] = x;
        mx = fmaxf(mx, x);
      }
    }
    mx = max_xor16(mx);
    mx = max_xor32(mx);
    const float m_cand = fmaxf(m_run, mx);
    const bool grow = m_cand > m_run + kRescaleThreshold;
    if (wave_any(grow)) {
      const float m_upd = grow ? m_cand : m_run;
      const float alpha = grow ? fast_exp2(m_run - m_upd) : 1.f;
      l_run *= alpha;
      m_run = m_upd;
#pragma unroll
      for (int db = 0; db < S::kDBlocks; ++db) o[db] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float pv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pv[e] = fast_exp2(acc[e >> 2][e & 3] - m_use);
      l_run += pv[e];
    }
    const u32x4_t pb = {E::pack2(pv[0], pv[1]), E::pack2(pv[2], pv[3]), E::pack2(pv[4], pv[5]),
                        E::pack2(pv[6], pv[7])};
    wave_lds_sync();
#pragma unroll
    for (int db = 0; db < S::kDBlocks; ++db) {
      u32x4_t a;
      if constexpr (Eb == 2) {
        u32x2_t part[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = 8 * g + 4 * r + (n >> 2);
          const int chunk = 2 * db + ((n & 3) >> 1);
          const uint8_t* src = tile + row * D * 2 + 16 * (chunk ^ vswz<D, Eb>(row)) + 8 * (n & 1);
          part[r] = __builtin_bit_cast(
              u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (__attribute__((address_space(3))) s16x4_t*)src));
        }
        a = u32x4_t{part[0][0], part[0][1], part[1][0], part[1][1]};
      } else {
        typedef int i32x2_t __attribute__((ext_vector_type(2)));
        const int row = 8 * g + (n >> 1);
        const uint8_t* src = tile + row * D + 16 * (db ^ vswz<D, Eb>(row)) + 8 * (n & 1);
        const u32x2_t w = __builtin_bit_cast(
            u32x2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                         (__attribute__((address_space(3))) i32x2_t*)src));
        a = fp8x8_operand<E>(w[0], w[1]);
      }
      o[db] = E::mfma16(a, pb, o[db]);
    }
    wave_lds_sync();  // the tile is rewritten by the next step
  };

  // ---- steps, the next one's rows in flight while one is computed ---------------------------------
  // s moves to the first step from itself on that reads anything
  auto seek = [&](int& s, Step& st) {
    for (; s < s_end; ++s) {
      st = find(s);
      if (reads(st)) return;
    }
  };
  Step st0{}, st1{};
  u32x4_t k0[2 * S::kKLoads], k1[2 * S::kKLoads], v0[S::kVLoads], v1[S::kVLoads];
  int s0 = s_beg, s1;
  seek(s0, st0);
  if (s0 < s_end) load(st0, k0, v0);
  while (s0 < s_end) {
    s1 = s0 + 1;
    seek(s1, st1);
    if (s1 < s_end) load(st1, k1, v1);
    compute(st0, k0, v0);
    if (s1 >= s_end) break;
    s0 = s1 + 1;
    seek(s0, st0);
    if (s0 < s_end) load(st0, k0, v0);
    compute(st1, k1, v1);
  }

  // ---- the waves' partials meet ---------------------------------------------------------------------
  const float l_tot = add_xor32(add_xor16(l_run));
  float* const own = reinterpret_cast<float*>(tile);
#pragma unroll
  for (int db = 0; db < S::kDBlocks; ++db)
    *reinterpret_cast<f32x4_t*>(own + n * D + 16 * db + 4 * g) = o[db];
  if (g == 0) {
    part_m[wave][n] = m_run;
    part_l[wave][n] = l_tot;
  }
  __syncthreads();
  constexpr int kRowChunks = D / 4;
  for (int c4 = threadIdx.x; c4 < p.group * kRowChunks; c4 += 64 * kWaves) {
    const int h = c4 / kRowChunks, d = 4 * (c4 % kRowChunks);
    float mt = part_m[0][h];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) mt = fmaxf(mt, part_m[i][h]);
    const float mu = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f;
    f32x4_t sum{};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const float a = fast_exp2(part_m[i][h] - mu);
      lt += a * part_l[i][h];
      sum += a * *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(tiles[i]) + h * D + d);
    }
    const int head = head0 + h;
    if (p.splits > 1) {
      const int64_t row = ((int64_t)split * p.total_q + t) * p.n_heads + head;
      *reinterpret_cast<f32x4_t*>(p.part_o + row * D + d) = sum;
      if (d == 0) p.part_ml[row] = make_float2(mt, lt);
      continue;
    }
    const float inv = lt > 0.f ? p.v_scale / lt : 0.f;
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + (int64_t)t * p.o_st +
                                (int64_t)head * p.o_sh + d) =
        u32x2_t{E::pack2(sum[0] * inv, sum[1] * inv), E::pack2(sum[2] * inv, sum[3] * inv)};
    if (p.lse != nullptr && d == 0)
      p.lse[(int64_t)head * p.lse_sh + t] = lt > 0.f ? (mt + __log2f(lt)) * kLn2 : -INFINITY;
  }
}

// Joins the shares of a list: D / 4 threads a (token, head).
constexpr int kJoinThreads = 256;
template <int D, typename Tag>
__global__ __launch_bounds__(kJoinThreads) void sparse_join_kernel(SparseParams p) {
  using E = Elem<Tag>;
  constexpr int kTpr = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / kTpr) + threadIdx.x / kTpr;
  const int64_t rows = (int64_t)p.total_q * p.n_heads;
  if (row >= rows) return;
  const int64_t t = row / p.n_heads;
  const int head = (int)(row - t * p.n_heads), d = 4 * ((int)threadIdx.x % kTpr);
  // tokens of no sequence have no shares
  if (t < max(p.cu_q[0], 0) || t >= p.cu_q[p.batch]) return;
  float mt = -INFINITY;
  for (int s = 0; s < p.splits; ++s) mt = fmaxf(mt, p.part_ml[s * rows + row].x);
  const float mu = mt == -INFINITY ? 0.f : mt;
  float lt = 0.f;
  f32x4_t sum{};
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.part_ml[s * rows + row];
    const float a = fast_exp2(ml.x - mu);
    lt += a * ml.y;
    sum += a * *reinterpret_cast<const f32x4_t*>(p.part_o + (s * rows + row) * D + d);
  }
  const float inv = lt > 0.f ? p.v_scale / lt : 0.f;
  *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + t * p.o_st + (int64_t)head * p.o_sh + d) =
      u32x2_t{E::pack2(sum[0] * inv, sum[1] * inv), E::pack2(sum[2] * inv, sum[3] * inv)};
  if (p.lse != nullptr && d == 0)
    p.lse[(int64_t)head * p.lse_sh + t] = lt > 0.f ? (mt + __log2f(lt)) * kLn2 : -INFINITY;
}

template <int D, typename Tag>
hipError_t launch_sparse_t(const SparseParams& p, hipStream_t stream) {
  const int64_t items = (int64_t)p.total_q * p.kv_heads * p.splits;
  const dim3 grid((unsigned)((items + 7) / 8 * 8)), block(64 * kWaves);
  if (p.kv_fp8)
    hipLaunchKernelGGL((sparse_fwd_kernel<D, Tag, 1>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((sparse_fwd_kernel<D, Tag, 2>), grid, block, 0, stream, p);
  if (p.splits > 1) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int kRows = kJoinThreads / (D / 4);
    const int64_t rows = (int64_t)p.total_q * p.n_heads;
    hipLaunchKernelGGL((sparse_join_kernel<D, Tag>), dim3((unsigned)((rows + kRows - 1) / kRows)),
                       dim3(kJoinThreads), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sparse(const SparseParams& p, int head_dim, int qkv_dtype, hipStream_t stream) {
  if (head_dim == 128)
    return qkv_dtype == 0 ? launch_sparse_t<128, Bf16Tag>(p, stream)
                          : launch_sparse_t<128, F16Tag>(p, stream);
  return qkv_dtype == 0 ? launch_sparse_t<64, Bf16Tag>(p, stream)
                        : launch_sparse_t<64, F16Tag>(p, stream);
}

}  // namespace ifa4
