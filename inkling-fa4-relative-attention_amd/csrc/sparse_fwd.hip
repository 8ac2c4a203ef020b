// Attention over listed blocks of a paged cache for gfx950 (MI355X): each token and kv head
// attends to the blocks that its own list names.  The reference has none.
//
//   x_j = scale q . k_j + bias[pos - j]  (0 <= pos - j < rel_extent) over the keys j <= pos,
//   j >= pos - window of the listed blocks, pos the token's position (bottom-right);
//   out = softmax(x) V, lse = log sum exp(x), as in the paged decode.
//
// Work decomposition.  A workgroup of kNw waves takes one (token, kv head) or, for few of them, one
// of `splits` shares of its list.  The listed rows laid end to end are cut into steps of 32 keys,
// dealt to the waves in turn, each with a softmax of its own; the waves meet in LDS, the shares in
// a second pass.  A step is two halves of 16 keys, each in one block (blocks of 8 rows:
// four runs of 8).  A wave holds 64 entries of the list, one a lane, with what the steps need of
// them as bit masks: which have a visible key at all (others are passed over), which are visible
// whole and away from the bias (their steps take neither mask nor bias).
//
// Products (16x16x32 MFMA, the group's query heads as the 16 columns, zero padded).  S^T = K Q^T,
// A = K rows through a swizzled LDS tile (16 bytes a lane; e4m3: they are the operands of two
// products, Q taken in the same order): lane (n, g) = (l % 16, l / 16) gets
// keys 16 blk + 4g + j of head n.  They are the k-slots 8g + 4 blk + j of O^T += V^T P^T as they
// stand; A = V^T through a swizzled LDS tile whose row 8g + 4 blk + j holds key 16 blk + 4g + j, by
// transposing reads of 16 or 8 bits.
//
// What bounds it: a decode step the bytes of the listed rows, and the chain of dependent reads
// before the first of them (offsets and list, lengths and table, rows), each of which is issued as
// early as its address is known; a chunk the instructions of a step, as every token reads blocks
// of its own (from L2), which is why a plain step has so few of them.
#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

constexpr int kStep = kSparseStep;
typedef int i32x4_t __attribute__((ext_vector_type(4)));

template <int D, int Eb>
struct SparseShape {
  static constexpr int kLpr = D * Eb / 16;    // lanes (16-byte chunks) per row
  static constexpr int kRpi = 64 / kLpr;      // rows per load
  static constexpr int kLoads = kStep / kRpi; // of K, and of V
  static constexpr int kKSteps = D / 32;      // products per half
  static constexpr int kDBlocks = D / 16;
  static constexpr int kBytes = kStep * D * Eb;  // of a tile
};

// K tile: chunk c of row `row` (the step's keys in order) sits at c ^ kswz(row): the 16 rows that a
// read of the A operand covers at one chunk lie in distinct banks.
template <int D, int Eb>
__device__ __forceinline__ int kswz(int row) {
  constexpr int kChunks = D * Eb / 16;
  return row / (16 / kChunks) & (kChunks - 1);
}
// V tile: row of key `key` of a step (see above).
__device__ __forceinline__ int tile_row(int key) {
  return 8 * ((key >> 2) & 3) + 4 * (key >> 4) + (key & 3);
}
// 16-byte chunk c of tile row `row` sits at c ^ vswz(row).  A transposing read of 16 bits covers rows
// 8g + 4r .. + 3 of two groups g at one chunk pair, one of 8 bits rows 8g .. 8g + 7 at one chunk: the
// swizzle gives these rows distinct banks.
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

// 16 bytes at a wave's address plus a lane's offset, declared global memory: an address made from
// integers counts as a flat one otherwise, and a wait for an LDS read then waits for the loads.
template <bool kOnce>
__device__ __forceinline__ u32x4_t ld_kv(uint64_t base, uint32_t off) {
  typedef const __attribute__((address_space(1))) char* bytes_t;
  typedef const __attribute__((address_space(1))) u32x4_t* vec_t;
  const vec_t p = reinterpret_cast<vec_t>(reinterpret_cast<bytes_t>(base) + off);
  if constexpr (kOnce) return __builtin_nontemporal_load(p);
  return *p;
}
// Bias at distances d, d - 1, d - 2, d - 3 of a row; anything where that is none.
__device__ __forceinline__ void rel_values(const SparseParams& p, int64_t row, int d, float* x) {
  if (p.rel_dtype == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[j] = static_cast<const float*>(p.rel)[row + min(max(d - j, 0), p.rel_extent - 1)];
    return;
  }
  uint16_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = static_cast<const uint16_t*>(p.rel)[row + min(max(d - j, 0), p.rel_extent - 1)];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j] = p.rel_dtype == 0 ? __uint_as_float((uint32_t)w[j] << 16) : (float)__builtin_bit_cast(_Float16, w[j]);
}

// kEight: blocks of 8 rows (not where one load takes 16: e4m3, d 64).  kOnce: one token a sequence,
// no other will read its rows, and they pass the caches by (64 sequences x 128 blocks of 16, a call,
// 39.8 -> 35.2 us, 128 x 256 111 -> 98; a branch in the kernel instead comes out as one plain load).
template <int D, typename Tag, int Eb, int kNw, bool kEight, bool kOnce>
__global__ __launch_bounds__(64 * kNw) __attribute__((amdgpu_waves_per_eu(2))) void
sparse_fwd_kernel(SparseParams p) {
  using E = Elem<Tag>;
  using S = SparseShape<D, Eb>;
  static_assert(!kEight || S::kRpi <= 8, "a load's rows lie in one block");
  // a wave's K and V tiles, and in the end its partial O [16][D] fp32
  constexpr int kTileBytes = 2 * S::kBytes < 16 * D * 4 ? 16 * D * 4 : 2 * S::kBytes;
  __shared__ __align__(16) uint8_t tiles[kNw][kTileBytes];
  __shared__ float part_m[kNw][16], part_l[kNw][16];
  const int lane = threadIdx.x & 63;
  const int wave = kNw > 1 ? (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int n = lane & 15, g = lane >> 4;

  // workgroup -> (share, token, kv head); tokens side by side on one XCD (workgroup i runs on XCD
  // i % 8), whose L2 then serves blocks that neighbours both list
  const uint32_t at = (blockIdx.x % 8) * (uint32_t)p.per_xcd + blockIdx.x / 8;
  if (at >= (uint32_t)p.groups) return;
  const uint32_t item = p.by_splits.div(at);
  const int split = (int)(at - item * (uint32_t)p.splits);
  const int kvh = (int)p.by_total.div(item), t = (int)(item - (uint32_t)kvh * (uint32_t)p.total_q);
  const int head0 = kvh * p.group;
  const int my_head = head0 + min(n, p.group - 1);  // of column n

  // ---- what hangs on nothing but the item: list entries, Q --------------------------------------
  const int32_t* const list = p.blocks + (int64_t)t * p.ls_st + (int64_t)kvh * p.ls_sh;
  // Own step k of a wave is step k * stride + first of the list: steps near the token's position
  // take the bias, and every wave has some of them.
  const int stride = kNw * p.splits, first_step = split * kNw + wave;
  const int s_end = first_step < p.steps ? (p.steps - first_step - 1) / stride + 1 : 0;
  // Lane l holds the list entry of own step win + l / 4 or l / 2 in blocks of 8 and 16,
  // which hold a quarter or a half of a step, else of win + l.
  const int per_shift = p.block_shift < 5 ? 5 - p.block_shift : 0;
  auto entry_of = [&](int step0) {
    const int s = (step0 + (lane >> per_shift)) * stride + first_step;
    return p.block_shift < 5 ? (s << per_shift) + (lane & ((1 << per_shift) - 1)) : s >> (p.block_shift - 5);
  };
  int win = 0, ent = -1;
  if (const int e = entry_of(0); e < p.n_select) ent = list[e];
  u32x4_t qf[S::kKSteps];
  {
    const uint16_t* const src = static_cast<const uint16_t*>(p.q) + (int64_t)t * p.q_st +
                                (int64_t)my_head * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < S::kKSteps; ++kk) {
      const int d = Eb == 2 ? 32 * kk + 8 * g : 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
      qf[kk] = ld_global_16(src + d);
      if (n >= p.group) qf[kk] = u32x4_t{0u, 0u, 0u, 0u};
    }
  }

  // ---- the token's sequence: the first whose tokens end past it ----------------------------------
  int seq = -1, q_beg = 0, q_end = 0;
  for (int b0 = 0; b0 < p.batch && seq < 0; b0 += 64) {
    const int b = min(b0 + lane, p.batch - 1);
    const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1];
    const uint64_t past = __builtin_amdgcn_ballot_w64(b0 + lane < p.batch && c1 > t);
    if (past != 0) {
      const int l = (int)__builtin_ctzll(past);
      seq = b0 + l;
      q_beg = min(max((int)__builtin_amdgcn_readlane(c0, l), 0), p.total_q);
      q_end = min(max((int)__builtin_amdgcn_readlane(c1, l), q_beg), p.total_q);
    }
  }
  if (seq < 0 || t < q_beg || t >= q_end) return;
  const int32_t* const table = p.block_table + (int64_t)seq * p.bt_stride;
  auto lookup = [&](int blk) {  // place in the pool, or -1
    const bool in = (uint32_t)blk < (uint32_t)p.max_blocks;
    const int phys = table[in ? blk : 0];
    return in && (uint32_t)phys < (uint32_t)p.num_blocks ? phys : -1;
  };
  int phys = lookup(ent);
  const int lk = min(max(p.seqused_k[seq], 0), p.max_blocks << p.block_shift);
  const int pos = lk - (q_end - q_beg) + (t - q_beg);
  const int kmin = p.window_left >= 0 ? max(0, pos - p.window_left) : 0;  // visible: kmin .. pos

  // ---- the window of list entries ---------------------------------------------------------------
  const int bs = 1 << p.block_shift, bmask = bs - 1;
  const char* const k_head = static_cast<const char*>(p.k) + (int64_t)kvh * p.k_sh * Eb;
  const char* const v_head = static_cast<const char*>(p.v) + (int64_t)kvh * p.v_sh * Eb;
  uint64_t some = 0, plain = 0;  // entries with a visible key; visible whole and off the band
  uint64_t k_at = 0, v_at = 0;   // the entry's block; the pool's first for one without a visible key
  auto classify = [&] {
    const int first = ent << p.block_shift;  // (meaningless where phys < 0)
    const bool any = phys >= 0 && first <= pos && first + bmask >= kmin;
    some = __builtin_amdgcn_ballot_w64(any);
    plain = __builtin_amdgcn_ballot_w64(any && first + bmask <= pos && first >= kmin &&
                                        pos - (first + bmask) >= p.rel_extent);
    k_at = reinterpret_cast<uint64_t>(k_head + (int64_t)(any ? phys : 0) * p.k_sblk * Eb);
    v_at = reinterpret_cast<uint64_t>(v_head + (int64_t)(any ? phys : 0) * p.v_sblk * Eb);
  };
  classify();
  constexpr int kRuns = kEight ? 4 : 2;
  const uint64_t step_bits = kEight ? 15 : bs == 16 ? 3 : 1;
  auto seek = [&](int s) {  // first own step from s on that reads anything
    for (; s < s_end; ++s) {
      if (s >= win + (64 >> per_shift)) {
        win = s;
        const int e = entry_of(win);
        ent = e < p.n_select ? list[e] : -1;
        phys = lookup(ent);
        classify();
      }
      if ((some >> ((s - win) << per_shift)) & step_bits) break;
    }
    return s;
  };
  // What a step's products have to know: the position of each run's first key (kFar: the run has no
  // visible key), and whether every key is visible without bias (then positions are not set).
  constexpr int kFar = 1 << 30;
  struct Step {
    i32x4_t pos;
    bool plain;
  };
  const int vr = lane / S::kLpr, vc = lane % S::kLpr;  // row layout of the loads
  const int k_rowb = (int)p.k_st * Eb, v_rowb = (int)p.v_st * Eb;
  const uint32_t k_lane = (uint32_t)vr * (uint32_t)k_rowb + 16 * vc;
  const uint32_t v_lane = (uint32_t)vr * (uint32_t)v_rowb + 16 * vc;
  auto scalar64 = [](uint64_t x, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)x, l);
  };
  auto load = [&](int s, u32x4_t* kr, u32x4_t* vv) -> Step {
    Step st;
    const int v0 = (s * stride + first_step) * kStep, e0 = (s - win) << per_shift;
    st.plain = ((plain >> e0) & step_bits) == step_bits;
    st.pos = i32x4_t{kFar, kFar, kFar, kFar};
    uint64_t kb[kRuns], vb[kRuns];
#pragma unroll
    for (int r = 0; r < kRuns; ++r) {
      const int v = v0 + kStep / kRuns * r, e = e0 + (kStep / kRuns * r >> p.block_shift);
      kb[r] = scalar64(k_at, e) + (uint32_t)((v & bmask) * k_rowb);
      vb[r] = scalar64(v_at, e) + (uint32_t)((v & bmask) * v_rowb);
      if (!st.plain) {
        const int first = ((int)__builtin_amdgcn_readlane(ent, e) << p.block_shift) + (v & bmask);
        if (((some >> e) & 1) && first <= pos && first + kStep / kRuns > kmin) st.pos[r] = first;
      }
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int r = S::kRpi * i / (kStep / kRuns);  // run, first row in it
      const int off = S::kRpi * i % (kStep / kRuns);
      kr[i] = ld_kv<kOnce>(kb[r] + (uint32_t)(off * k_rowb), k_lane);
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int r = S::kRpi * i / (kStep / kRuns);
      const int off = S::kRpi * i % (kStep / kRuns);
      vv[i] = ld_kv<kOnce>(vb[r] + (uint32_t)(off * v_rowb), v_lane);
    }
    return st;
  };

  const int64_t rel_row = (int64_t)t * p.rel_st + (int64_t)my_head * p.rel_sh;
  const float c2 = p.scale_log2;
  float m_run = -INFINITY, l_run = 0.f;  // of head n (same over g; the sum over this lane's keys)
  f32x4_t o[S::kDBlocks];
#pragma unroll
  for (int db = 0; db < S::kDBlocks; ++db) o[db] = f32x4_t{};
  uint8_t* const k_tile = tiles[wave];
  uint8_t* const tile = k_tile + S::kBytes;

  auto stage = [&](const Step& st, const u32x4_t* kr, u32x4_t* vv) {
    if (!st.plain) {  // V rows that the token does not see hold anything: zero
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int key = S::kRpi * i + vr;
        int first;
        if constexpr (kEight) {
          const int r = key >> 3;
          first = (r == 0 ? st.pos[0] : r == 1 ? st.pos[1] : r == 2 ? st.pos[2] : st.pos[3]) + (key & 7);
        } else {
          first = (key < 16 ? st.pos[0] : st.pos[1]) + (key & 15);
        }
        if (first > pos || first < kmin) vv[i] = u32x4_t{0u, 0u, 0u, 0u};
      }
    }
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int key = S::kRpi * i + vr, row = tile_row(key);
      *reinterpret_cast<u32x4_t*>(k_tile + key * D * Eb + 16 * (vc ^ kswz<D, Eb>(key))) = kr[i];
      *reinterpret_cast<u32x4_t*>(tile + row * D * Eb + 16 * (vc ^ vswz<D, Eb>(row))) = vv[i];
    }
  };
  auto compute = [&](const Step& st) {
    wave_lds_sync();
    f32x4_t acc[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      acc[b] = f32x4_t{};
      const uint8_t* const k_row = k_tile + (16 * b + n) * D * Eb;
      const int sw = kswz<D, Eb>(16 * b + n);
#pragma unroll
      for (int i = 0; i < D * Eb / 64; ++i) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(k_row + 16 * ((4 * i + g) ^ sw));
        if constexpr (Eb == 2) {
          acc[b] = E::mfma16(w, qf[i], acc[b]);
        } else {
          acc[b] = E::mfma16(fp8x8_operand<E>(w[0], w[1]), qf[2 * i], acc[b]);
          acc[b] = E::mfma16(fp8x8_operand<E>(w[2], w[3]), qf[2 * i + 1], acc[b]);
        }
      }
    }
    if (!st.plain) {
      // positions of the lane's four keys of either half
      int kp[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if constexpr (kEight)
          kp[b] = (g < 2 ? st.pos[2 * b] : st.pos[2 * b + 1]) + 4 * (g & 1);
        else
          kp[b] = st.pos[b] + 4 * g;
      }
      // bias / softmax_scale joins the products, keys out of sight become -inf
      const float inv = kLog2e / c2;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int d0 = pos - kp[b];
        if (p.rel_extent > 0 && wave_any(d0 >= 0 && d0 - 3 < p.rel_extent)) {
          float bias[4];  // loads in flight together
          rel_values(p, rel_row, d0, bias);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[b][j] = fmaf((uint32_t)(d0 - j) < (uint32_t)p.rel_extent ? bias[j] : 0.f, inv, acc[b][j]);
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int hi = pos - kp[b], lo = kmin - kp[b];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[b][j] = j >= lo && j <= hi ? acc[b][j] : -INFINITY;
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(acc[0][0], acc[0][1]), fmaxf(acc[0][2], acc[0][3])),
                     fmaxf(fmaxf(acc[1][0], acc[1][1]), fmaxf(acc[1][2], acc[1][3])));
    mx = max_xor16(mx);
    mx = max_xor32(mx) * c2;
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
      pv[e] = fast_exp2(fmaf(acc[e >> 2][e & 3], c2, -m_use));
      l_run += pv[e];
    }
    // The second product takes the weights in q's type, as in the framework's other attentions (its
    // 16-bit matrix instructions; half a step of each weight, about as much as the output's own
    // rounding); their sum is that of the fp32 ones.
    const u32x4_t pb = {E::pack2(pv[0], pv[1]), E::pack2(pv[2], pv[3]), E::pack2(pv[4], pv[5]),
                        E::pack2(pv[6], pv[7])};
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
    wave_lds_sync();  // the tiles are rewritten by the next step
  };

  // ---- steps, the next one's rows in flight while one is computed ---------------------------------
  u32x4_t kr[S::kLoads], vv[S::kLoads];
  Step next{};
  int s = seek(0);
  if (s < s_end) next = load(s, kr, vv);
  while (s < s_end) {
    const Step st = next;
    stage(st, kr, vv);
    s = seek(s + 1);
    if (s < s_end) next = load(s, kr, vv);
    compute(st);
  }

  // ---- the waves' partials meet ---------------------------------------------------------------------
  const float l_tot = add_xor32(add_xor16(l_run));
  auto put = [&](int h, int d, f32x4_t sum, float m, float l) {
    const int head = head0 + h;
    if (p.splits > 1) {
      const int64_t row = ((int64_t)split * p.total_q + t) * p.n_heads + head;
      *reinterpret_cast<f32x4_t*>(p.part_o + row * D + d) = sum;
      if (d == 0) p.part_ml[row] = make_float2(m, l);
      return;
    }
    // l is 0 for a row without keys, NaN where a key is: then the LSE is too
    const float inv = l == 0.f ? 0.f : p.v_scale / l;
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + (int64_t)t * p.o_st +
                                (int64_t)head * p.o_sh + d) =
        u32x2_t{E::pack2(sum[0] * inv, sum[1] * inv), E::pack2(sum[2] * inv, sum[3] * inv)};
    if (p.lse != nullptr && d == 0)
      p.lse[(int64_t)head * p.lse_sh + t] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
  };
  if constexpr (kNw == 1) {
    if (n < p.group) {
#pragma unroll
      for (int db = 0; db < S::kDBlocks; ++db) put(n, 16 * db + 4 * g, o[db], m_run, l_tot);
    }
  } else {
    float* const own = reinterpret_cast<float*>(k_tile);
    if (n < p.group) {
#pragma unroll
      for (int db = 0; db < S::kDBlocks; ++db)
        *reinterpret_cast<f32x4_t*>(own + n * D + 16 * db + 4 * g) = o[db];
      if (g == 0) {
        part_m[wave][n] = m_run;
        part_l[wave][n] = l_tot;
      }
    }
    __syncthreads();
    constexpr int kRowChunks = D / 4;
    for (int c4 = threadIdx.x; c4 < p.group * kRowChunks; c4 += 64 * kNw) {
      const int h = c4 / kRowChunks, d = 4 * (c4 % kRowChunks);
      float mt = part_m[0][h];
#pragma unroll
      for (int i = 1; i < kNw; ++i) mt = fmaxf(mt, part_m[i][h]);
      const float mu = mt == -INFINITY ? 0.f : mt;
      float lt = 0.f;
      f32x4_t sum{};
#pragma unroll
      for (int i = 0; i < kNw; ++i) {
        const float a = fast_exp2(part_m[i][h] - mu);
        lt += a * part_l[i][h];
        sum += a * *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(tiles[i]) + h * D + d);
      }
      put(h, d, sum, mt, lt);
    }
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
  const float inv = lt == 0.f ? 0.f : p.v_scale / lt;
  *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + t * p.o_st + (int64_t)head * p.o_sh + d) =
      u32x2_t{E::pack2(sum[0] * inv, sum[1] * inv), E::pack2(sum[2] * inv, sum[3] * inv)};
  if (p.lse != nullptr && d == 0)
    p.lse[(int64_t)head * p.lse_sh + t] = lt == 0.f ? -INFINITY : (mt + __log2f(lt)) * kLn2;
}

template <int D, typename Tag, int Eb, int kNw, bool kOnce>
void launch_sparse_w(const SparseParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.per_xcd * 8), block(64 * kNw);
  if constexpr (SparseShape<D, Eb>::kRpi <= 8) {
    if (p.block_shift == 3) {
      hipLaunchKernelGGL((sparse_fwd_kernel<D, Tag, Eb, kNw, true, kOnce>), grid, block, 0, stream, p);
      return;
    }
  }
  hipLaunchKernelGGL((sparse_fwd_kernel<D, Tag, Eb, kNw, false, kOnce>), grid, block, 0, stream, p);
}

template <int D, typename Tag, int Eb, bool kOnce>
void launch_sparse_o(const SparseParams& p, hipStream_t stream) {
  switch (p.waves) {
    case 1: launch_sparse_w<D, Tag, Eb, 1, kOnce>(p, stream); break;
    case 2: launch_sparse_w<D, Tag, Eb, 2, kOnce>(p, stream); break;
    case 4: launch_sparse_w<D, Tag, Eb, 4, kOnce>(p, stream); break;
    default: launch_sparse_w<D, Tag, Eb, 8, kOnce>(p, stream);
  }
}

template <int D, typename Tag, int Eb>
hipError_t launch_sparse_t(const SparseParams& p, hipStream_t stream) {
  if (p.once)
    launch_sparse_o<D, Tag, Eb, true>(p, stream);
  else
    launch_sparse_o<D, Tag, Eb, false>(p, stream);
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

template <int D, typename Tag>
hipError_t launch_sparse_d(const SparseParams& p, hipStream_t stream) {
  return p.kv_fp8 ? launch_sparse_t<D, Tag, 1>(p, stream) : launch_sparse_t<D, Tag, 2>(p, stream);
}

}  // namespace

hipError_t launch_sparse(const SparseParams& p, int head_dim, int qkv_dtype, hipStream_t stream) {
  if (head_dim == 128)
    return qkv_dtype == 0 ? launch_sparse_d<128, Bf16Tag>(p, stream)
                          : launch_sparse_d<128, F16Tag>(p, stream);
  return qkv_dtype == 0 ? launch_sparse_d<64, Bf16Tag>(p, stream)
                        : launch_sparse_d<64, F16Tag>(p, stream);
}

}  // namespace ifa4
