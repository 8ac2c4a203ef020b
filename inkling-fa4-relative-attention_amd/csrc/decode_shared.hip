// Decode attention of a batch whose sequences begin with the same keys, for gfx950.
//
// Semantics are those of paged decode with bottom-right alignment (decode_fwd.hip): one
// query per sequence, at key position lk - 1, sees keys [max(0, lk - 1 - window), lk) with
// the bias rel[lk - 1 - j] where that distance is below rel_extent.  Here the first
// prefix_len keys of every sequence are the rows of the same blocks (prefix_table).  With
// K V of the prefix alike, the scores and sums of all sequences over it are two matrix
// products per kv head,
//   S = Q K^T,  O = P V   with  Q [batch * group, D],
// so the prefix is read once per 128 rows of Q instead of once per sequence, and its work
// sits on the matrix cores.  What each sequence holds past the prefix is streamed per
// sequence; the two and their parts meet by log-sum-exp.
//
// One launch of two kinds of workgroups (4 waves), then the merge:
//   prefix  128 rows (32 a wave; row = sequence * group + head of the kv head) x a chunk of
//           64-key tiles, in two LDS stages: the DMA of the next tile (16-bit cache), or its
//           loads into registers (e4m3, converted on the way to LDS), run under the products
//           of the current one;
//   own     one (sequence, kv head) x a chunk of its own keys: wave w takes the 32-key steps
//           w, w + 4, ... in its own quarter of the LDS, its group's heads in the columns of
//           the product; the waves' sums meet in LDS.
// Both leave one row per part and query head in the workspace: the unnormalised o, the maximum
// and the sum.  Maximum and sum stay apart: next to a bias of -3e38 the log of the sum would
// vanish, and with it the parts' shares.
//
// Scores as in prefill_fwd.hip: S^T = K Q^T on v_mfma_f32_32x32x16 (a lane holds one row and
// 16 consecutive keys of every 32), P goes from the accumulator straight into O^T = V^T P^T,
// V^T by transposing LDS reads.  Tiles that meet no mask and no bias for any row of the wave
// take one FMA and one exp2 per score.  The others are computed in natural units,
// exp2((s - m) log2 e), so that biases down to the lowest finite fp32 stay finite: a row that
// has nothing else gives the softmax over them.
#include <type_traits>

#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // rows of a prefix workgroup
constexpr int kTile = 64;           // keys of a prefix tile
constexpr int kOwnStep = 32;        // keys of a wave's step over a sequence's own keys
static_assert(kSharedTile == kTile && kSharedRows == kRows, "the host plans with these");
static_assert(kSharedOwnStep == kOwnStep * kWaves, "the host plans with these");

// s_waitcnt immediates: no vector-memory operation, no LDS operation of this wave outstanding.
constexpr int kVm0 = (7 << 4) | (15 << 8);
constexpr int kLgkm0 = 15 | (7 << 4) | (3 << 14);
// Barrier after this wave's LDS writes (loads from memory stay in flight across it).
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kLgkm0);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
constexpr float kGrow = kRescaleThreshold * kLn2;  // deferred rescale, natural units

template <int D>
struct Lds {
  static constexpr int kChunks = D / 8;               // 16-byte chunks of a 16-bit row
  static constexpr int kRowsPerDma = 512 / D;         // rows of one wave DMA (1 KiB)
  static constexpr int kTensor = kTile * D;           // elements of a K or V tile
  static constexpr int kStage = 2 * kTensor;          // K tile, V tile
  static constexpr int kOwn = kOwnStep * D;           // elements of a wave's own K or V step
};

// Keys of a 32-key block in the S^T tile: MFMA row r reads K row perm32(r), so that lane half
// h holds the sixteen consecutive keys 16 h .. 16 h + 15.
__device__ __forceinline__ int perm32(int r) {
  return (((r >> 2) & 1) << 4) | ((r >> 3) << 2) | (r & 3);
}
// Chunk c of LDS row `row` sits at c ^ swz(row): the K reads (16 rows at one chunk) and the
// transposing V reads (four rows, four chunks) hit every bank once a pass.
template <int kChunks>
__device__ __forceinline__ int swz(int row) {
  if constexpr (kChunks == 16)
    return ((row & 3) << 2) | ((row >> 2) & 1) | (((row >> 4) & 1) << 1);
  else
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 1) | (((row >> 4) & 1) << 1);
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x = min(x, __shfl_xor(x, off));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// A query row: its sequence's position (keys - 1; -1 without a query or keys) and q / out row.
struct Row {
  int pos, token;
};
__device__ __forceinline__ Row row_of(const SharedParams& p, int seq) {
  const SeqBounds bq = seq_bounds(p.cu_q, seq, p.total_q);
  const int cap = p.max_blocks << p.block_shift;
  const int lk = min(max(p.seqused_k[seq], 0), cap);
  return Row{bq.len == 1 ? lk - 1 : -1, bq.start};
}
__device__ __forceinline__ int first_key(const SharedParams& p, int pos) {
  return p.window_left >= 0 ? max(0, pos - p.window_left) : 0;
}

// Table entry of key k0 (wave-uniform), by a scalar load: a load through the vector memory
// counter would have to wait for the K and V rows in flight before it.
__device__ __forceinline__ int page_at(const int32_t* table, int i, int entries) {
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  return ((scalar_ptr)(uintptr_t)table)[min(i, entries - 1)];
}

template <int D, typename Tag, typename Rel, int Eb>
__global__ __launch_bounds__(kThreads, 2) void decode_shared_kernel(SharedParams p) {
  using E = Elem<Tag>;
  using L = Lds<D>;
  constexpr int kKSteps = D / 16, kDBlocks = D / 32;
  __shared__ __align__(1024) uint16_t stages[2 * L::kStage];
  __shared__ float merge_m[kWaves][16], merge_l[kWaves][16];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int G = p.group;

  // ---- which piece of work ------------------------------------------------------------------
  // Prefix workgroups first: those of one (kv head, chunk) sit on one XCD (workgroup i runs on
  // XCD i % 8), whose L2 then serves the chunk's K and V to all their rows.
  const bool prefix = (int)blockIdx.x < p.prefix_blocks;
  int kvh, part, seq = 0, row0 = 0, key_beg, key_end;
  if (prefix) {
    const int at = blockIdx.x >> 3;
    const int pair = (at / p.row_tiles) * 8 + (blockIdx.x & 7);
    if (pair >= p.kv_heads * p.prefix_chunks) return;
    kvh = pair % p.kv_heads;
    part = pair / p.kv_heads;
    row0 = at % p.row_tiles * kRows;
    key_beg = part * p.chunk_keys;
    key_end = min(key_beg + p.chunk_keys, p.prefix_keys);
  } else {
    const int at = blockIdx.x - p.prefix_blocks;
    kvh = at % p.kv_heads;
    seq = at / p.kv_heads % p.batch;
    const int chunk = at / p.kv_heads / p.batch;
    part = p.prefix_chunks + chunk;
    key_beg = p.prefix_keys + chunk * p.own_keys;
    key_end = key_beg + p.own_keys;
  }

  // ---- this lane's row, and the keys that the workgroup's rows see ----------------------------
  const int r = prefix ? row0 + 32 * wave + col : col;
  const int row_seq = prefix ? r / G : seq;
  const int g = prefix ? r - row_seq * G : r;
  bool ok = prefix ? row_seq < p.batch : r < G;
  const Row mine = row_of(p, ok ? row_seq : 0);
  const int pos = ok ? mine.pos : -1;
  ok = pos >= 0;
  const int head = kvh * G + g;
  const int lo = first_key(p, pos);
  // over the rows of this wave that have keys
  const int pos_min = wave_min(ok ? pos : INT32_MAX), pos_max = wave_max(pos);
  const int lo_min = wave_min(ok ? lo : INT32_MAX), lo_max = wave_max(ok ? lo : 0);
  int all_lo = lo_min, all_pos = pos_max;
  if (prefix) {  // over all waves' rows
    __shared__ int range[2][kWaves];
    if (lane == 0) {
      range[0][wave] = lo_min;
      range[1][wave] = pos_max;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      all_lo = min(all_lo, range[0][w]);
      all_pos = max(all_pos, range[1][w]);
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_pos = __builtin_amdgcn_readfirstlane(all_pos);
  }
  key_beg = max(key_beg, all_lo);
  key_end = min(key_end, all_pos + 1);
  if (key_beg >= key_end) return;

  // ---- Q (B operand) --------------------------------------------------------------------------
  u32x4_t qf[kKSteps];
  {
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t)mine.token * p.q_st +
                          (int64_t)head * p.q_sh + 8 * half;
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk)
      qf[kk] = ok ? ld_global_16(src + 16 * kk) : u32x4_t{0u, 0u, 0u, 0u};
  }

  float m_run = -INFINITY, l_run = 0.f;  // m alike in both halves, l over this half's keys
  f32x16_t o[kDBlocks];
#pragma unroll
  for (int db = 0; db < kDBlocks; ++db) o[db] = f32x16_t{};

  // ---- bias -------------------------------------------------------------------------------------
  // The 16 keys of a lane in a 32-key block have 16 consecutive distances dtop - e, contiguous in
  // the row's bias.  One resource covers the bias of all rows; 16-bit types are read as the nine
  // dwords around them and shifted.  A wave with a window that would start before the resource or
  // end past it takes one load per element.
  const rsrc_t rrel = make_rsrc(p.rel, (uint32_t)p.rel_span * Rel::kBytes);
  const int rel_row = (int)(mine.token * p.rel_st + head * p.rel_sh);
  const int rel_odd = Rel::kBytes == 2 ? (int)(reinterpret_cast<uintptr_t>(p.rel) >> 1) & 1 : 0;
  auto bias16 = [&](int dtop, float* bias) {
    constexpr int kSpan = Rel::kBytes == 2 ? 18 : 16;
    const bool any = ok && dtop >= 0 && dtop - 15 < p.rel_extent;
    const int low = rel_row + dtop - 15;
    const int start = Rel::kBytes == 2 ? low - ((low + rel_odd) & 1) : low;
    if (wave_any(any && (start < 0 || start + kSpan > (int)p.rel_span))) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        bias[e] = Rel::load(rrel, any && (uint32_t)(dtop - e) < (uint32_t)p.rel_extent
                                      ? (uint32_t)(rel_row + dtop - e) * Rel::kBytes
                                      : kOutOfRange);
      return;
    }
    const uint32_t off = any ? (uint32_t)start * Rel::kBytes : kOutOfRange;
    if constexpr (Rel::kBytes == 4) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const u32x4_t w = buf_load_16(rrel, off + 16 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[15 - 4 * c - j] = __uint_as_float(w[j]);
      }
    } else {
      const u32x4_t w0 = buf_load_16(rrel, off), w1 = buf_load_16(rrel, off + 16);
      const uint32_t w[9] = {w0[0], w0[1], w0[2], w0[3], w1[0],
                             w1[1], w1[2], w1[3], buf_load_4(rrel, off + 32)};
      const uint32_t sh = 16u * (uint32_t)(low - start);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t pr = __builtin_amdgcn_alignbit(w[k + 1], w[k], sh);
        bias[15 - 2 * k] = Rel::lo(pr);
        bias[14 - 2 * k] = Rel::hi(pr);
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      bias[e] = (uint32_t)(dtop - e) < (uint32_t)p.rel_extent ? bias[e] : 0.f;
  };

  const float c2 = p.scale * kLog2e;
  const int tr_i = lane & 15;
  const int tr_row = tr_i >> 2, tr_col = 16 * ((lane >> 4) & 1) + 4 * (tr_i & 3);

  // ---- one tile of 32 * nb keys from kb on, K rows at kl, V rows at vl ----------------------------
  auto compute = [&](auto nb, int kb, const uint16_t* kl, const uint16_t* vl) {
    constexpr int kNb = decltype(nb)::value;
    const int klast = kb + 32 * kNb - 1;
    const bool masked = klast > pos_min || kb < lo_max;
    const bool biased = p.rel_extent > 0 && pos_max >= kb && pos_min - klast < p.rel_extent;
    f32x16_t s[kNb];
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int blk = 0; blk < kNb; ++blk) {
      s[blk] = f32x16_t{};
      const int row = 32 * blk + perm32(col);
      const int sw = swz<L::kChunks>(row);
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk)
        s[blk] = E::mfma32(
            *reinterpret_cast<const u32x4_t*>(kl + row * D + 8 * ((2 * kk + half) ^ sw)), qf[kk],
            s[blk]);
    }
    // four fragment reads in flight ahead of the products
    constexpr int kReads = kNb * kKSteps, kAhead = 4;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < kReads - kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
    __builtin_amdgcn_s_setprio(0);
    auto read_vt = [&](int db, int t) -> u32x4_t {
      u32x2_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 32 * (t >> 1) + 16 * half + 8 * (t & 1) + 4 * i + tr_row;
        const int c = 32 * db + tr_col;
        const uint16_t* src = vl + row * D + 8 * ((c >> 3) ^ swz<L::kChunks>(row)) + (c & 7);
        w[i] = __builtin_bit_cast(u32x2_t,
                                  __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      (__attribute__((address_space(3))) s16x4_t*)src));
      }
      return u32x4_t{w[0][0], w[0][1], w[1][0], w[1][1]};
    };
    u32x4_t vfr[kDBlocks];
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db) vfr[db] = read_vt(db, 0);

    float mx = -INFINITY;
    if (masked || biased) {
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk) {
        const int k0 = kb + 32 * blk + 16 * half;  // the lane's first key
        float bias[16];
        if (biased) bias16(pos - k0, bias);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float y = s[blk][e] * p.scale;
          if (biased) y += bias[e];
          if (masked) y = k0 + e >= lo && k0 + e <= pos ? y : -INFINITY;
          s[blk][e] = y;
          mx = fmaxf(mx, y);
        }
      }
    } else {
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[blk][e]);
      mx *= p.scale;
    }
    mx = max_xor32(mx);
    const bool grow = mx > m_run + kGrow;
    if (wave_any(grow)) {
      const float m_new = grow ? mx : m_run;
      const float a = grow ? fast_exp2((m_run - m_new) * kLog2e) : 1.f;
      l_run *= a;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] *= a;
      m_run = m_new;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    float mul = c2, add = -m_use * kLog2e;
    if (masked || biased) {
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[blk][e] -= m_use;
      mul = kLog2e;
      add = 0.f;
    }
    auto make_p = [&](int t) -> u32x4_t {
      float pv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = fast_exp2(fmaf(s[t >> 1][8 * (t & 1) + e], mul, add));
        l_run += pv[e];
      }
      return u32x4_t{E::pack2(pv[0], pv[1]), E::pack2(pv[2], pv[3]), E::pack2(pv[4], pv[5]),
                     E::pack2(pv[6], pv[7])};
    };
    u32x4_t pcur = make_p(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < 2 * kNb; ++t) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db) {
        o[db] = E::mfma32(vfr[db], pcur, o[db]);
        if (t + 1 < 2 * kNb) vfr[db] = read_vt(db, t + 1);
      }
      if (t + 1 < 2 * kNb) pcur = make_p(t + 1);
    }
    // each product followed by the two reads of the next block's fragment and a share of its
    // exponentials (about 28 vector instructions over the products of a block)
#pragma unroll
    for (int t = 0; t < 2 * kNb - 1; ++t) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        __builtin_amdgcn_sched_group_barrier(0x402, 28 / kDBlocks, 1);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kDBlocks, 1);
    __builtin_amdgcn_s_setprio(0);
  };

  // ---- K / V rows to LDS ----------------------------------------------------------------------
  // 32 rows of one tensor at a time, in groups of rows that lie in one block (blocks hold eight
  // or more, or the rows of one load where that is more).  The groups' table entries are read
  // ahead of their rows.
  const int bmask = (1 << p.block_shift) - 1;
  const int32_t* const table =
      prefix ? p.prefix_table : p.block_table + (int64_t)seq * p.bt_stride;
  const int entries = prefix ? p.prefix_entries : (pos_max >> p.block_shift) + 1;
  constexpr int kLoadRows = 1024 / (D * Eb);  // rows of one wave load or DMA
  constexpr int kLoads32 = 32 / kLoadRows;
  constexpr int kGroupRows = kLoadRows > 8 ? kLoadRows : 8;
  constexpr int kGroups = 32 / kGroupRows, kPerGroup = kGroupRows / kLoadRows;
  constexpr int kLpr = D * Eb / 16;           // lanes per row
  const int ld_row = lane / kLpr, ld_chunk = lane % kLpr;
  struct Pages {
    int ent[kGroups];
  };
  auto pages_of = [&](int k0) {
    Pages pg;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      pg.ent[i] = page_at(table, (k0 + kGroupRows * i) >> p.block_shift, entries);
    return pg;
  };
  // One tensor's rows: pool base of the kv head, bytes between blocks and rows, LDS byte offset
  // of a lane in each load (row times pitch, and the chunk's place).
  struct Tensor {
    const char* pool;
    int64_t block;
    uint32_t row;
  };
  auto tensor = [&](bool is_v) {
    return Tensor{static_cast<const char*>(is_v ? p.v : p.k) +
                      (int64_t)kvh * (is_v ? p.v_sh : p.k_sh) * Eb,
                  (is_v ? p.v_sblk : p.k_sblk) * Eb, (uint32_t)(is_v ? p.v_st : p.k_st) * Eb};
  };
  // Resource over the group's rows [k0, min(k0 + kGroupRows, stop)): what lies past it, and a
  // whole group whose entry lies outside the pool, reads as zero.
  auto group_rsrc = [&](const Tensor& t, int ent, int k0, int stop) {
    const int n = min(kGroupRows, stop - k0);
    const bool good = (unsigned)ent < (unsigned)p.num_blocks && n > 0;
    const uint32_t at = good ? (uint32_t)ent : 0u;
    const char* base = t.pool + (int64_t)at * t.block + (uint32_t)(k0 & bmask) * t.row;
    return make_rsrc_uniform(base, good ? (uint32_t)(n - 1) * t.row + D * Eb : 0u);
  };
  const uint32_t lds0 = lds_addr(stages);
  // 16-bit: rows k0 .. k0 + 31 by DMA to LDS rows tile_row .. of the tensor at LDS address dst
  auto dma32 = [&](const Tensor& t, const Pages& pg, int k0, int stop, int tile_row, uint32_t dst) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const rsrc_t rs = group_rsrc(t, pg.ent[i], k0 + kGroupRows * i, stop);
#pragma unroll
      for (int u = 0; u < kPerGroup; ++u) {
        const int at = kGroupRows * i + kLoadRows * u;
        const int chunk = ld_chunk ^ swz<L::kChunks>(tile_row + at + ld_row);
        dma_16_tile(rs, (uint32_t)(kLoadRows * u + ld_row) * t.row + 16u * (uint32_t)chunk,
                    dst + (uint32_t)((tile_row + at) * D * 2));
      }
    }
  };
  // e4m3: the same rows into registers, and from there to LDS in the 16-bit type
  auto load32 = [&](const Tensor& t, const Pages& pg, int k0, int stop, u32x4_t* reg) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const rsrc_t rs = group_rsrc(t, pg.ent[i], k0 + kGroupRows * i, stop);
#pragma unroll
      for (int u = 0; u < kPerGroup; ++u)
        reg[kPerGroup * i + u] =
            buf_load_16(rs, (uint32_t)(kLoadRows * u + ld_row) * t.row + 16u * ld_chunk);
    }
  };
  auto put32 = [&](const u32x4_t* reg, int tile_row, uint16_t* dst) {
#pragma unroll
    for (int u = 0; u < kLoads32; ++u) {
      const int row = tile_row + kLoadRows * u + ld_row;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a = reg[u][2 * h], b = reg[u][2 * h + 1];
        *reinterpret_cast<u32x4_t*>(dst + row * D +
                                    8 * ((2 * ld_chunk + h) ^ swz<L::kChunks>(row))) =
            u32x4_t{E::template fp8x2<false>(a), E::template fp8x2<true>(a),
                    E::template fp8x2<false>(b), E::template fp8x2<true>(b)};
      }
    }
  };

  // Row of the workspace of this lane's query head in this workgroup's part.
  const int64_t rows_all = (int64_t)p.batch * p.n_heads;
  if (prefix) {
    // waves 0, 1 bring K, waves 2, 3 V; 32 rows each
    const bool is_v = wave >= 2;
    const int my_row = 32 * (wave & 1);
    const Tensor mine_kv = tensor(is_v);
    const int kt0 = key_beg / kTile, kt1 = (key_end + kTile - 1) / kTile;
    auto run_tile = [&](int kt, const uint16_t* stage) {
      const int kb = kt * kTile;
      if (kb <= pos_max && kb + kTile > lo_min)
        compute(std::integral_constant<int, 2>{}, kb, stage, stage + L::kTensor);
    };
    Pages pg = pages_of(kt0 * kTile + my_row);
    if constexpr (Eb == 2) {
      auto fetch = [&](int kt, int stage) {
        dma32(mine_kv, pg, kt * kTile + my_row, p.prefix_keys, my_row,
              lds0 + (uint32_t)(stage * L::kStage + (is_v ? L::kTensor : 0)) * 2);
        pg = pages_of((kt + 1) * kTile + my_row);
      };
      fetch(kt0, 0);
      for (int kt = kt0; kt < kt1; ++kt) {
        const int cur = (kt - kt0) & 1;
        __builtin_amdgcn_s_waitcnt(kVm0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + 1 < kt1) fetch(kt + 1, cur ^ 1);
        run_tile(kt, stages + cur * L::kStage);
      }
    } else {
      u32x4_t reg[kLoads32];
      auto fetch = [&](int kt) {
        load32(mine_kv, pg, kt * kTile + my_row, p.prefix_keys, reg);
        pg = pages_of((kt + 1) * kTile + my_row);
      };
      fetch(kt0);
      for (int kt = kt0; kt < kt1; ++kt) {
        uint16_t* stage = stages + ((kt - kt0) & 1) * L::kStage;
        put32(reg, my_row, stage + (is_v ? L::kTensor : 0));
        if (kt + 1 < kt1) fetch(kt + 1);
        lds_barrier();
        run_tile(kt, stage);
      }
    }
    const float l = add_xor32(l_run);
    // rows that see none of this part leave none
    if (ok && lo < key_end && pos >= key_beg) {
      const int64_t at = part * rows_all + (int64_t)row_seq * p.n_heads + head;
      float* dst = p.part_o + at * D + 4 * half;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4_t*>(dst + 32 * db + 8 * i) =
              f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
      if (half == 0) p.part_ml[at] = float2{m_run, l};
    }
    return;
  }

  // ---- own keys ---------------------------------------------------------------------------------
  uint16_t* const kown = stages + wave * 2 * L::kOwn;
  uint16_t* const vown = kown + L::kOwn;
  const Tensor tk = tensor(false), tv = tensor(true);
  const int s0 = (key_beg & ~(kOwnStep - 1)) + kOwnStep * wave;
  Pages pg = pages_of(s0);
  for (int k0 = s0; k0 < key_end; k0 += kOwnStep * kWaves) {
    if constexpr (Eb == 2) {
      const uint32_t dst = lds0 + (uint32_t)(wave * 2 * L::kOwn) * 2;
      dma32(tk, pg, k0, key_end, 0, dst);
      dma32(tv, pg, k0, key_end, 0, dst + L::kOwn * 2);
      pg = pages_of(k0 + kOwnStep * kWaves);
      __builtin_amdgcn_s_waitcnt(kVm0);
      asm volatile("" ::: "memory");
    } else {
      u32x4_t kr[kLoads32], vr[kLoads32];
      load32(tk, pg, k0, key_end, kr);
      load32(tv, pg, k0, key_end, vr);
      pg = pages_of(k0 + kOwnStep * kWaves);
      put32(kr, 0, kown);
      put32(vr, 0, vown);
    }
    wave_lds_sync();
    compute(std::integral_constant<int, 1>{}, k0, kown, vown);
    wave_lds_sync();  // the step's reads come before the next step's rows
    if constexpr (Eb == 2) __builtin_amdgcn_s_waitcnt(kLgkm0);
  }
  // the waves' sums meet: each leaves its O [head][D] in its own rows
  static_assert(16 * D * 4 <= 2 * L::kOwn * 2, "a wave's O fits its rows");
  const float l_tot = add_xor32(l_run);
  float* const left = reinterpret_cast<float*>(kown);
  if (col < G && col < 16) {
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4_t*>(left + col * D + 32 * db + 8 * i + 4 * half) =
            f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
    if (half == 0) {
      merge_m[wave][col] = m_run;
      merge_l[wave][col] = l_tot;
    }
  }
  __syncthreads();
  constexpr int kRowChunks = D / 4;
  for (int c = tid; c < G * kRowChunks; c += kThreads) {
    const int h = c / kRowChunks, d = 4 * (c % kRowChunks);
    float m = merge_m[0][h];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, merge_m[w][h]);
    const float mu = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4_t acc{};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float a = fast_exp2((merge_m[w][h] - mu) * kLog2e);
      l += a * merge_l[w][h];
      acc += a * *reinterpret_cast<const f32x4_t*>(
                     reinterpret_cast<const float*>(stages + w * 2 * L::kOwn) + h * D + d);
    }
    const int64_t at = part * rows_all + (int64_t)seq * p.n_heads + kvh * G + h;
    *reinterpret_cast<f32x4_t*>(p.part_o + at * D + d) = acc;
    if (d == 0) p.part_ml[at] = float2{m, l};
  }
}

// Merge of a query head's parts: a workgroup per (sequence, head), teams of D / 4 lanes over the
// parts, then in LDS; the parts meet in the same order whatever the other sequences hold.
template <int D, typename Tag>
__global__ __launch_bounds__(kThreads) void decode_shared_merge_kernel(SharedParams p) {
  using E = Elem<Tag>;
  constexpr int kTeam = D / 4, kTeams = kThreads / kTeam;
  __shared__ f32x4_t part_o[kTeams][kTeam];
  __shared__ float part_m[kTeams], part_l[kTeams];
  const int seq = blockIdx.x / p.n_heads, head = blockIdx.x - seq * p.n_heads;
  const int c = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
  const SeqBounds bq = seq_bounds(p.cu_q, seq, p.total_q);
  if (bq.len != 1) {
    // not one query token: its rows, if any, get out = 0 and lse = -inf
    for (int i = team; i < bq.len; i += kTeams) {
      uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)(bq.start + i) * p.o_st +
                      (int64_t)head * p.o_sh + 4 * c;
      *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{0u, 0u};
      if (p.lse != nullptr && c == 0) p.lse[(int64_t)head * p.lse_sh + bq.start + i] = -INFINITY;
    }
    return;
  }
  const int pos = row_of(p, seq).pos, lo = first_key(p, pos);
  // parts of the prefix, then of the sequence's own keys
  const int pend = min(pos + 1, p.prefix_keys);
  const int p0 = lo / p.chunk_keys;
  const int np = lo < pend ? (pend - 1) / p.chunk_keys - p0 + 1 : 0;
  const int obeg = max(lo, p.prefix_keys) - p.prefix_keys, oend = pos + 1 - p.prefix_keys;
  const int o0 = obeg / p.own_keys;
  const int no = obeg < oend ? min((oend - 1) / p.own_keys, p.own_chunks - 1) - o0 + 1 : 0;
  const int64_t rows_all = (int64_t)p.batch * p.n_heads;
  float m = -INFINITY, l = 0.f;
  f32x4_t acc{};
#pragma unroll 4
  for (int i = team; i < np + no; i += kTeams) {
    const int part = i < np ? p0 + i : p.prefix_chunks + o0 + i - np;
    const int64_t at = part * rows_all + blockIdx.x;
    const float2 x = p.part_ml[at];
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p.part_o + at * D + 4 * c);
    const float mn = fmaxf(m, x.x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float a = fast_exp2((m - mu) * kLog2e), b = fast_exp2((x.x - mu) * kLog2e);
    l = l * a + b * x.y;
    acc = acc * a + b * v;
    m = mn;
  }
  part_o[team][c] = acc;
  if (c == 0) {
    part_m[team] = m;
    part_l[team] = l;
  }
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int t = 1; t < kTeams; ++t) m = fmaxf(m, part_m[t]);
  const float mu = m == -INFINITY ? 0.f : m;
  l = 0.f;
  acc = f32x4_t{};
#pragma unroll
  for (int t = 0; t < kTeams; ++t) {
    const float a = fast_exp2((part_m[t] - mu) * kLog2e);
    l += a * part_l[t];
    acc += a * part_o[t][c];
  }
  const float inv = l > 0.f ? p.v_scale / l : 0.f;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)bq.start * p.o_st +
                  (int64_t)head * p.o_sh + 4 * c;
  // a row without keys is zero whatever its parts hold
  const bool some = l > 0.f || l != l;
  *reinterpret_cast<u32x2_t*>(dst) =
      some ? u32x2_t{E::pack2(acc[0] * inv, acc[1] * inv), E::pack2(acc[2] * inv, acc[3] * inv)}
           : u32x2_t{0u, 0u};
  if (p.lse != nullptr && c == 0)
    p.lse[(int64_t)head * p.lse_sh + bq.start] = some ? m + __log2f(l) * kLn2 : -INFINITY;
}

template <int D, typename Tag, typename Rel>
hipError_t launch_rel(const SharedParams& p, hipStream_t stream) {
  const int64_t blocks =
      (int64_t)p.prefix_blocks + (int64_t)p.batch * p.kv_heads * p.own_chunks;
  if (blocks > 0) {
    if (p.kv_fp8)
      hipLaunchKernelGGL((decode_shared_kernel<D, Tag, Rel, 1>), dim3((unsigned)blocks),
                         dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((decode_shared_kernel<D, Tag, Rel, 2>), dim3((unsigned)blocks),
                         dim3(kThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((decode_shared_merge_kernel<D, Tag>),
                     dim3((unsigned)((int64_t)p.batch * p.n_heads)), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

template <int D, typename Tag>
hipError_t launch_tag(const SharedParams& p, hipStream_t stream) {
  switch (p.rel_dtype) {
    case 0: return launch_rel<D, Tag, RelBf16>(p, stream);
    case 1: return launch_rel<D, Tag, RelF16>(p, stream);
    default: return launch_rel<D, Tag, RelF32>(p, stream);
  }
}

}  // namespace

hipError_t launch_decode_shared(const SharedParams& p, int head_dim, int qkv_dtype,
                                hipStream_t stream) {
  if (p.batch <= 0) return hipSuccess;
  if (head_dim == 128)
    return qkv_dtype == 0 ? launch_tag<128, Bf16Tag>(p, stream) : launch_tag<128, F16Tag>(p, stream);
  return qkv_dtype == 0 ? launch_tag<64, Bf16Tag>(p, stream) : launch_tag<64, F16Tag>(p, stream);
}

}  // namespace ifa4
