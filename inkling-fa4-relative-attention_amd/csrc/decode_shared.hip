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
// One launch of workgroups of 4 waves, two on a CU, each with a piece of the prefix, pieces of own
// keys, or both; then the merge:
//   prefix  128 rows (32 a wave; row = sequence * group + head of the kv head) x a chunk of
//           64-key tiles, in two LDS stages: the DMA of the next tile (16-bit cache), or its
//           loads into registers (e4m3, converted on the way to LDS), run under the products
//           of the current one;
//   own     one (sequence, kv head) x a chunk of its own keys: the waves take 32-key steps in
//           turn, each in its own quarter of the LDS, the group's heads in the columns of the
//           product; the waves' sums meet in LDS.
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
//
// Bounds.  The tiles of a long prefix are bound by what two waves of a SIMD issue: a tile takes 4000
// cycles for two workgroups of a CU, of which the matrix products are 2048 (32 products of 32 cycles
// a wave) and the vector instructions (180, 32 of them exp2) nearly all the rest, with little
// overlap; 5000 where it meets a bias.  One common barrier for eight waves with the K and V of both
// halves cost 4700 to 5400.  Measured, bf16, d 128, Hq 8 / Hkv 2, bias extent 1024: 256 sequences
// behind 32768 keys 57 us traced (a whole call 59, 580 TFLOP/s), the matrix cores busy for 0.35 of
// it: by the plan's cycles 80000 of a workgroup's 98000 are its 20 tiles and 13000 its start and
// exit, and 96 of the 512 workgroups hold own keys only, whose rounds wait for their rows.  The merge
// takes 9 us, of which 4 are a launch over nothing and the rest the 28 MB of parts at 5.6 TB/s.  64
// sequences behind 16384 keys 21 + 7 us: there a workgroup's four tiles take less than its first
// rows, its parts and its launch.
#include <type_traits>

#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // rows of a prefix piece
constexpr int kMergeThreads = 256;
constexpr int kTile = 64;           // keys of a prefix tile
constexpr int kOwnStep = 32;        // keys of a wave's step over a sequence's own keys
static_assert(kSharedTile == kTile && kSharedRows == kRows, "the host plans with these");
static_assert(kSharedOwnRound == kOwnStep * kWaves, "the host plans with these");

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

// Least x of the wave (VALU lane exchanges: through LDS the four reductions of a workgroup's start
// took over a microsecond).
template <int kCtrl>
__device__ __forceinline__ int min_dpp(int x) {
  return min(x, __builtin_amdgcn_mov_dpp(x, kCtrl, 0xf, 0xf, false));
}
__device__ __forceinline__ int wave_min(int x) {
  x = min_dpp<0xb1>(x);   // lane ^ 1
  x = min_dpp<0x4e>(x);   // lane ^ 2
  x = min_dpp<0x141>(x);  // the other quad of eight
  x = min_dpp<0x140>(x);  // the other eight of sixteen
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = min((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = min((int)r[0], (int)r[1]);
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }
template <int kCtrl>
__device__ __forceinline__ float max_dpp(float x) {
  const int y = __builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xf, 0xf, false);
  return fmaxf(x, __int_as_float(y));
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4e>(max_dpp<0xb1>(x))));
  const int i = __float_as_int(x);
  auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  x = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
  const int j = __float_as_int(x);
  r = __builtin_amdgcn_permlane32_swap(j, j, false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}

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

struct Whole {};  // every row of a group is there

// Table entry of key k0 (wave-uniform), by a scalar load: a load through the vector memory
// counter would have to wait for the K and V rows in flight before it.
__device__ __forceinline__ int page_at(const int32_t* table, int i) {
  typedef const __attribute__((address_space(4))) char* scalar_ptr;
  typedef const __attribute__((address_space(4))) int32_t* entry_ptr;
  return *(entry_ptr)((scalar_ptr)(uintptr_t)table + 4u * (uint32_t)i);  // an offset of 32 bits
}

template <int D, typename Tag, typename Rel, int Eb>
__global__ __launch_bounds__(kThreads, 2) void decode_shared_kernel(SharedParams call) {
  using E = Elem<Tag>;
  using L = Lds<D>;
  constexpr int kKSteps = D / 16, kDBlocks = D / 32;
  __shared__ __align__(1024) uint16_t stages[2 * L::kStage];
  __shared__ float merge_m[kWaves][32], merge_l[kWaves][32];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, col = lane & 31, half = lane >> 5;

  // ---- this lane's row: set for the prefix, then for each piece of own keys ----------------------
  int pos = -1, lo = 0, head = 0, rel_row = 0;  // key position, first key seen, query head, bias row
  bool ok = false;                              // the lane has a query with keys
  int pos_min = 0, pos_max = -1, lo_min = 0, lo_max = 0;  // over the wave's rows that have keys
  u32x4_t qf[kKSteps];                          // Q (B operand)
  float m_run = -INFINITY, l_run = 0.f;         // m alike in both halves, l over this half's keys
  f32x16_t o[kDBlocks];
  auto load_q = [&](const SharedParams& p, int token, int h) {
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t)token * p.q_st +
                          (int64_t)h * p.q_sh + 8 * half;
#pragma unroll
    for (int kk = 0; kk < kKSteps; ++kk) qf[kk] = ld_global_16(src + 16 * kk);
  };
  // `there`: the lane has a row; head set, its Q on the way for token `guess`
  auto set_row = [&](const SharedParams& p, const Row& row, bool there, int guess) {
    pos = there ? row.pos : -1;
    ok = pos >= 0;
    lo = first_key(p, pos);
    pos_min = wave_min(ok ? pos : INT32_MAX);  // lo grows with pos
    pos_max = wave_max(pos);
    lo_min = first_key(p, pos_min);
    lo_max = first_key(p, pos_max);
    rel_row = (int)(row.token * p.rel_st + head * p.rel_sh);
    // cu_seqlens_q is arange in every call that keeps the contract: q is read without waiting for
    // it (total_q == batch), and again where it is not
    if (wave_any(ok && row.token != guess)) load_q(p, ok ? row.token : 0, head);
    m_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int db = 0; db < kDBlocks; ++db) o[db] = f32x16_t{};
  };

  // ---- K / V rows to LDS ----------------------------------------------------------------------
  // 32 rows of one tensor at a time, in groups of rows that lie in one block (blocks hold eight
  // or more, or the rows of one load where that is more).  The groups' table entries are read
  // ahead of their rows.
  constexpr int kLoadRows = 1024 / (D * Eb);  // rows of one wave load or DMA
  constexpr int kLoads32 = 32 / kLoadRows;
  constexpr int kGroupRows = kLoadRows > 8 ? kLoadRows : 8;
  constexpr int kGroups = 32 / kGroupRows, kPerGroup = kGroupRows / kLoadRows;
  constexpr int kLpr = D * Eb / 16;           // lanes per row
  const int ld_row = lane / kLpr, ld_chunk = lane % kLpr;
  struct Pages {
    int ent[kGroups];
  };
  auto pages_of = [&](const SharedParams& p, const int32_t* table, int entries, int k0) {
    Pages pg;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      pg.ent[i] = page_at(table, min((k0 + kGroupRows * i) >> p.block_shift, entries - 1));
    return pg;
  };
  // One tensor's rows: pool base of the kv head, bytes between blocks and rows, LDS byte offset
  // of a lane in each load (row times pitch, and the chunk's place).
  struct Tensor {
    const char* pool;
    int64_t block;
    uint32_t row;
  };
  auto tensor = [&](const SharedParams& p, int kvh, bool is_v) {
    return Tensor{static_cast<const char*>(is_v ? p.v : p.k) +
                      (int64_t)kvh * (is_v ? p.v_sh : p.k_sh) * Eb,
                  (is_v ? p.v_sblk : p.k_sblk) * Eb, (uint32_t)(is_v ? p.v_st : p.k_st) * Eb};
  };
  // Resource over the group's rows [k0, min(k0 + kGroupRows, stop)): what lies past it, and a
  // whole group whose entry lies outside the pool, reads as zero.
  auto group_rsrc = [&](const SharedParams& p, const Tensor& t, int ent, int k0, auto stop) {
    uint32_t seen = (uint32_t)(kGroupRows - 1) * t.row + D * Eb;
    if constexpr (!std::is_same<decltype(stop), Whole>::value) {
      const int n = min(kGroupRows, stop - k0);
      seen = n > 0 ? (uint32_t)(n - 1) * t.row + D * Eb : 0u;
    }
    seen = (uint32_t)ent < (uint32_t)p.num_blocks ? seen : 0u;
    // (no address is formed from the base of an empty resource)
    const uint64_t base = reinterpret_cast<uint64_t>(t.pool) + (uint64_t)(uint32_t)ent * (uint64_t)t.block +
                          (uint32_t)(k0 & ((1 << p.block_shift) - 1)) * t.row;
    return make_rsrc_uniform(reinterpret_cast<const void*>(base), seen);
  };
  const uint32_t lds0 = lds_addr(stages);
  // 16-bit: rows k0 .. k0 + 31 by DMA to LDS rows tile_row .. of the tensor at LDS address dst
  auto dma32 = [&](const SharedParams& p, const Tensor& t, const Pages& pg, int k0, auto stop, int tile_row,
                   uint32_t dst) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const rsrc_t rs = group_rsrc(p, t, pg.ent[i], k0 + kGroupRows * i, stop);
#pragma unroll
      for (int u = 0; u < kPerGroup; ++u) {
        const int at = kGroupRows * i + kLoadRows * u;
        // (tile_row is a multiple of 32, which swz does not look at)
        const int chunk = ld_chunk ^ swz<L::kChunks>(at + ld_row);
        dma_16_tile(rs, (uint32_t)(kLoadRows * u + ld_row) * t.row + 16u * (uint32_t)chunk,
                    dst + (uint32_t)((tile_row + at) * D * 2));
      }
    }
  };
  // e4m3: the same rows into registers, and from there to LDS in the 16-bit type
  auto load32 = [&](const SharedParams& p, const Tensor& t, const Pages& pg, int k0, auto stop, u32x4_t* reg) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const rsrc_t rs = group_rsrc(p, t, pg.ent[i], k0 + kGroupRows * i, stop);
#pragma unroll
      for (int u = 0; u < kPerGroup; ++u)
        reg[kPerGroup * i + u] =
            buf_load_16(rs, (uint32_t)(kLoadRows * u + ld_row) * t.row + 16u * ld_chunk);
    }
  };
  auto put32 = [&](const u32x4_t* reg, int tile_row, uint16_t* dst) {
    int ln = lane;
    asm volatile("" : "+v"(ln));  // addresses computed here: kept across the tiles they would spill
#pragma unroll
    for (int u = 0; u < kLoads32; ++u) {
      const int row = tile_row + kLoadRows * u + ln / kLpr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t a = reg[u][2 * h], b = reg[u][2 * h + 1];
        *reinterpret_cast<u32x4_t*>(dst + row * D +
                                    8 * ((2 * (ln % kLpr) + h) ^ swz<L::kChunks>(row))) =
            u32x4_t{E::template fp8x2<false>(a), E::template fp8x2<true>(a),
                    E::template fp8x2<false>(b), E::template fp8x2<true>(b)};
      }
    }
  };

  // ---- bias -------------------------------------------------------------------------------------
  // The 16 keys of a lane in a 32-key block have 16 consecutive distances dtop - e, contiguous in
  // the row's bias.  One resource covers the bias of all rows; 16-bit types are read as the nine
  // dwords around them and shifted.  A wave with a window that would start before the resource or
  // end past it takes one load per element.
  auto rel_rsrc = [&](const SharedParams& p) {
    return make_rsrc(p.rel, (uint32_t)p.rel_span * Rel::kBytes);
  };
  constexpr int kRaw = Rel::kBytes == 2 ? 9 : 16;
  struct Bias {
    uint32_t w[kRaw];
    bool slow;  // wave-uniform
  };
  auto bias_any = [&](const SharedParams& p, int dtop) { return ok && dtop >= 0 && dtop - 15 < p.rel_extent; };
  // first element of the vector loads whose lowest value is element low
  auto bias_start = [&](const SharedParams& p, int low) {
    return Rel::kBytes == 2 ? low - ((low + (int)(reinterpret_cast<uintptr_t>(p.rel) >> 1)) & 1) : low;
  };
  auto bias_issue = [&](const SharedParams& p, int dtop, Bias& b) {
    constexpr int kSpan = Rel::kBytes == 2 ? 18 : 16;
    const bool any = bias_any(p, dtop);
    const int start = bias_start(p, rel_row + dtop - 15);
    b.slow = wave_any(any && (start < 0 || start + kSpan > (int)p.rel_span));
    if (b.slow) return;
    const uint32_t off = any ? (uint32_t)start * Rel::kBytes : kOutOfRange;
    const rsrc_t rrel = rel_rsrc(p);
#pragma unroll
    for (int c = 0; c < kRaw / 4; ++c) {
      const u32x4_t w = buf_load_16(rrel, off + 16 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) b.w[4 * c + j] = w[j];
    }
    if constexpr (Rel::kBytes == 2) b.w[8] = buf_load_4(rrel, off + 32);
  };
  auto bias_finish = [&](const SharedParams& p, int dtop, const Bias& b, float* bias) {
    const bool any = bias_any(p, dtop);
    if (b.slow) {
#pragma unroll 1
      for (int e = 0; e < 16; e += 4) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = Rel::load(rel_rsrc(p), any && (uint32_t)(dtop - e - j) < (uint32_t)p.rel_extent
                                     ? (uint32_t)(rel_row + dtop - e - j) * Rel::kBytes
                                     : kOutOfRange);
#pragma unroll
        for (int i = 0; i < 16; ++i) bias[i] = (i & ~3) == e ? x[i & 3] : bias[i];
      }
      return;
    }
    if constexpr (Rel::kBytes == 4) {
#pragma unroll
      for (int k = 0; k < 16; ++k) bias[15 - k] = __uint_as_float(b.w[k]);
    } else {
      const int low = rel_row + dtop - 15;
      const uint32_t sh = 16u * (uint32_t)(low - bias_start(p, low));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t pr = __builtin_amdgcn_alignbit(b.w[k + 1], b.w[k], sh);
        bias[15 - 2 * k] = Rel::lo(pr);
        bias[14 - 2 * k] = Rel::hi(pr);
      }
    }
    if (!wave_all(!any || (dtop - 15 >= 0 && dtop < p.rel_extent))) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        bias[e] = (uint32_t)(dtop - e) < (uint32_t)p.rel_extent ? bias[e] : 0.f;
    }
  };

  const int tr_i = lane & 15;
  const int tr_row = tr_i >> 2, tr_col = 16 * ((lane >> 4) & 1) + 4 * (tr_i & 3);

  // ---- one tile of 32 * nb keys from kb on, K rows at kl, V rows at vl ----------------------------
  // next() brings the rows of the tile after it: at once, or where this tile's bias is loaded from
  // memory after that has come (loads complete in order)
  auto tile_biased = [&](const SharedParams& p, int kb, int keys) {
    return p.rel_extent > 0 && pos_max >= kb && pos_min - (kb + keys - 1) < p.rel_extent;
  };
  auto compute = [&](const SharedParams& p, auto nb, int kb, const uint16_t* kl, const uint16_t* vl, bool biased,
                     const Bias* ahead, auto next) {
    constexpr int kNb = decltype(nb)::value;
    const int klast = kb + 32 * kNb - 1;
    const bool masked = klast > pos_min || kb < lo_max;
    const int key0 = kb + 16 * half;  // the lane's first key
    if (!biased) next();
    f32x16_t s[kNb];
    // The chunk of a fragment is an XOR away from the first one's, so that one address register a
    // tensor (two for V) serves all of them: kept apart they would spill.
    const int k_at = (int)(kl - stages) + perm32(col) * D + 8 * (half ^ swz<L::kChunks>(perm32(col)));
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int blk = 0; blk < kNb; ++blk) {
      s[blk] = f32x16_t{};
#pragma unroll
      for (int kk = 0; kk < kKSteps; ++kk)
        s[blk] = E::mfma32(
            *reinterpret_cast<const u32x4_t*>(stages + (k_at ^ (16 * kk)) + 32 * blk * D), qf[kk],
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
    int v_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * half + 4 * i + tr_row;
      v_at[i] = (int)(vl - stages) + row * D + 8 * ((tr_col >> 3) ^ swz<L::kChunks>(row)) + (tr_col & 7);
    }
    auto read_vt = [&](int db, int t) -> u32x4_t {
      u32x2_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint16_t* src = stages + (v_at[i] ^ (32 * db)) + (32 * (t >> 1) + 8 * (t & 1)) * D;
        w[i] = __builtin_bit_cast(u32x2_t,
                                  __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                      (__attribute__((address_space(3))) s16x4_t*)src));
      }
      return u32x4_t{w[0][0], w[0][1], w[1][0], w[1][1]};
    };
    // the first V fragments come under the softmax (a biased tile needs the registers)
    u32x4_t vfr[kDBlocks];
    if (!biased) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db) vfr[db] = read_vt(db, 0);
    }

    float mx = -INFINITY;
    if (biased) {
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk) {
        float bias[16];
        Bias late;
        if (ahead == nullptr) bias_issue(p, pos - key0 - 32 * blk, late);
        bias_finish(p, pos - key0 - 32 * blk, ahead != nullptr ? ahead[blk] : late, bias);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[blk][e] = fmaf(s[blk][e], p.scale, bias[e]);
      }
      next();
    } else if (masked) {
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[blk][e] *= p.scale;
    }
    if (masked) {  // visible: lo <= key <= pos
      const uint32_t from = (uint32_t)(key0 - lo), span = (uint32_t)(pos - lo);
#pragma unroll
      for (int blk = 0; blk < kNb; ++blk)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[blk][e] = from + (uint32_t)(32 * blk + e) <= span ? s[blk][e] : -INFINITY;
    }
#pragma unroll
    for (int blk = 0; blk < kNb; ++blk)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[blk][e]);
    if (!masked && !biased) mx *= p.scale;
    if (biased) {
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db) vfr[db] = read_vt(db, 0);
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
    float mul = p.scale * kLog2e, add = -m_use * kLog2e;
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

  // Each phase takes the call's fields from a copy of its own: fields of the second kept through
  // the first one's loop would spill.
  auto fields = [] {
    typedef const __attribute__((address_space(4))) uint32_t* scalar_ptr;
    auto at = (scalar_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(at));
    struct Words {
      uint32_t w[sizeof(SharedParams) / 4];
    } x;
    static_assert(sizeof(SharedParams) % 4 == 0 && std::is_trivially_copyable<SharedParams>::value, "");
#pragma unroll
    for (int i = 0; i < (int)(sizeof(SharedParams) / 4); ++i) x.w[i] = at[i];
    return __builtin_bit_cast(SharedParams, x);
  };

  // ---- the prefix ---------------------------------------------------------------------------------
  // Workgroups of one (kv head, chunk) sit on one XCD (workgroup i runs on XCD i % 8), whose L2 then
  // serves the chunk's K and V to all their rows.
  {
  const uint32_t at8 = blockIdx.x >> 3;
  const SharedParams p = fields();
  const int G = p.group;
  const int64_t rows_all = (int64_t)p.batch * p.n_heads;  // of a part
  const uint32_t group8 = p.by_tiles.div(at8);
  const uint32_t pair = group8 * 8 + (blockIdx.x & 7);
  if (blockIdx.x < (uint32_t)p.prefix_blocks && pair < (uint32_t)(p.kv_heads * p.prefix_chunks)) {
    const int part = (int)p.by_kv.div(pair);
    const int kvh = (int)pair - part * p.kv_heads;
    int key_beg = part * p.chunk_keys;
    int key_end = min(key_beg + p.chunk_keys, p.prefix_keys);
    const int r = (int)(at8 - group8 * p.row_tiles) * kRows + 32 * wave + col;
    const int seq = (int)p.by_group.div((uint32_t)r);
    const bool there = seq < p.batch;
    head = kvh * G + (there ? r - seq * G : 0);
    const Row row = row_of(p, there ? seq : 0);
    load_q(p, there ? seq : 0, head);

    // waves 0, 1 bring K, waves 2, 3 V; 32 rows each
    const bool is_v = wave >= 2;
    const int my_row = 32 * (wave & 1);
    const Tensor kv = tensor(p, kvh, is_v);
    Pages pg;
    u32x4_t reg[Eb == 1 ? kLoads32 : 1];  // e4m3: the rows of the next tile
    auto pages = [&](int kt) {
      pg = pages_of(p, p.prefix_table, p.prefix_entries, kt * kTile + my_row);
    };
    auto fetch = [&](int kt, int stage) {
      if constexpr (Eb == 2)
        dma32(p, kv, pg, kt * kTile + my_row, Whole{}, my_row,
              lds0 + (uint32_t)(stage * L::kStage + (is_v ? L::kTensor : 0)) * 2);
      else
        load32(p, kv, pg, kt * kTile + my_row, Whole{}, reg);
      pages(kt + 1);
    };
    // the first tile's rows go out ahead of everything that they do not depend on
    const bool early = Eb == 2 && p.window_left < 0;
    if (early) {
      pages(key_beg / kTile);
      fetch(key_beg / kTile, 0);
    }
    set_row(p, row, there, seq);
    if (p.window_left >= 0) {
      // a window hides most of the prefix: only the tiles that some row of the workgroup sees
      if (lane == 0) {
        merge_m[wave][0] = __int_as_float(lo_min);
        merge_l[wave][0] = __int_as_float(pos_max);
      }
      __syncthreads();
      int all_lo = lo_min, all_pos = pos_max;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        all_lo = min(all_lo, __float_as_int(merge_m[w][0]));
        all_pos = max(all_pos, __float_as_int(merge_l[w][0]));
      }
      key_beg = max(key_beg, __builtin_amdgcn_readfirstlane(all_lo));
      key_end = min(key_end, __builtin_amdgcn_readfirstlane(all_pos) + 1);
    }
    const int kt0 = key_beg / kTile, kt1 = key_beg < key_end ? (key_end + kTile - 1) / kTile : kt0;
    if (!early && kt0 < kt1) {
      pages(kt0);
      fetch(kt0, 0);
    }
    for (int kt = kt0, cur = 0; kt < kt1; ++kt, cur ^= 1) {
      const int kb = kt * kTile;
      uint16_t* const stage = stages + cur * L::kStage;
      // this wave's rows of the tile have landed (are written); then every wave's, and all are done
      // with the tile before, whose stage the next tile takes
      if constexpr (Eb == 2) {
        __builtin_amdgcn_s_waitcnt(kVm0);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      } else {
        put32(reg, my_row, stage + (is_v ? L::kTensor : 0));
        lds_barrier();
      }
      auto next = [&] {
        if (kt + 1 < kt1) fetch(kt + 1, cur ^ 1);
      };
      if (kb > pos_max || kb + kTile <= lo_min) {  // no row of this wave sees the tile
        next();
        continue;
      }
      // 16-bit biases are loaded ahead of the products (the 32 registers of an fp32 one, or those
      // beside an e4m3 tile's rows, would spill)
      constexpr bool kAhead = Rel::kBytes == 2 && Eb == 2;
      const bool biased = tile_biased(p, kb, kTile);
      Bias raw[2];
      if (kAhead && biased) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) bias_issue(p, pos - kb - 16 * half - 32 * blk, raw[blk]);
        asm volatile("" ::: "memory");
      }
      compute(p, std::integral_constant<int, 2>{}, kb, stage, stage + L::kTensor, biased,
              kAhead ? raw : nullptr, next);
    }

    // rows that see none of this part leave none
    const float l = add_xor32(l_run);
    if (ok && lo < key_end && pos >= key_beg) {
      const int64_t at = part * rows_all + (int64_t)seq * p.n_heads + head;
      float* dst = p.part_o + at * D + 4 * half;
#pragma unroll
      for (int db = 0; db < kDBlocks; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4_t*>(dst + 32 * db + 8 * i) =
              f32x4_t{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
      if (half == 0) p.part_ml[at] = float2{m_run, l};
    }
    lds_barrier();  // every wave is done with its last tile, whose stage the rows below take
  }
  }

  // ---- own keys -----------------------------------------------------------------------------------
  // The workgroups by rank, those without a prefix piece first: each of these takes own_first
  // pieces, then all take one after the other.  (Padding of the XCDs' shares makes some workgroups
  // of the prefix's range idle: the last `pad` of each eight at the range's end.)
  const SharedParams p = fields();
  const int G = p.group;
  const int64_t rows_all = (int64_t)p.batch * p.n_heads;
  uint16_t* const kown = stages + wave * 2 * L::kOwn;
  uint16_t* const vown = kown + L::kOwn;
  const int pairs = p.kv_heads * p.prefix_chunks, pad = -pairs & 7;
  const int idle = (int)gridDim.x - pairs * p.row_tiles;
  int rank = (int)blockIdx.x - p.prefix_blocks;
  if (rank < 0) {
    const uint32_t at8 = blockIdx.x >> 3, group8 = p.by_tiles.div(at8);
    const int pair = (int)group8 * 8 + (int)(blockIdx.x & 7);
    const int tile = (int)at8 - (int)group8 * p.row_tiles;
    rank = pair < pairs ? idle + pair * p.row_tiles + tile
                        : (int)gridDim.x - p.prefix_blocks + tile * pad + pair - pairs;
  }
  const int mine = rank < idle ? p.own_first : 0;
  for (int i = 0;; ++i) {
    const int piece = i < mine ? rank + i * idle
                               : p.own_first * idle + rank + (i - mine) * (int)gridDim.x;
    if (piece >= p.own_pieces) break;
    const uint32_t each = p.by_kv.div((uint32_t)piece);
    const int kvh = piece - (int)each * p.kv_heads;
    const int chunk = (int)p.by_batch.div(each);
    const int seq = (int)each - chunk * p.batch;
    const int32_t* const table = p.block_table + (int64_t)seq * p.bt_stride;
    const bool there = col < G;
    head = kvh * G + (there ? col : 0);
    // the table's entries come with the lengths
    const Tensor tk = tensor(p, kvh, false), tv = tensor(p, kvh, true);
    const Row row = row_of(p, seq);
    load_q(p, seq, head);
    int key0 = p.prefix_keys;
    Pages pg = pages_of(p, table, p.max_blocks, key0 + kOwnStep * (chunk * kWaves + wave));
    // (an empty sequence has no first key either)
    if (__builtin_amdgcn_readfirstlane(row.pos) < p.prefix_keys) continue;  // no own keys
    set_row(p, row, there, seq);
    // 32-key steps of the keys that the sequence sees of its own; the chunk's waves take every
    // kWaves * own_chunks-th
    const int key_end = pos_max + 1;
    const bool moved = lo_min > key0;  // by a window
    if (moved) key0 = lo_min & ~(kOwnStep - 1);
    if (key0 + chunk * kWaves * kOwnStep >= key_end) continue;  // none for this chunk
    const int stride = kOwnStep * kWaves * p.own_chunks;
    const int s0 = key0 + kOwnStep * (chunk * kWaves + wave);
    if (moved) pg = pages_of(p, table, p.max_blocks, s0);
    // e4m3: the next step's rows are on their way, in registers, while a step is computed (128
    // sequences behind 8192 keys 22.0 -> 21.5 us).  The twice as many of a 16-bit cache would spill
    // at d 128 (64 behind 16384 19.9 -> 24.4 us) and lose at d 64 (24.5 -> 25.3 a call): their rows go
    // to LDS by DMA ahead of each step.
    constexpr bool kFetch = Eb == 1;
    u32x4_t kr[kFetch ? kLoads32 : 1], vr[kFetch ? kLoads32 : 1];
    auto fetch = [&](int k0) {
      load32(p, tk, pg, k0, key_end, kr);
      load32(p, tv, pg, k0, key_end, vr);
      pg = pages_of(p, table, p.max_blocks, k0 + stride);
    };
    if constexpr (kFetch) {
      if (s0 < key_end) fetch(s0);
    }
    // The first step under a window begins up to 31 keys left of it.  Their weights are 0, and 0
    // times an infinite or NaN value would reach the sum: those rows of V are cleared.
    auto clear_rows = [&](uint16_t* rows, int n) {
      for (int e = 8 * lane; e < n * D; e += 8 * 64) *reinterpret_cast<u32x4_t*>(rows + e) = u32x4_t{};
    };
    for (int k0 = s0; k0 < key_end; k0 += stride) {
      const bool biased = tile_biased(p, k0, kOwnStep);
      Bias raw;
      if constexpr (kFetch) {
        put32(kr, 0, kown);
        put32(vr, 0, vown);
      }
      if (biased) bias_issue(p, pos - k0 - 16 * half, raw);
      asm volatile("" ::: "memory");
      if constexpr (kFetch) {
        if (k0 + stride < key_end) fetch(k0 + stride);
      } else {
        const uint32_t dst = lds0 + (uint32_t)(wave * 2 * L::kOwn) * 2;
        dma32(p, tk, pg, k0, key_end, 0, dst);
        dma32(p, tv, pg, k0, key_end, 0, dst + L::kOwn * 2);
        pg = pages_of(p, table, p.max_blocks, k0 + stride);
        __builtin_amdgcn_s_waitcnt(kVm0);
        asm volatile("" ::: "memory");
      }
      if (k0 < lo_min) clear_rows(vown, lo_min - k0);
      wave_lds_sync();
      compute(p, std::integral_constant<int, 1>{}, k0, kown, vown, biased, &raw, [] {});
      wave_lds_sync();  // the step's reads come before the next step's rows
      if constexpr (!kFetch) __builtin_amdgcn_s_waitcnt(kLgkm0);
    }
    // the waves' sums meet: each leaves its O [head][D] in its own rows
    static_assert(16 * D * 4 <= 2 * L::kOwn * 2, "a wave's O fits its rows");
    const float l_tot = add_xor32(l_run);
    float* const left = reinterpret_cast<float*>(kown);
    if (col < G) {
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
    lds_barrier();
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
      const int64_t at = (int64_t)(p.prefix_chunks + chunk) * rows_all +
                         (int64_t)seq * p.n_heads + kvh * G + h;
      *reinterpret_cast<f32x4_t*>(p.part_o + at * D + d) = acc;
      if (d == 0) p.part_ml[at] = float2{m, l};
    }
    lds_barrier();
  }
}

// Merge of a query head's parts, a workgroup per (sequence, head).  256 parts at a time: a thread a
// part for the weights exp(m_i - m), which go to LDS; teams of D / 4 lanes sum every kTeams-th
// part's O by them, their first kAhead rows on the way while the weights are made.  The parts meet
// in the same order whatever the other sequences hold.  Without a window nearly every part is a
// row's own, and they are read without waiting for its length (a part that is not is left out of the
// sums): one dependent memory round less.
template <int D, typename Tag>
__global__ __launch_bounds__(kMergeThreads, 8) void decode_shared_merge_kernel(SharedParams p) {
  using E = Elem<Tag>;
  constexpr int kTeam = D / 4, kTeams = kMergeThreads / kTeam, kAhead = 8;
  constexpr int kMergeWaves = kMergeThreads / 64;
  __shared__ f32x4_t part_o[kTeams][kTeam];
  __shared__ float weight[kMergeThreads], weighted[kMergeThreads], wave_m[kMergeWaves];
  __shared__ float part_l[kTeams];
  const int row = blockIdx.x;
  const int seq = (int)p.by_heads.div((uint32_t)row), head = row - seq * p.n_heads;
  const int tid = threadIdx.x, c = tid % kTeam, team = tid / kTeam;
  const int64_t rows_all = (int64_t)p.batch * p.n_heads;
  const SeqBounds bq = seq_bounds(p.cu_q, seq, p.total_q);
  const int pos = row_of(p, seq).pos, lo = first_key(p, pos);
  // part i, prefix first: read, and counted if the row has left something in it
  const bool window = p.window_left >= 0;
  const int skip = window ? (int)p.by_chunk.div((uint32_t)lo) : 0;  // parts left of the window
  const int np = min(pos + 1, p.prefix_keys) > lo
                     ? (int)p.by_chunk.div((uint32_t)(min(pos + 1, p.prefix_keys) - 1)) + 1 : 0;
  const int own0 = max(lo, p.prefix_keys) & ~(kOwnStep - 1);
  const int rounds = pos >= own0 ? (pos - own0) / (kOwnStep * kWaves) + 1 : 0;
  const int no = min(rounds, p.own_chunks);  // chunk c takes rounds c, c + own_chunks, ...
  const int n = p.prefix_chunks + p.own_chunks;
  auto counts = [&](int i) { return (i >= skip && i < np) || (i >= p.prefix_chunks && i < p.prefix_chunks + no); };
  auto reads = [&](int i) { return i < n && (!window || counts(i)); };
  float m = -INFINITY, l = 0.f;  // m alike in all threads, l over the team's parts
  f32x4_t acc{};
  for (int base = window ? skip / kMergeThreads * kMergeThreads : 0; base < n; base += kMergeThreads) {
    float2 ml{-INFINITY, 0.f};
    if (reads(base + tid)) ml = p.part_ml[(base + tid) * rows_all + row];
    auto load = [&](int j) {
      const int i = base + team + kTeams * j;
      return reads(i) ? *reinterpret_cast<const f32x4_t*>(p.part_o + (i * rows_all + row) * D + 4 * c)
                      : f32x4_t{};
    };
    f32x4_t rows[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) rows[j] = load(j);
    if (!counts(base + tid)) ml = float2{-INFINITY, 0.f};
    const float mx = wave_max(ml.x);
    if (base > 0) __syncthreads();  // the weights of the parts before are read
    if ((tid & 63) == 0) wave_m[tid >> 6] = mx;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) mn = fmaxf(mn, wave_m[w]);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float wgt = fast_exp2((ml.x - mu) * kLog2e), keep = fast_exp2((m - mu) * kLog2e);
    weight[tid] = wgt;
    weighted[tid] = wgt * ml.y;
    __syncthreads();
    l *= keep;
    acc *= keep;
    m = mn;
    for (int j0 = 0; base + kTeams * j0 < n && kTeams * j0 < kMergeThreads; j0 += kAhead) {
      if (j0 > 0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) rows[j] = load(j0 + j);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = team + kTeams * (j0 + j);
        if (i < kMergeThreads && counts(base + i)) {
          acc += weight[i] * rows[j];
          l += weighted[i];
        }
      }
    }
  }
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
  part_o[team][c] = acc;
  if (c == 0) part_l[team] = l;
  __syncthreads();
  if (team != 0) return;
#pragma unroll
  for (int t = 1; t < kTeams; ++t) {
    acc += part_o[t][c];
    l += part_l[t];
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
  // one workgroup a piece up to the resident ones; past them, the pieces of own keys go round
  const int64_t pieces = (int64_t)p.prefix_blocks + p.own_pieces;
  const int64_t most = p.prefix_blocks > kSharedSlots ? p.prefix_blocks : kSharedSlots;
  const int64_t blocks = pieces < most ? pieces : most;
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
                     dim3((unsigned)((int64_t)p.batch * p.n_heads)), dim3(kMergeThreads), 0, stream, p);
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
