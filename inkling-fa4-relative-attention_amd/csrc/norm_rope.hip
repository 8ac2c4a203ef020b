// RMS norm of query and key heads with the position rotation in the same pass
// (forward, backward), and the same on the way into a paged KV cache, for gfx950.
//
// Mathematics, per head row x of D elements at position p:
//   r = 1 / sqrt(mean(x^2) + eps),  z = x r w                      (w NULL: z = x)
//   y_e = z_e c_e + z_e' s_e   for the rot leading elements, e' the partner of e:
//     half-split   e' = e +- rot / 2,  angle index e mod (rot / 2)
//     interleaved  e' = e ^ 1,         angle index e / 2
//   c = cos[p], s = -sin[p] for the first of a pair and +sin[p] for the second;
//   elements from rot on: y = z.
// Written y = r (x A + x' B) with A = w c, B = w' s: A and B depend on the token and
// on q or k alone, so a token's heads share them.
// Backward, with g the gradient of y: the rotation's transpose is the rotation by -p, so
//   gz_e = g_e c_e - g_e' s_e;   dw = sum over rows of gz x r;
//   dx = r gz w - x (r^3 / D) sum_e(gz_e w_e x_e),
// taken as r (gz w - (x r) (r / D) sum): r^3 leaves fp32 for rows of rms 1e13 and more, and for
// tiny ones next to a tiny eps, where the outputs and gradients are ordinary numbers.
// r is computed again from x, which the backward pass reads anyway: nothing but the
// inputs is kept between the passes.  All of it is in fp32 with one rounding at the end.
//
// Layout.  A row is held by D / 8 neighbouring lanes, 16 bytes each; such a lane group
// takes a token and walks over a chunk of its heads (q heads, then k heads, then for
// the cache v heads) with the token's A and B in registers.  The forward has kAhead rows' loads
// in flight and asks for the first ahead of the token's position, whose search is the longest
// chain of a small append; the backward has two rows' x and g.  Row sums meet by DPP adds,
// partners by lane exchange of the packed 16-bit row (half-split) or inside the lane
// (interleaved).
//
// Bound: memory, and for small calls the launch.  bf16, d 128, 32768 tokens of 8 + 2 heads on fresh
// inputs: forward 37.0 us (168 MB at 4.5 TB/s), backward 47.6 us (252 MB at 5.3 TB/s, the rate of a
// copy) and 4 us for the weights, into a cache with values 45.4 us (203 MB at 4.5 TB/s).  Where
// the caches hold part of the inputs forward takes 29 us (45.5 with two rows in flight and none ahead
// of the position), into a cache 34.5; 64 decode tokens into a cache take 4.7 us.
#include <type_traits>

#include "ifa4_device.hpp"
#include "ifa4_kernels.h"

namespace ifa4 {
namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // rows a lane group has in flight: 2 / 4 / 6 take 29.1 / 28.3 / 28.9 us for
                           // 32768 tokens of 8 + 2 heads, 3.1 / 3.1 / 3.2 for 64

template <int D>
struct RowShape {
  static constexpr int kLpr = D / 8;            // lanes per row
  static constexpr int kPerWave = 64 / kLpr;    // rows side by side in a wave
  static constexpr int kPerBlock = kThreads / kLpr;
};

template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), kCtrl, 0xf, 0xf, false));
}
// Sum over the lanes of a row (16 or 8), in every lane.
template <int kLpr>
__device__ __forceinline__ float row_sum(float x) {
  if constexpr (kLpr == 16) {
    x += dpp<0x128>(x);  // row_ror 8, 4, 2, 1
    x += dpp<0x124>(x);
    x += dpp<0x122>(x);
    x += dpp<0x121>(x);
  } else {
    x += dpp<0xb1>(x);   // lane ^ 1, lane ^ 2, then the other quad of the eight
    x += dpp<0x4e>(x);
    x += dpp<0x141>(x);
  }
  return x;
}

template <typename Tag>
__device__ __forceinline__ void unpack8(u32x4_t w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = Elem<Tag>::lo(w[i]);
    f[2 * i + 1] = Elem<Tag>::hi(w[i]);
  }
}
template <typename Tag>
__device__ __forceinline__ u32x4_t pack8(const float* f) {
  return u32x4_t{Elem<Tag>::pack2(f[0], f[1]), Elem<Tag>::pack2(f[2], f[3]),
                 Elem<Tag>::pack2(f[4], f[5]), Elem<Tag>::pack2(f[6], f[7])};
}

// Elements i to i + 7 of a norm weight (dtype: ifa4_dtype) as fp32; 1 without a weight.  A
// weight is aligned to its elements only.
template <typename T>
struct __attribute__((packed, aligned(2))) Loose {
  T v;
};
__device__ __forceinline__ void weights8(const void* w, int dtype, int i, float* f) {
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 1.f;
  } else if (dtype == 2) {
    const auto* at = reinterpret_cast<const Loose<f32x4_t>*>(static_cast<const float*>(w) + i);
    const f32x4_t a = at[0].v, b = at[1].v;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < 4 ? a[e] : b[e - 4];
  } else {
    const u32x4_t a =
        reinterpret_cast<const Loose<u32x4_t>*>(static_cast<const uint16_t*>(w) + i)->v;
    if (dtype == 0)
      unpack8<Bf16Tag>(a, f);
    else
      unpack8<F16Tag>(a, f);
  }
}

// Where the elements of a lane turn: the partner lane's distance (half-split) and the
// first angle of the lane; turns: the lane lies in the rot leading elements.
struct Turn {
  int hop;    // half-split: partner = lane + hop
  int angle;  // index of the lane's first cos / sin
  bool turns, second;
};
template <bool kPairs>
__device__ __forceinline__ Turn turn_of(const NormRopeParams& p, int c) {
  Turn t;
  const int half = p.rot / 2;
  t.turns = 8 * c < p.rot;
  t.second = !kPairs && 8 * c >= half;
  t.hop = kPairs || !t.turns ? 0 : (t.second ? -(half / 8) : half / 8);
  t.angle = kPairs ? 4 * c : 8 * c - (t.second ? half : 0);
  return t;
}

// cos and signed sin of the lane's eight elements at position pos (1 and 0 where nothing turns).
template <bool kPairs>
__device__ __forceinline__ void angles(const NormRopeParams& p, const Turn& t, int pos, float* cs,
                                       float* sn) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (!t.turns) return;
  // positions outside the table read its nearest row, never past it
  const int64_t row = (int64_t)min(max(pos, 0), p.max_position - 1) * p.angle_stride + t.angle;
  const f32x4_t* cp = reinterpret_cast<const f32x4_t*>(p.cos + row);
  const f32x4_t* sp = reinterpret_cast<const f32x4_t*>(p.sin + row);
  if constexpr (kPairs) {
    const f32x4_t a = cp[0], b = sp[0];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = a[e / 2];
      sn[e] = (e & 1) ? b[e / 2] : -b[e / 2];
    }
  } else {
    const f32x4_t a0 = cp[0], a1 = cp[1], b0 = sp[0], b1 = sp[1];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = e < 4 ? a0[e] : a1[e - 4];
      const float b = e < 4 ? b0[e] : b1[e - 4];
      sn[e] = t.second ? b : -b;
    }
  }
}

// Partners of the lane's eight elements (packed): the row of lane + hop, or the lane's own
// with neighbours swapped; zeros where nothing turns (an infinity there times a sine of 0
// would be NaN).
template <bool kPairs>
__device__ __forceinline__ u32x4_t partners(u32x4_t w, const Turn& t, int lane) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = kPairs ? __builtin_amdgcn_alignbit(w[i], w[i], 16)
                              : (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (lane + t.hop), (int)w[i]);
    r[i] = t.turns ? x : 0u;
  }
  return r;
}

// A and B of the lane's elements for one weight: w and, at the partners, w'.
template <bool kPairs>
__device__ __forceinline__ void coefficients(const NormRopeParams& p, const void* weight,
                                             const Turn& t, int c, const float* cs,
                                             const float* sn, float* a, float* b) {
  float w[8], wp[8];
  weights8(weight, p.w_dtype, 8 * c, w);
  if constexpr (!kPairs) weights8(weight, p.w_dtype, 8 * (c + t.hop), wp);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    a[e] = w[e] * cs[e];
    b[e] = (kPairs ? w[e ^ 1] : wp[e]) * sn[e];
  }
}

// x / d in fp32 by inv = 1 / d and the residual: the division's own bits wherever e4m3 has a
// value (checked for every 16-bit x and 51 d).  The product with inv alone turns ties of e4m3 the
// wrong way, 30 of the bf16 values at d = 7.  Past the range x * inv is as good.
__device__ __forceinline__ float quotient(float x, float d, float inv) {
  const float q = x * inv;
  return fabsf(q) < 1024.f ? fmaf(fmaf(-q, d, x), inv, q) : q;
}

// Eight fp32 values -> OCP e4m3, nearest even; magnitudes past 448 become 448, NaN stays.
__device__ __forceinline__ u32x2_t pack_fp8(const float* f) {
  u32x2_t r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = f[4 * h + i];
      x[i] = v != v ? v : fminf(fmaxf(v, -448.f), 448.f);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    r[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  }
  return r;
}

// Last sequence b with cu[b] <= t, by the lanes of a group together (one of them probes
// one entry a round: 16 or 8 ways); a guess that holds, as with one token a sequence,
// skips the search.  Whatever cu holds the result lies in [0, batch).
template <int kLpr>
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, int t, int lane) {
  const int guess = min(t, batch - 1);
  int lo = 0, hi = batch;
  if (cu[guess] <= t && t < cu[guess + 1]) {
    lo = guess;
    hi = guess + 1;
  }
  const int c = lane % kLpr, g0 = lane - c;
  while (wave_any(hi - lo > 1)) {
    const int step = max((hi - lo + kLpr - 1) / kLpr, 1);
    const int at = lo + c * step;
    const bool below = c == 0 || (at < hi && cu[at] <= t);
    const uint64_t m = __builtin_amdgcn_ballot_w64(below) >> g0;
    const int n = __builtin_ctzll(~(m & ((1ull << kLpr) - 1)));  // leading probes that hold
    const int from = lo;
    lo = from + (n - 1) * step;
    hi = min(hi, from + n * step);
  }
  return lo;
}

// Where a new token's key and value go: its position, and the block and row (row -1: nowhere);
// covered: the token belongs to a sequence.
struct Slot {
  int pos, row;
  int64_t block;
  bool covered;
};
template <int kLpr>
__device__ __forceinline__ Slot find_slot(const AppendParams& a, int t, int lane) {
  const int b = find_sequence<kLpr>(a.cu, a.batch, t, lane);
  const int s = a.cu[b], e = a.cu[b + 1];
  Slot r;
  r.pos = a.seqused_k[b] - (e - t);
  r.row = -1;
  r.block = 0;
  r.covered = t >= s && t < e;
  const int cap = a.max_blocks << a.block_shift;
  if (r.covered && r.pos >= 0 && r.pos < cap) {
    const int ent = a.block_table[(int64_t)b * a.bt_stride + (r.pos >> a.block_shift)];
    if ((unsigned)ent < (unsigned)a.num_blocks) {
      r.block = ent;
      r.row = r.pos & ((1 << a.block_shift) - 1);
    }
  }
  return r;
}

// ---- forward, and the append to a paged cache -------------------------------------------------
// kCache: 0 none (q and k come back), 1 cache of the inputs' type, 2 e4m3 cache.
template <int D, typename Tag, bool kPairs, int kCache>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeParams p, AppendParams ap) {
  using S = RowShape<D>;
  constexpr int kLpr = S::kLpr;
  const int lane = threadIdx.x & 63, c = lane % kLpr;
  const int64_t t64 = p.first_token + (int64_t)blockIdx.x * S::kPerBlock + threadIdx.x / kLpr;
  const bool in = t64 < p.total;
  const int t = in ? (int)t64 : (int)p.total - 1;  // idle groups follow the last token, and store nothing
  const Turn turn = turn_of<kPairs>(p, c);

  const int hq = p.n_heads, hk = hq + p.kv_heads;
  const int h_end = min((int)(blockIdx.y + 1) * p.heads_per, kCache != 0 ? hk + p.kv_heads : hk);
  const int64_t lane_q = t * p.q_st + 8 * c, lane_k = t * p.k_st + 8 * c;
  const int64_t lane_v = kCache != 0 ? t * ap.v_st + 8 * c : 0;
  auto load = [&](int h, u32x4_t* raw) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int g = h + i;
      if (g >= h_end) continue;
      if (g < hq)
        raw[i] = ld_global_16(static_cast<const uint16_t*>(p.q) + lane_q + g * p.q_sh);
      else if (g < hk)
        raw[i] = ld_global_16(static_cast<const uint16_t*>(p.k) + lane_k + (g - hq) * p.k_sh);
      else if constexpr (kCache != 0)
        raw[i] = ld_global_16(static_cast<const uint16_t*>(ap.v) + lane_v + (g - hk) * ap.v_sh);
    }
  };
  int h = (int)blockIdx.y * p.heads_per;
  u32x4_t raw[kAhead] = {};
  load(h, raw);  // on their way while the position is looked up

  Slot slot{};
  int pos = 0;
  if constexpr (kCache != 0) {
    slot = find_slot<kLpr>(ap, t, lane);
    pos = slot.pos;
  } else if (p.positions != nullptr) {
    pos = p.positions[t];
  }
  float aq[8], bq[8], ak[8], bk[8];
  {
    float cs[8], sn[8];
    angles<kPairs>(p, turn, pos, cs, sn);
    coefficients<kPairs>(p, p.q_weight, turn, c, cs, sn, aq, bq);
    coefficients<kPairs>(p, p.k_weight, turn, c, cs, sn, ak, bk);
  }
  const bool stores = in && (kCache == 0 || slot.covered);

  auto turned = [&](u32x4_t w, const float* a, const float* b, bool norm, float* y) {
    float x[8], px[8];
    unpack8<Tag>(w, x);
    unpack8<Tag>(partners<kPairs>(w, turn, lane), px);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
    ss = row_sum<kLpr>(ss);
    const float r = norm ? rsqrtf(ss * (1.f / D) + p.eps) : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = r * fmaf(x[e], a[e], px[e] * b[e]);
  };
  auto put_cache = [&](void* cache, int64_t at, const float* y, float scale, float inv, u32x4_t raw16) {
    if constexpr (kCache == 1) {
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(cache) + at + 8 * c) = raw16;
    } else {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = quotient(y[e], scale, inv);
      *reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(cache) + at + 8 * c) = pack_fp8(z);
    }
  };
  auto put = [&](int g, u32x4_t w) {
    float y[8];
    if (g < hq) {
      turned(w, aq, bq, p.q_weight != nullptr, y);
      uint16_t* dst = static_cast<uint16_t*>(p.q_out) + t * p.qo_st + g * p.qo_sh + 8 * c;
      if (stores) *reinterpret_cast<u32x4_t*>(dst) = pack8<Tag>(y);
    } else if (g < hk) {
      turned(w, ak, bk, p.k_weight != nullptr, y);
      if constexpr (kCache == 0) {
        uint16_t* dst = static_cast<uint16_t*>(p.k_out) + t * p.ko_st + (g - hq) * p.ko_sh + 8 * c;
        if (stores) *reinterpret_cast<u32x4_t*>(dst) = pack8<Tag>(y);
      } else if (stores && slot.row >= 0) {
        put_cache(ap.k_cache, slot.block * ap.kc_sblk + slot.row * ap.kc_st + (g - hq) * ap.kc_sh, y,
                  ap.k_scale, ap.inv_k_scale, pack8<Tag>(y));
      }
    } else if constexpr (kCache != 0) {
      if (!stores || slot.row < 0) return;
      unpack8<Tag>(w, y);
      put_cache(ap.v_cache, slot.block * ap.vc_sblk + slot.row * ap.vc_st + (g - hk) * ap.vc_sh, y,
                ap.v_scale, ap.inv_v_scale, w);
    }
  };
  while (true) {
    u32x4_t next[kAhead] = {};
    const bool more = h + kAhead < h_end;
    if (more) load(h + kAhead, next);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (h + i < h_end) put(h + i, raw[i]);
    if (!more) break;
    h += kAhead;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) raw[i] = next[i];
  }
}

// ---- backward -------------------------------------------------------------------------------
// A workgroup walks over tokens and a chunk of their heads, and leaves its sums of the weight
// gradients in one row of the workspace, [q or k][D]; the second kernel adds the rows in a fixed
// order.
template <int D, typename Tag, bool kPairs>
__global__ __launch_bounds__(kThreads) void norm_rope_bwd_kernel(NormRopeParams p, NormRopeGrad g) {
  using S = RowShape<D>;
  constexpr int kLpr = S::kLpr;
  __shared__ float sums[S::kPerBlock][2][D];
  const int lane = threadIdx.x & 63, c = lane % kLpr, grp = threadIdx.x / kLpr;
  const Turn turn = turn_of<kPairs>(p, c);
  float wq[8], wk[8], dwq[8] = {}, dwk[8] = {};
  weights8(p.q_weight, p.w_dtype, 8 * c, wq);
  weights8(p.k_weight, p.w_dtype, 8 * c, wk);
  const int hq = p.n_heads;
  const int h_beg = max(g.gq != nullptr ? 0 : hq, (int)blockIdx.y * p.heads_per);
  const int h_all = min(g.gk != nullptr ? hq + p.kv_heads : hq, (int)(blockIdx.y + 1) * p.heads_per);
  for (int64_t t0 = (int64_t)blockIdx.x * S::kPerBlock; t0 < p.total;
       t0 += (int64_t)gridDim.x * S::kPerBlock) {
    const bool in = t0 + grp < p.total;
    const int64_t t = in ? t0 + grp : p.total - 1;
    float cs[8], sn[8];
    angles<kPairs>(p, turn, p.positions != nullptr ? p.positions[t] : 0, cs, sn);
    auto load = [&](int h, u32x4_t& xr, u32x4_t& gr) {
      const bool is_q = h < hq;
      const int64_t k = h - hq;
      xr = ld_global_16(is_q ? static_cast<const uint16_t*>(p.q) + t * p.q_st + h * p.q_sh + 8 * c
                             : static_cast<const uint16_t*>(p.k) + t * p.k_st + k * p.k_sh + 8 * c);
      gr = ld_global_16(is_q ? static_cast<const uint16_t*>(g.gq) + t * g.gq_st + h * g.gq_sh + 8 * c
                             : static_cast<const uint16_t*>(g.gk) + t * g.gk_st + k * g.gk_sh + 8 * c);
    };
    auto put = [&](int h, u32x4_t xr, u32x4_t gr) {
      const bool is_q = h < hq;
      float x[8], gy[8], pg[8], gw[8];
      unpack8<Tag>(xr, x);
      unpack8<Tag>(gr, gy);
      const u32x4_t pgr = partners<kPairs>(gr, turn, lane);
      unpack8<Tag>(pgr, pg);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        gy[e] = fmaf(gy[e], cs[e], -pg[e] * sn[e]);  // gz
        gw[e] = gy[e] * (is_q ? wq[e] : wk[e]);
        ss = fmaf(x[e], x[e], ss);
        dot = fmaf(gw[e], x[e], dot);
      }
      ss = row_sum<kLpr>(ss);
      dot = row_sum<kLpr>(dot);
      if ((is_q ? p.q_weight : p.k_weight) != nullptr) {
        const float r = rsqrtf(ss * (1.f / D) + p.eps);
        const float mean = r * dot * (1.f / D);  // of the gradient along x r
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xr = x[e] * r;
          const float dw = in ? gy[e] * xr : 0.f;
          if (is_q)
            dwq[e] += dw;
          else
            dwk[e] += dw;
          gw[e] = r * fmaf(-xr, mean, gw[e]);
        }
      }
      if (!in) return;
      uint16_t* dst = is_q ? static_cast<uint16_t*>(g.dq) + t * g.dq_st + h * g.dq_sh
                           : static_cast<uint16_t*>(g.dk) + t * g.dk_st + (h - hq) * g.dk_sh;
      *reinterpret_cast<u32x4_t*>(dst + 8 * c) = pack8<Tag>(gw);
    };
    for (int h = h_beg; h < h_all; h += 2) {
      u32x4_t x0, g0, x1{}, g1{};
      load(h, x0, g0);
      const bool two = h + 1 < h_all;
      if (two) load(h + 1, x1, g1);
      put(h, x0, g0);
      if (two) put(h + 1, x1, g1);
    }
  }
  if (g.partial == nullptr) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sums[grp][0][8 * c + e] = dwq[e];
    sums[grp][1][8 * c + e] = dwk[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < S::kPerBlock; ++k) s += sums[k][i / D][i % D];
    g.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * D + i] = s;
  }
}

// dw of 32 columns of [q or k][D]: 32 threads a column over the partial rows, then a tree in LDS.
constexpr int kSumCols = 32, kSumRows = 32;
__global__ __launch_bounds__(kSumCols * kSumRows) void norm_rope_dw_kernel(NormRopeGrad g,
                                                                           int head_dim, int rows,
                                                                           int w_dtype) {
  __shared__ float part[kSumRows / 2][kSumCols + 1];
  const int col = threadIdx.x % kSumCols, rg = threadIdx.x / kSumCols;
  const int i = blockIdx.x * kSumCols + col;
  float s = 0.f;
#pragma unroll 8
  for (int r = rg; r < rows; r += kSumRows) s += g.partial[(int64_t)r * 2 * head_dim + i];
#pragma unroll
  for (int n = kSumRows / 2; n > 0; n /= 2) {
    if (rg >= n && rg < 2 * n) part[rg - n][col] = s;
    __syncthreads();
    if (rg < n) s += part[rg][col];
    __syncthreads();
  }
  if (rg != 0) return;
  void* dst = i < head_dim ? g.dq_weight : g.dk_weight;
  if (dst == nullptr) return;
  const int e = i % head_dim;
  if (w_dtype == 2)
    static_cast<float*>(dst)[e] = s;
  else if (w_dtype == 0)
    static_cast<__bf16*>(dst)[e] = (__bf16)s;
  else
    static_cast<_Float16*>(dst)[e] = (_Float16)s;
}

// Workgroups from which on a token's heads stay together.  Forward, bf16, d 128, heads split for
// 256 / 512 / 1024 / 2048 workgroups: 512 tokens of 64 + 8 heads 6.9 / 6.0 / 5.6 / 6.8 us, 2048 of
// them 19.3 / 15.8 / 14.9 / 18.2, 2048 of 8 + 2 5.1 / 4.5 / 4.6 / 4.5, 8192 of 8 + 2 alike.
constexpr int64_t kFill = 1024;
// Backward: workgroups over tokens at most, and those up to which heads are split; each leaves a
// row of partial sums for the second kernel.  Both kernels, heads split / together: 512 tokens of
// 64 + 8 heads 11.4 / 46.4 us, 2048 of them 23.8 / 53.7, one token of 8 + 2 6.1 / 10.1.
// 32768 tokens of 8 + 2 heads on 256 / 512 / 768 / 1024 / 2048 / 4096 workgroups: 65.8 / 43.9 / 37.5 /
// 37.3 / 39.3 / 39.0.
constexpr int64_t kBwdTokenBlocks = 1024, kBwdFill = 896;
// Workgroups of one launch along the tokens: a launch holds less than 2^32 threads.
constexpr int64_t kMostBlocks = 1 << 20;
int heads_per(int heads, int64_t fill, int64_t blocks) {
  int64_t chunks = fill / blocks;
  if (chunks > (heads + 1) / 2) chunks = (heads + 1) / 2;
  return chunks > 1 ? (int)((heads + chunks - 1) / chunks) : heads;
}

template <int D, typename Tag, bool kPairs>
hipError_t launch_fwd(NormRopeParams p, const AppendParams& a, int cache, hipStream_t stream) {
  using S = RowShape<D>;
  const int heads = p.n_heads + (cache != 0 ? 2 : 1) * p.kv_heads;
  const int64_t blocks = (p.total + S::kPerBlock - 1) / S::kPerBlock;
  // Heads a lane group walks over: all of a token's where the tokens alone make kFill
  // workgroups, fewer, but two or more, for fewer tokens.
  p.heads_per = heads_per(heads, kFill, blocks);
  const unsigned chunks = (unsigned)((heads + p.heads_per - 1) / p.heads_per);
  for (int64_t at = 0; at < blocks; at += kMostBlocks) {
    const dim3 grid((unsigned)(blocks - at < kMostBlocks ? blocks - at : kMostBlocks), chunks);
    p.first_token = at * S::kPerBlock;
    if (cache == 0)
      hipLaunchKernelGGL((norm_rope_kernel<D, Tag, kPairs, 0>), grid, dim3(kThreads), 0, stream, p, a);
    else if (cache == 1)
      hipLaunchKernelGGL((norm_rope_kernel<D, Tag, kPairs, 1>), grid, dim3(kThreads), 0, stream, p, a);
    else
      hipLaunchKernelGGL((norm_rope_kernel<D, Tag, kPairs, 2>), grid, dim3(kThreads), 0, stream, p, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int D, typename Tag, bool kPairs>
hipError_t launch_bwd(NormRopeParams p, const NormRopeGrad& g, hipStream_t stream) {
  const NormRopeBwdGrid grid = norm_rope_bwd_grid(p.total, p.n_heads + p.kv_heads, D);
  const int64_t rows = (int64_t)grid.x * grid.y;
  p.heads_per = grid.heads_per;
  hipLaunchKernelGGL((norm_rope_bwd_kernel<D, Tag, kPairs>), dim3(grid.x, grid.y), dim3(kThreads), 0,
                     stream, p, g);
  if (g.partial != nullptr) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(norm_rope_dw_kernel, dim3(2 * D / kSumCols), dim3(kSumCols * kSumRows), 0,
                       stream, g, D, (int)rows, p.w_dtype);
  }
  return hipGetLastError();
}

// f(D, Tag, pairs) for the call's head_dim, type and kind of rotation.
template <typename F>
hipError_t dispatch(const NormRopeParams& p, int head_dim, int dtype, F f) {
  auto by_pairs = [&](auto d, auto tag) {
    return p.pairs ? f(d, tag, std::true_type{}) : f(d, tag, std::false_type{});
  };
  auto by_type = [&](auto d) {
    return dtype == 0 ? by_pairs(d, Bf16Tag{}) : by_pairs(d, F16Tag{});
  };
  return head_dim == 128 ? by_type(std::integral_constant<int, 128>{})
                         : by_type(std::integral_constant<int, 64>{});
}

}  // namespace

NormRopeBwdGrid norm_rope_bwd_grid(int64_t total, int heads, int head_dim) {
  const int64_t per = kThreads / (head_dim / 8);
  int64_t blocks = (total + per - 1) / per;
  if (blocks > kBwdTokenBlocks) blocks = kBwdTokenBlocks;
  NormRopeBwdGrid g;
  g.x = (unsigned)blocks;
  g.heads_per = heads_per(heads, kBwdFill, blocks);
  g.y = (unsigned)((heads + g.heads_per - 1) / g.heads_per);
  return g;
}

hipError_t launch_norm_rope(const NormRopeParams& p, const AppendParams& a, int cache, int head_dim,
                            int dtype, hipStream_t stream) {
  return dispatch(p, head_dim, dtype, [&](auto d, auto tag, auto pairs) {
    return launch_fwd<decltype(d)::value, decltype(tag), decltype(pairs)::value>(p, a, cache, stream);
  });
}

hipError_t launch_norm_rope_bwd(const NormRopeParams& p, const NormRopeGrad& g, int head_dim,
                                int dtype, hipStream_t stream) {
  return dispatch(p, head_dim, dtype, [&](auto d, auto tag, auto pairs) {
    return launch_bwd<decltype(d)::value, decltype(tag), decltype(pairs)::value>(p, g, stream);
  });
}

}  // namespace ifa4
