// Prefill over contiguous K/V (prefill_kernel.hpp): the plain form and the fused relative-logit
// projection.
#include "prefill_kernel.hpp"

namespace ifa4 {
namespace {

template <int D, typename Tag>
hipError_t launch_prefill_rel(const PrefillParams& p, hipStream_t stream) {
  if (p.wt == nullptr) return launch_prefill_form<D, Tag, KvRows>(p, stream);
  // fused projection: r in bf16 or fp32
  return p.rel_dtype == 2
             ? launch_prefill_t<ProjShape, D, Tag, RelF32, KvRows, true, false, false>(p, stream)
             : launch_prefill_t<ProjShape, D, Tag, RelBf16, KvRows, true, false, false>(p, stream);
}

}  // namespace

int prefill_block_q() { return Shape::kBlockQ; }
int prefill_proj_block_q() { return ProjShape::kBlockQ; }
int prefill_block_k() { return Shape::kBlockK; }
bool prefill_tab_packs(int rel_extent, int pack) {
  return pack * bias_pack_pitch(rel_extent, pack, Shape::kBiasPad) <= kBiasPackFloats;
}
bool prefill_tab(const PrefillParams& p) {
  return IFA4_BIAS_LDS && p.rel_st == 0 && p.rel_extent > 0 && p.rel_extent <= kBiasLdsMax;
}
int prefill_waves() { return Shape::kWaves; }

hipError_t launch_prefill(const PrefillParams& p, int head_dim, int qkv_dtype,
                          hipStream_t stream) {
  if (head_dim == 128) {
    return qkv_dtype == 0 ? launch_prefill_rel<128, Bf16Tag>(p, stream)
                          : launch_prefill_rel<128, F16Tag>(p, stream);
  }
  return qkv_dtype == 0 ? launch_prefill_rel<64, Bf16Tag>(p, stream)
                        : launch_prefill_rel<64, F16Tag>(p, stream);
}

}  // namespace ifa4
