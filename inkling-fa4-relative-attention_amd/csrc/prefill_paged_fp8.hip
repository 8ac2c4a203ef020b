// Prefill over a paged cache of e4m3 values (prefill_kernel.hpp).
#include "prefill_kernel.hpp"

namespace ifa4 {

hipError_t launch_prefill_paged_fp8(const PrefillParams& p, int head_dim, int qkv_dtype,
                                   hipStream_t stream) {
  return launch_prefill_types<KvPaged8>(p, head_dim, qkv_dtype, stream);
}

}  // namespace ifa4
