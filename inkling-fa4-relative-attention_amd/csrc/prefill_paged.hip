// Prefill over a paged cache of the inputs' type (prefill_kernel.hpp).
#include "prefill_kernel.hpp"

namespace ifa4 {

hipError_t launch_prefill_paged(const PrefillParams& p, int head_dim, int qkv_dtype,
                               hipStream_t stream) {
  return launch_prefill_types<KvPaged>(p, head_dim, qkv_dtype, stream);
}

}  // namespace ifa4
