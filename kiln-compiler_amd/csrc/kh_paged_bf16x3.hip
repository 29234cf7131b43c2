// kh_paged_bf16x3.hip - attention over a paged cache of bf16, fp32 activations in three passes (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_bf16x3(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_BF16, 3, 3>(w, dt, rt, stream);
}

}  // namespace kh
