// kh_paged_f16x2.hip - attention over a paged cache of fp16, fp32 activations in two passes (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_f16x2(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_F16, 2, 2>(w, dt, rt, stream);
}

}  // namespace kh
