// kh_paged_f16.hip - attention over a paged cache of fp16, products in one pass (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_f16(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_F16, 1, 1>(w, dt, rt, stream);
}

}  // namespace kh
