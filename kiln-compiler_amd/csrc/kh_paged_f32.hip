// kh_paged_f32.hip - attention over a paged cache of fp32, products in fp32 (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_f32(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_F32, 1, 1>(w, dt, rt, stream);
}

}  // namespace kh
