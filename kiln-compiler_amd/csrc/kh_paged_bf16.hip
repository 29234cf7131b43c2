// kh_paged_bf16.hip - attention over a paged cache of bf16, products in one pass (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_bf16(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_BF16, 1, 1>(w, dt, rt, stream);
}

}  // namespace kh
