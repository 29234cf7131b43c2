// kh_paged_mx4x2.hip - attention over a paged cache in 4 bits, fp16 activations: two bf16 parts of q and of the
// weights (kh_paged_mx4.hpp).
#include "kh_paged_mx4.hpp"

namespace kh {

hipError_t launch_paged_mx4x2(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_mx4<2, 2>(w, dt, rt, stream);
}

}  // namespace kh
