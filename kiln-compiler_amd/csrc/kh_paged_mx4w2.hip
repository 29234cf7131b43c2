// kh_paged_mx4w2.hip - attention over a paged cache in 4 bits, bf16 activations: scores in one pass, weights in two
// parts (kh_paged_mx4.hpp).
#include "kh_paged_mx4.hpp"

namespace kh {

hipError_t launch_paged_mx4w2(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_mx4<1, 2>(w, dt, rt, stream);
}

}  // namespace kh
