// kh_paged_bf16w2.hip - attention over a paged cache of bf16, bf16 activations: scores in one pass, weights in two
// parts (kh_paged_attn.hpp).
#include "kh_paged_attn.hpp"

namespace kh {

hipError_t launch_paged_bf16w2(const PagedWork &w, int dt, int rt, hipStream_t stream) {
  return launch_passes<KH_TYPE_BF16, 1, 2>(w, dt, rt, stream);
}

}  // namespace kh
