// Sequences that begin alike (kq_attend_shared.cu): the parts on the tensor cores of kq_attend_many.cuh.
#include "kq_attend_many.cuh"

namespace kq {

// The common keys of groups whose sequences together make more than `beyond` query rows a kv head.
cudaError_t attend_shared_prefix_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh) {
  return launch_many<true>(env, a, beyond, sh, true);
}

cudaError_t attend_shared_rest_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh) {
  return launch_many<true>(env, a, beyond, sh, false);
}

}  // namespace kq
