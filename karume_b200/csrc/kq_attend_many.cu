// Attention of prompts over the paged 4-bit cache: the kernel of kq_attend_many.cuh over whole sequences.
#include "kq_attend_many.cuh"

namespace kq {

bool attend_many_supports(const AttendArgs& a) { return a.cache.head_dim <= 128; }

cudaError_t launch_attend_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond) {
  return launch_many<false>(env, a, beyond, SharedArgs{}, false);
}

}  // namespace kq
