// Sequences that begin alike (kq_attend_shared.cu): the parts on the tensor cores of kq_attend_many.cuh.
#include "kq_attend_many.cuh"

namespace kq {

// The common keys of groups whose sequences together make more query rows a kv head than the other kernel is for.
bool attend_shared_prefix_many(const LaunchEnv& env, const AttendArgs& a, const SharedArgs& sh, cudaError_t* e) {
  const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * (a.heads / a.cache.kv_heads) / sh.groups;
  if (rows <= 32 || !attend_many_supports(a)) return false;
  *e = launch_many<true>(env, a, 0, sh, true);
  return true;
}

cudaError_t attend_shared_rest_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh) {
  return launch_many<true>(env, a, beyond, sh, false);
}

}  // namespace kq
