// Attention over the paged 4-bit cache: which kernel a call's sequences are the work of (kq_attend_few.cuh, kq_attend_many.cuh).
#include "kq_attend_few.cuh"

namespace kq {

cudaError_t launch_attend(const LaunchEnv& env, const AttendArgs& a, int* launches) {
  // Each sequence is the work of one kernel, by its own rows: a call may hold prompts and single tokens.
  const uint64_t rows = static_cast<uint64_t>(a.batch.most) * (a.heads / a.cache.kv_heads);
  const bool many = rows > kFewRows && attend_many_supports(a);
  const uint32_t beyond = many ? kFewRows : 0xFFFFFFFFu;
  cudaError_t e = launch_few<kWhole>(env, few_params(env, a, beyond), many ? kFewRows : rows);
  *launches = many ? 2 : 1;
  if (e == cudaSuccess && many) e = launch_attend_many(env, a, beyond);
  return e;
}

}  // namespace kq
