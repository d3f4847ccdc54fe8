// Sequences that begin alike (kq_attend_shared.cu): few rows of float16 queries.
#include "kq_attend_few.cuh"

namespace kq {

cudaError_t attend_shared_few_f16(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, bool prefix, const SharedArgs& sh, uint64_t rows) {
  return few_shared<__half>(env, a, beyond, prefix, sh, rows);
}

}  // namespace kq
