// Attention of few query rows over the tokens of selected pages (kq_attend_few.cuh): every row of the call and kv head has a list of them.
#include "kq_attend_few.cuh"

namespace kq {

cudaError_t launch_attend_selected(const LaunchEnv& env, const AttendArgs& a, const SelectedArgs& selected) {
  FewParams p = few_params(env, a, 0xFFFFFFFFu);
  p.sel = selected;
  return launch_few<kSelected>(env, p, a.heads / a.cache.kv_heads);
}

}  // namespace kq
