// Attention of few query rows over the tokens of selected pages (kq_attend_few.cuh): every row of the call and kv head has a list of them.
//
// As there, 16-bit queries (rotated) and their weights are rounded to binary16 once, 2^-11 each, f32 ones are two parts: against 64 bits f16 3.9e-4 of the
// result (its own rounding 2.1e-4), bf16 1.69e-3 (1.66e-3), f32 4.4e-7.  The parts are an eighth of the whole step: 64 sequences, 64 pages each, with their
// summaries and selection 120 us with f32 queries, 111 with bf16 ones; so the type of the queries chooses here too.
#include "kq_attend_few.cuh"

namespace kq {

cudaError_t launch_attend_selected(const LaunchEnv& env, const AttendArgs& a, const SelectedArgs& selected) {
  FewParams p = few_params(env, a, 0xFFFFFFFFu);
  p.sel = selected;
  return launch_few<kSelected>(env, p, a.heads / a.cache.kv_heads);
}

}  // namespace kq
