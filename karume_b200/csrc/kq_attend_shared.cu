// Attention of sequences that begin alike: the keys that a group of them has in common are read once.
//
//   out = (2^(M - m) O + 2^(M' - m) O') / (2^(M - m) l + 2^(M' - m) l'),   m = max(M, M')
//
// for the sums (M, l, O) over the common keys and (M', l', O') over a sequence's own: l sums 2^(s - M), O the same times the values.
// Two launches over the same call: the first makes groups sequences of their own, whose rows are all their members' new ones and whose
// keys are the common ones, and leaves (M, l, O) in the scratch; the second walks over the keys behind them and joins.
//
// M, l, O and the joining are f32.  What enters the tensor cores has fewer bits where the queries have 16, as in kq_cache_attention: rotated queries and
// weights are binary16, one rounding of 2^-11 each, and where a group's rows fill blocks of 128 (kq_attend_many.cuh) keys and values are too.  Against
// 64 bits, rms of the result: f16 drafts of five tokens 3.8e-4, where the output's own rounding alone is 2.1e-4; bf16, 64 sequences behind 32768 common
// tokens, 1.73e-3 of 1.66e-3.  f32 queries keep two binary16 parts of each (4.3e-7), which doubles the MMAs: those cases with f32 queries 35.7 for 28.3 and
// 206 for 109 us.  So the type of the queries chooses.
#include "kq_attend_few.cuh"

namespace kq {

// The walk for few rows with f32 and float16 queries, each in a source of its own: they take the compiler longest.
cudaError_t attend_shared_few_f32(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, bool prefix, const SharedArgs& sh, uint64_t rows);
cudaError_t attend_shared_few_f16(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, bool prefix, const SharedArgs& sh, uint64_t rows);
cudaError_t attend_shared_prefix_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh);
cudaError_t attend_shared_rest_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh);

// Bytes that are read once instead of often, from about which on that is faster: without it they come from L2 mostly, with it there is a launch more
// and every row's sums are joined.  This way / the other, 32 heads over 8: bfloat16, 16 sequences behind 8192 common tokens (134 MB saved, just under the line)
// 47 / 41 us, f32 51 / 45; bfloat16, 64 behind 2048 (140 MB, which the rule has on the slower side) 52 / 48, behind 4096 (281 MB) 55 / 75, behind 32768
// (2.2 GB) 104 / 450. 8 heads over 4 of 64, 64 behind 8192 (149 MB) 37 / 46.
constexpr uint64_t kWorth = 128ull << 20;
// Sequences of so many query rows a kv head fill the tensor cores' blocks of rows by themselves: 16 of up to 300 new tokens behind 16384, 4 heads a
// kv head, bfloat16 1511 / 1045 us; 8 of up to 100 behind 32768, 497 / 648.
constexpr uint64_t kAlone = 512;

namespace {

cudaError_t attend_shared_few(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, bool prefix, const SharedArgs& sh, uint64_t rows) {
  if (a.dtype == KQ_F32) return attend_shared_few_f32(env, a, beyond, prefix, sh, rows);
  if (a.dtype == KQ_F16) return attend_shared_few_f16(env, a, beyond, prefix, sh, rows);
  return few_shared<__nv_bfloat16>(env, a, beyond, prefix, sh, rows);
}

}  // namespace

cudaError_t launch_attend_shared(const LaunchEnv& env, const AttendArgs& a, SharedArgs sh, int* launches) {
  // What a call can save at most; then what it does save, as the lengths say on the device.
  const double most = static_cast<double>(a.batch.sequences) * a.batch.width * static_cast<double>(cache_block_bytes(a.cache.page_tokens, a.cache.head_dim)) *
                      a.cache.kv_heads;
  const uint64_t group = a.heads / a.cache.kv_heads;
  if (sh.least == KQ_SHARED_AUTO) sh.least = static_cast<uint64_t>(a.batch.tokens) * group / a.batch.sequences > kAlone ? ~0ull : kWorth;
  // The end of the scratch: a place for each row, and its sums where they are in one part; in front of it the parts of the sums over common
  // keys, a third of the rest.  Where the rows would take more than half of it, every sequence walks over all of its keys.
  // (Places count in pairs of floats, so no more than 32 GB of the scratch is used.)
  const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * a.heads, each = 16 + 4ull * (a.cache.head_dim + 2);
  const uint64_t scratch = std::min<uint64_t>(env.workspace_bytes, 32ull << 30);
  const uint64_t kept = rows * each + 4ull * sh.groups;
  const bool once = most >= static_cast<double>(sh.least) && env.workspace && kept + 64 <= scratch / 2;
  const uint64_t mine = static_cast<uint64_t>(a.batch.most) * group;
  const bool many = mine > kFewRows && attend_many_supports(a);
  if (!once && many) return launch_attend(env, a, launches);
  sh.all_first = sh.first;
  sh.all_tokens = sh.tokens;
  sh.all_groups = sh.groups;
  *launches = 0;
  LaunchEnv in = env;
  cudaError_t e = cudaSuccess;
  if (once) {
    uint8_t* const base = static_cast<uint8_t*>(env.workspace);
    const uint64_t left = (scratch - kept) / 16 * 16, own = left / 3 * 2 / 16 * 16;
    sh.scratch = static_cast<float*>(env.workspace);
    sh.quads = static_cast<uint32_t>(scratch / 16);
    sh.places = reinterpret_cast<uint4*>(base + left);
    sh.sums = (left + rows * 16) / 4;
    sh.keys = reinterpret_cast<int*>(base + left + rows * each);
    LaunchEnv parts = env;
    in.workspace_bytes = own;
    parts.workspace = base + own;
    parts.workspace_bytes = left - own;
    LaunchEnv alone = parts;  // groups that come in turns: none may leave its parts where the next one's go
    if (sh.groups > groups::kAtOnce) alone.workspace = nullptr;
    // Each group is the work of one kernel, by its own rows; where they are many on the average, all are the tensor cores'.  (The few rows' kernel
    // first: what it leaves in the parts' place it has joined itself.)
    const uint64_t all = static_cast<uint64_t>(a.batch.tokens) * group;
    const bool tensor = all > kFewRows && attend_many_supports(a), both = tensor && all / sh.groups <= kFewRows;
    for (uint32_t g = 0; g < sh.groups && e == cudaSuccess; g += groups::kAtOnce) {
      SharedArgs some = sh;
      some.first += g;
      some.tokens += g;
      some.keys += g;
      some.groups = std::min(sh.groups - g, groups::kAtOnce);
      if (!tensor || both) {
        e = attend_shared_few(parts, a, both ? kFewRows : 0xFFFFFFFFu, true, some,
                              both ? kFewRows : (a.batch.tokens + sh.groups - 1) / sh.groups * group);
        *launches += 1;
      }
      if (e == cudaSuccess && tensor) {
        e = attend_shared_prefix_many(alone, a, both ? kFewRows : 0, some);
        *launches += 1;
      }
    }
    if (e != cudaSuccess) return e;
  } else {
    sh.least = ~0ull;  // nothing is common
  }
  e = attend_shared_few(in, a, many ? kFewRows : 0xFFFFFFFFu, false, sh, many ? kFewRows : mine);
  if (e == cudaSuccess && many) e = attend_shared_rest_many(in, a, kFewRows, sh);
  *launches += many ? 2 : 1;
  return e;
}

}  // namespace kq
