// Attention over the paged 4-bit cache (layout in kq_cache.cuh):
//   out = sum_j softmax_j(scale q . k_j) v_j,  k_j = u_j s_j + o_j,  v_j likewise
// A block takes one query row (token and head): a thread per key for the scores, a running maximum and sum, a thread per
// value for the output.
#include <algorithm>

#include "kq_cache.cuh"

namespace kq {
namespace {

constexpr int kAttendThreads = 128;

template <typename T>
__device__ __forceinline__ void store_as(T* p, float v);
template <>
__device__ __forceinline__ void store_as<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store_as<__half>(__half* p, float v) { *p = __float2half_rn(v); }
template <>
__device__ __forceinline__ void store_as<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int D>
__global__ void __launch_bounds__(kAttendThreads) attend_row_kernel(const AttendArgs a) {
  constexpr int kPer = (D + kAttendThreads - 1) / kAttendThreads;
  __shared__ float q_s[D];
  __shared__ float p_s[kAttendThreads], pv_s[kAttendThreads];  // weight, and weight * scale of the value
  __shared__ const uint8_t* v_s[kAttendThreads];
  __shared__ float part[kAttendThreads / 32];
  const uint32_t tid = threadIdx.x, token = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
  const uint32_t kv_head = head / (a.heads / a.cache.kv_heads);
  const uint32_t seq = sequence_of(a.batch, token);
  const Span span = span_of(a.batch, seq);
  const int position = span.length - span.count + static_cast<int>(token) - span.first;
  const bool mine = static_cast<int>(token) >= span.first && static_cast<int>(token) < span.first + span.count;
  T* out = static_cast<T*>(a.out) + token * a.out_stride + head * D;
  if (!mine || position < 0) {
    for (uint32_t d = tid; d < D; d += kAttendThreads) store_as(out + d, 0.0f);
    return;
  }
  if (tid < D / 8) {
    float v[8];
    load8_rotated(static_cast<const T*>(a.q) + token * a.q_stride + head * D, tid * 8, a.rope, position, v);
    for (int i = 0; i < 8; ++i) q_s[tid * 8 + i] = v[i] * (a.scale * 1.4426950408889634f);
  }
  __syncthreads();
  const int from = a.window && position + 1 > static_cast<int>(a.window) ? position + 1 - static_cast<int>(a.window) : 0;
  const uint32_t P = a.cache.page_tokens;
  float top = -INFINITY, total = 0.0f, o[kPer] = {}, off_sum = 0.0f;
  for (int at = from; at <= position; at += kAttendThreads) {
    const int key = at + static_cast<int>(tid);
    float s = -INFINITY, v_scale = 0.0f, v_off = 0.0f;
    const uint8_t* v_row = nullptr;
    if (key <= position) {
      const uint8_t* block = cache_block(a.cache, a.batch, seq, static_cast<uint32_t>(key) / P, kv_head);
      if (block) {
        const uint32_t slot = static_cast<uint32_t>(key) % P;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(block + static_cast<size_t>(slot) * (D / 2));
        float dot = 0.0f, sum = 0.0f;
        for (int w = 0; w < D / 8; ++w) {
          const uint32_t word = row[w];
          for (int i = 0; i < 8; ++i) {
            dot = fmaf(q_s[w * 8 + i], static_cast<float>((word >> (4 * i)) & 15u), dot);
            sum += q_s[w * 8 + i];
          }
        }
        const __half2* par = reinterpret_cast<const __half2*>(block + static_cast<size_t>(P) * D);
        const __half2 ks = par[slot], vs = par[P + slot];
        s = fmaf(dot, __low2float(ks), sum * __high2float(ks));
        v_scale = __low2float(vs);
        v_off = fmaf(7.5f, v_scale, __high2float(vs));  // of codes around zero: sums of many values that cancel keep their bits
        v_row = block + static_cast<size_t>(P + slot) * (D / 2);
      } else {
        s = quiet_nan();
      }
    }
    const bool nan = __syncthreads_or(s != s);
    float m = s;
    for (int x = 16; x > 0; x /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    if (tid % 32 == 0) part[tid / 32] = m;
    __syncthreads();
    float now = top;
    for (int w = 0; w < kAttendThreads / 32; ++w) now = fmaxf(now, part[w]);
    if (nan) now = quiet_nan();
    const float keep = top == -INFINITY ? 0.0f : exp2f(top - now);
    const float p = key <= position ? exp2f(s - now) : 0.0f;
    top = now;
    total = total * keep + p;
    off_sum = off_sum * keep + (key <= position ? p * v_off : 0.0f);
    p_s[tid] = p;
    pv_s[tid] = key <= position ? p * v_scale : 0.0f;
    v_s[tid] = v_row;
    for (int i = 0; i < kPer; ++i) o[i] *= keep;
    __syncthreads();
    for (int i = 0; i < kPer; ++i) {
      const uint32_t d = tid + i * kAttendThreads;
      if (d >= D) break;
      float sum = 0.0f;
      for (int j = 0; j < kAttendThreads && at + j <= position; ++j) {
        const uint32_t byte = v_s[j] ? v_s[j][d / 2] : 0u;
        sum = fmaf(pv_s[j], static_cast<float>((byte >> (4 * (d & 1))) & 15u) - 7.5f, sum);
      }
      o[i] += sum;
    }
    __syncthreads();
  }
  total = warp_sum(total);
  off_sum = warp_sum(off_sum);
  if (tid % 32 == 0) {
    p_s[tid / 32] = total;
    pv_s[tid / 32] = off_sum;
  }
  __syncthreads();
  total = off_sum = 0.0f;
  for (int w = 0; w < kAttendThreads / 32; ++w) {
    total += p_s[w];
    off_sum += pv_s[w];
  }
  for (int i = 0; i < kPer; ++i) {
    const uint32_t d = tid + i * kAttendThreads;
    if (d < D) store_as(out + d, (o[i] + off_sum) / total);
  }
}

template <typename T>
cudaError_t attend_as(const LaunchEnv& env, const AttendArgs& a) {
  const unsigned grid = a.batch.tokens * a.heads;
  switch (a.cache.head_dim) {
    case 64: attend_row_kernel<T, 64><<<grid, kAttendThreads, 0, env.stream>>>(a); break;
    case 128: attend_row_kernel<T, 128><<<grid, kAttendThreads, 0, env.stream>>>(a); break;
    case 256: attend_row_kernel<T, 256><<<grid, kAttendThreads, 0, env.stream>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attend(const LaunchEnv& env, const AttendArgs& a, int* launches) {
  *launches = 1;
  if (a.dtype == KQ_F32) return attend_as<float>(env, a);
  if (a.dtype == KQ_F16) return attend_as<__half>(env, a);
  return attend_as<__nv_bfloat16>(env, a);
}

}  // namespace kq
