// Rotary positions, and rows into and out of the paged 4-bit cache (layout in kq_cache.cuh).
//
//   rope    (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) for the pairs of a head
//   append  key rows rotated, then each row of D values as codes 0..15 with a binary16 scale and offset
//   read    the f32 values that rows stand for
//
// All three are bound by memory: a value is read once and written once.  Measured: 8191 tokens of 32 heads of 128, bfloat16, half of
// each head rotated, 32.7 us (4.2 TB/s; the latency of loads that depend on one another: position, angles, values); one token 3.2 us,
// a launch.  Ten thousand rows appended and read back, 14.8 us; one row each of 64 sequences 7.2 us, two launches.
#include <algorithm>

#include "kq_cache.cuh"

namespace kq {
namespace {

constexpr int kThreads = 256;

// ---- rope -----------------------------------------------------------------------------------
// A thread owns one run of V values of a head (half layout: and the run it is paired with) and loops over heads with the
// angles in registers.
template <typename T, int V>
struct alignas(V * sizeof(T)) Run {
  T v[V];
};
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

struct RopeParams {
  const void* x;
  void* out;
  uint64_t x_stride, out_stride;
  const int* positions;
  RopeTable rope;
  uint32_t tokens, heads, dim;
  uint32_t units;        // runs (or pairs of runs) a head
  uint32_t head_groups;  // threads that share a token's heads for one unit
  bool wide;             // the table's rows can be read sixteen bytes at a time
};

template <int N>
__device__ __forceinline__ void load_angles(const float2* p, bool inside, bool wide, float2 (&cs)[N]) {
  if (!inside) {
#pragma unroll
    for (int i = 0; i < N; ++i) cs[i] = make_float2(quiet_nan(), quiet_nan());
  } else if (N % 2 == 0 && wide) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float4 v = reinterpret_cast<const float4*>(p)[i / 2];
      cs[i] = make_float2(v.x, v.y);
      if (i + 1 < N) cs[i + 1] = make_float2(v.z, v.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) cs[i] = p[i];
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rope_kernel(const RopeParams p) {
  using R = Run<T, V>;
  pdl_launch_dependents();
  const uint32_t across = min(p.units, static_cast<uint32_t>(kThreads)), slots = kThreads / across;  // (token, head group)s of a block
  const uint32_t slot = threadIdx.x / across, unit = blockIdx.y * kThreads + threadIdx.x - slot * across;
  const uint32_t at_slot = blockIdx.x * slots + slot, token = at_slot / p.head_groups, group = at_slot - token * p.head_groups;
  pdl_wait_prior_grid();
  if (slot >= slots || unit >= p.units || token >= p.tokens) return;
  const uint32_t half = p.rope.rotary / 2, turning = p.rope.interleaved && V > 1 ? p.rope.rotary / V : half / V;
  const T* x = static_cast<const T*>(p.x) + token * p.x_stride;
  T* out = static_cast<T*>(p.out) + token * p.out_stride;
  // What is behind the rotated part takes the same way and keeps its values: on a way of its own its lanes would wait for the
  // others of their warp (half of each head rotated: 45 us instead of 33).
  const bool turns = unit < turning;
  const int position = p.positions[token];
  const bool inside = position >= 0 && static_cast<uint32_t>(position) < p.rope.positions;
  const float2* row = p.rope.table + static_cast<size_t>(inside ? position : 0) * half;
  if constexpr (V > 1) {
    if (p.rope.interleaved) {
      float2 cs[V / 2];
      load_angles(row + (turns ? unit * (V / 2) : 0), inside, p.wide, cs);
#pragma unroll 4
      for (uint32_t h = group; h < p.heads; h += p.head_groups) {
        const size_t at = static_cast<size_t>(h) * p.dim + unit * V;
        R r = *reinterpret_cast<const R*>(x + at);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float2 y = rotate_pair(to_f32(r.v[i]), to_f32(r.v[i + 1]), cs[i / 2]);
          r.v[i] = turns ? from_f32<T>(y.x) : r.v[i];
          r.v[i + 1] = turns ? from_f32<T>(y.y) : r.v[i + 1];
        }
        *reinterpret_cast<R*>(out + at) = r;
      }
      return;
    }
  }
  // runs of V values and what they are paired with: rotary / 2 further on, or (interleaved, one value at a time) the next one
  const uint32_t pair = p.rope.interleaved ? 1 : half;
  const uint32_t first = !turns ? p.rope.rotary + (unit - turning) * V : unit * (p.rope.interleaved ? 2 : V);
  float2 cs[V];
  load_angles(row + (turns ? unit * V : 0), inside, p.wide, cs);
#pragma unroll 4
  for (uint32_t h = group; h < p.heads; h += p.head_groups) {
    const size_t at = static_cast<size_t>(h) * p.dim + first;
    R a = *reinterpret_cast<const R*>(x + at), b = a;
    if (turns) b = *reinterpret_cast<const R*>(x + at + pair);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 y = rotate_pair(to_f32(a.v[i]), to_f32(b.v[i]), cs[i]);
      a.v[i] = turns ? from_f32<T>(y.x) : a.v[i];
      b.v[i] = from_f32<T>(y.y);
    }
    *reinterpret_cast<R*>(out + at) = a;
    if (turns) *reinterpret_cast<R*>(out + at + pair) = b;
  }
}

// A launch that may begin while its predecessor drains (the kernels wait for it before they read anything).
template <typename Kernel, typename Params>
cudaError_t launch_overlapped(const LaunchEnv& env, Kernel kernel, dim3 grid, const Params& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T, int V>
cudaError_t rope_as(const LaunchEnv& env, RopeParams& p) {
  const uint32_t half = p.rope.rotary / 2;
  p.units = (p.rope.interleaved && V > 1 ? p.rope.rotary / V : half / V) + (p.dim - p.rope.rotary) / V;
  p.wide = (reinterpret_cast<uintptr_t>(p.rope.table) & 15u) == 0 && half % 2 == 0;
  // Heads a thread takes one after the other, the angles in registers: as many as leave the SMs full of threads
  const uint64_t units = static_cast<uint64_t>(p.tokens) * p.units;
  uint32_t each = 1;
  while (each < 8 && each < p.heads && units * (p.heads / (2 * each)) >= static_cast<uint64_t>(env.sm_count) * 2048) each *= 2;
  p.head_groups = (p.heads + each - 1) / each;
  const uint32_t across = std::min<uint32_t>(p.units, kThreads), slots = kThreads / across;
  const dim3 grid(static_cast<unsigned>((static_cast<uint64_t>(p.tokens) * p.head_groups + slots - 1) / slots), (p.units + kThreads - 1) / kThreads);
  return launch_overlapped(env, rope_kernel<T, V>, grid, p);
}

// The longest run, up to 16 bytes, that divides the rotated part, the rest of a head and every address.
template <typename T>
cudaError_t rope_of(const LaunchEnv& env, RopeParams& p) {
  const uint64_t part = p.rope.interleaved ? p.rope.rotary : p.rope.rotary / 2;
  const uint64_t all = part | p.dim | p.x_stride | p.out_stride | (reinterpret_cast<uint64_t>(p.x) | reinterpret_cast<uint64_t>(p.out)) / sizeof(T);
  if constexpr (sizeof(T) == 2)
    if (all % 8 == 0) return rope_as<T, 8>(env, p);
  if (all % 4 == 0) return rope_as<T, 4>(env, p);
  if (all % 2 == 0) return rope_as<T, 2>(env, p);
  return rope_as<T, 1>(env, p);
}

// ---- append and read ------------------------------------------------------------------------
// D / 8 neighbouring lanes hold a row, eight values each.
struct AppendParams {
  Cache cache;
  CacheBatch batch;
  RopeTable rope;
  const void *k, *v;
  uint64_t k_stride, v_stride;
};

// The row number of the calling lanes: token-major, then K rows, then V rows of the heads.
struct RowOf {
  uint32_t token, head;
  bool value;
};
__device__ __forceinline__ RowOf row_of(uint64_t row, uint32_t heads) {
  RowOf r;
  r.token = static_cast<uint32_t>(row / (2 * heads));
  const uint32_t in = static_cast<uint32_t>(row % (2 * heads));
  r.value = in >= heads;
  r.head = r.value ? in - heads : in;
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const AppendParams p) {
  constexpr int kLanes = D / 8;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t lane = threadIdx.x % kLanes;
  const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  const bool there = row < static_cast<uint64_t>(p.batch.tokens) * 2 * p.cache.kv_heads;
  const RowOf r = row_of(there ? row : 0, p.cache.kv_heads);
  const uint32_t seq = sequence_of(p.batch, r.token);
  const Span span = span_of(p.batch, seq);
  const int position = span.length - span.count + static_cast<int>(r.token) - span.first;
  const bool mine = there && static_cast<int>(r.token) >= span.first && static_cast<int>(r.token) < span.first + span.count && position >= 0;
  float x[8];
  const T* from = r.value ? static_cast<const T*>(p.v) + r.token * p.v_stride : static_cast<const T*>(p.k) + r.token * p.k_stride;
  from += r.head * D;
  if (r.value) load8(from + lane * 8, x);
  else load8_rotated(from, lane * 8, p.rope, position, x);
  float low = x[0], high = x[0];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
    nan |= x[i] != x[i];
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o /= 2) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    nan |= __shfl_xor_sync(0xffffffffu, static_cast<int>(nan), o) != 0;
  }
  __half offset = __float2half_rn(low);
  const float off = __half2float(offset);
  __half scale = __float2half_rn(__fmul_rn(__fsub_rn(high, off), 1.0f / 15.0f));
  float step = __half2float(scale);
  const bool lost = nan || isinf(off) || isinf(step) || step != step;
  if (lost) scale = offset = __ushort_as_half(0x7E00);
  else if (!(step > 0.0f)) scale = __ushort_as_half(0);
  uint32_t word = 0;
  if (!lost && step > 0.0f) {
    const float inv = __fdiv_rn(1.0f, step);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], off), inv)), 0.0f), 15.0f);
      word |= static_cast<uint32_t>(u) << (4 * i);
    }
  }
  if (!mine) return;
  const uint32_t P = p.cache.page_tokens, slot = static_cast<uint32_t>(position) % P;
  uint8_t* block = cache_block(p.cache, p.batch, seq, static_cast<uint32_t>(position) / P, r.head);
  if (!block) return;
  *reinterpret_cast<uint32_t*>(block + ((r.value ? P : 0u) + slot) * (D / 2) + lane * 4) = word;
  if (lane == 0) *reinterpret_cast<__half2*>(block + static_cast<size_t>(P) * D + ((r.value ? P : 0u) + slot) * 4) = __halves2half2(scale, offset);
}

struct ReadParams {
  Cache cache;
  CacheBatch batch;
  float *k, *v;
};

template <int D>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const ReadParams p) {
  constexpr int kLanes = D / 8;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t lane = threadIdx.x % kLanes;
  const uint64_t row = (static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  if (row >= static_cast<uint64_t>(p.batch.tokens) * 2 * p.cache.kv_heads) return;
  const RowOf r = row_of(row, p.cache.kv_heads);
  const uint32_t seq = sequence_of(p.batch, r.token);
  const Span span = span_of(p.batch, seq);
  const int position = span.length - span.count + static_cast<int>(r.token) - span.first;
  const bool mine = static_cast<int>(r.token) >= span.first && static_cast<int>(r.token) < span.first + span.count && position >= 0;
  const uint32_t P = p.cache.page_tokens, slot = static_cast<uint32_t>(position) % P;
  const uint8_t* block = mine ? cache_block(p.cache, p.batch, seq, static_cast<uint32_t>(position) / P, r.head) : nullptr;
  float scale = quiet_nan(), off = quiet_nan();
  uint32_t word = 0;
  if (block) {
    word = *reinterpret_cast<const uint32_t*>(block + ((r.value ? P : 0u) + slot) * (D / 2) + lane * 4);
    const __half2 so = *reinterpret_cast<const __half2*>(block + static_cast<size_t>(P) * D + ((r.value ? P : 0u) + slot) * 4);
    scale = __low2float(so);
    off = __high2float(so);
  }
  float4 o[2];
  float* f = reinterpret_cast<float*>(o);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = fmaf(static_cast<float>((word >> (4 * i)) & 15u), scale, off);
  float4* to = reinterpret_cast<float4*>((r.value ? p.v : p.k) + (static_cast<size_t>(r.token) * p.cache.kv_heads + r.head) * D + lane * 8);
  to[0] = o[0];
  to[1] = o[1];
}

unsigned blocks_for(const Cache& cache, const CacheBatch& batch) {
  const uint64_t threads = static_cast<uint64_t>(batch.tokens) * 2 * cache.kv_heads * (cache.head_dim / 8);
  return static_cast<unsigned>((threads + kThreads - 1) / kThreads);
}

template <typename T>
cudaError_t append_as(const LaunchEnv& env, const AppendParams& p) {
  const unsigned grid = blocks_for(p.cache, p.batch);
  switch (p.cache.head_dim) {
    case 64: return launch_overlapped(env, cache_append_kernel<T, 64>, grid, p);
    case 128: return launch_overlapped(env, cache_append_kernel<T, 128>, grid, p);
    case 256: return launch_overlapped(env, cache_append_kernel<T, 256>, grid, p);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_rope(const LaunchEnv& env, const void* x, int dtype, uint32_t tokens, uint32_t heads, uint32_t dim, uint64_t x_stride,
                        const int* positions, const RopeTable& rope, void* out, uint64_t out_stride) {
  RopeParams p = {x, out, x_stride, out_stride, positions, rope, tokens, heads, dim, 0, 0, false};
  if (dtype == KQ_F32) return rope_of<float>(env, p);
  if (dtype == KQ_F16) return rope_of<__half>(env, p);
  return rope_of<__nv_bfloat16>(env, p);
}

cudaError_t launch_cache_append(const LaunchEnv& env, const Cache& cache, const CacheBatch& batch, const void* k, uint64_t k_stride,
                                const void* v, uint64_t v_stride, int dtype, const RopeTable& rope) {
  const AppendParams p = {cache, batch, rope, k, v, k_stride, v_stride};
  if (dtype == KQ_F32) return append_as<float>(env, p);
  if (dtype == KQ_F16) return append_as<__half>(env, p);
  return append_as<__nv_bfloat16>(env, p);
}

cudaError_t launch_cache_read(const LaunchEnv& env, const Cache& cache, const CacheBatch& batch, float* k, float* v) {
  const ReadParams p = {cache, batch, k, v};
  const unsigned grid = blocks_for(cache, batch);
  switch (cache.head_dim) {
    case 64: return launch_overlapped(env, cache_read_kernel<64>, grid, p);
    case 128: return launch_overlapped(env, cache_read_kernel<128>, grid, p);
    case 256: return launch_overlapped(env, cache_read_kernel<256>, grid, p);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kq
