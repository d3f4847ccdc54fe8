// The paged 4-bit cache: addressing, the sequences of a call, and what a row stands for.  Shared by the kernels that
// append to it, read it back and attend over it.
//
// A page of P tokens holds, for each kv head, one contiguous block of P * (D + 8) bytes:
//   [K codes: P x D/2][V codes: P x D/2][K (scale, offset): P x 2 binary16][V (scale, offset): P x 2 binary16]
// so that any run of tokens of a page is four contiguous pieces whose sizes are multiples of 16 bytes from 16 tokens up
// (asynchronous bulk copies).  Code u of a row stands for fround(u * scale + offset): u * scale is exact in f32.
#pragma once

#include "kq_common.cuh"
#include "kq_internal.h"

namespace kq {

__host__ __device__ __forceinline__ uint64_t cache_block_bytes(uint32_t page_tokens, uint32_t dim) {
  return static_cast<uint64_t>(page_tokens) * (dim + 8u);
}

// Page `index` of sequence b, or null where the table or the pool has none.
__device__ __forceinline__ uint8_t* cache_block(const Cache& c, const CacheBatch& batch, uint32_t b, uint32_t index, uint32_t head) {
  if (index >= batch.width) return nullptr;
  const uint32_t page = static_cast<uint32_t>(batch.pages[static_cast<size_t>(b) * batch.width + index]);
  if (page >= c.pages) return nullptr;  // a negative number too
  return c.pool + (static_cast<uint64_t>(page) * c.kv_heads + head) * cache_block_bytes(c.page_tokens, c.head_dim);
}

// The new tokens of sequence b: rows first .. first + count of the call, positions length - count + i.
struct Span {
  int first, count, length;
};
__device__ __forceinline__ Span span_of(const CacheBatch& batch, uint32_t b) {
  Span s;
  const int tokens = static_cast<int>(batch.tokens);
  s.length = max(batch.lengths[b], 0);
  if (batch.starts) {
    s.first = min(max(batch.starts[b], 0), tokens);
    s.count = min(max(batch.starts[b + 1], s.first), tokens) - s.first;
  } else {
    s.first = static_cast<int>(b);
    s.count = static_cast<int>(b) < tokens ? 1 : 0;
  }
  return s;
}
// The sequence of a row, by halving over the ascending starts: the last b with starts[b] <= row.
__device__ __forceinline__ uint32_t sequence_of(const CacheBatch& batch, uint32_t row) {
  if (!batch.starts) return row;
  uint32_t lo = 0, hi = batch.sequences;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (batch.starts[mid] <= static_cast<int>(row)) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The rotation of one pair, every product and sum rounded to f32 (what a key is held as does not depend on the kernel).
__device__ __forceinline__ float2 rotate_pair(float x0, float x1, float2 cs) {
  return make_float2(__fsub_rn(__fmul_rn(x0, cs.x), __fmul_rn(x1, cs.y)), __fadd_rn(__fmul_rn(x1, cs.x), __fmul_rn(x0, cs.y)));
}
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7FC00000); }

// Eight consecutive values as f32, 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const T* h = reinterpret_cast<const T*>(&a);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(h[i]);
}

// Values at .. at + 8 of a head's row (`row` its first value), rotated for `position`; at is a multiple of eight.
template <typename T>
__device__ __forceinline__ void load8_rotated(const T* row, uint32_t at, const RopeTable& rope, int position, float (&v)[8]) {
  load8(row + at, v);
  if (!rope.table || at >= rope.rotary) return;
  if (position < 0 || static_cast<uint32_t>(position) >= rope.positions) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i < rope.rotary) v[i] = quiet_nan();
    return;
  }
  const uint32_t half = rope.rotary / 2;
  const float2* cs = rope.table + static_cast<size_t>(position) * half;
  if (rope.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      if (at + i >= rope.rotary) break;  // rotary is even
      const float2 r = rotate_pair(v[i], v[i + 1], cs[(at + i) / 2]);
      v[i] = r.x;
      v[i + 1] = r.y;
    }
    return;
  }
  float other[8];
  if (half % 8 == 0) {
    load8(row + (at < half ? at + half : at - half), other);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = at < half ? rotate_pair(v[i], other[i], cs[at + i]).x : rotate_pair(other[i], v[i], cs[at + i - half]).y;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = at + i;
    if (e >= rope.rotary) break;
    v[i] = e < half ? rotate_pair(v[i], to_f32(row[e + half]), cs[e]).x : rotate_pair(to_f32(row[e - half]), v[i], cs[e - half]).y;
  }
}

// Half layout with angles that can be read sixteen bytes at a time.
__host__ __device__ __forceinline__ bool rope_is_plain(const RopeTable& rope) {
  return rope.table && !rope.interleaved && rope.rotary % 4 == 0 && (reinterpret_cast<uintptr_t>(rope.table) & 15u) == 0 && rope.positions > 0;
}

}  // namespace kq
