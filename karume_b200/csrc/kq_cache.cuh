// The paged 4-bit cache: addressing, the sequences of a call, and what a row stands for.  Shared by the kernels that
// append to it, read it back and attend over it.
//
// A page of P tokens holds, for each kv head, one contiguous block of P * (D + 8) bytes:
//   [K codes: P x D/2][V codes: P x D/2][K (scale, offset): P x 2 binary16][V (scale, offset): P x 2 binary16]
// so that any run of tokens of a page is four contiguous pieces whose sizes are multiples of 16 bytes from 16 tokens up
// (asynchronous bulk copies).  Code u of a row stands for fround(u * scale + offset): u * scale is exact in f32.
#pragma once

#include "kq_common.cuh"
#include "kq_groups.h"
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

// Position of the sequence's token that row `row` of the call is, and how many tokens the sequence has in front of its new ones.
__device__ __forceinline__ int2 place_of_row(const CacheBatch& batch, uint32_t row) {
  const Span s = span_of(batch, sequence_of(batch, row));
  const int before = s.length - s.count;
  return make_int2(before + static_cast<int>(row) - s.first, max(before, 0));
}

// ---- sequences that begin alike ---------------------------------------------------------------
// By a warp: whether reading what the groups have in common once saves enough (the other way re-reads it, mostly from L2).  Not where their
// boundaries are out of order: groups with rows in common would ask for more blocks than there are.  (`starts` are looked at last: a trip to memory
// behind the boundaries, 1.4 us of a call that saves nothing.)
__device__ __forceinline__ bool worth_sharing(const AttendArgs& a, const SharedArgs& sh) {
  unsigned long long keys = 0;
  bool ordered = true;
  for (uint32_t g = threadIdx.x % 32; g < sh.all_groups; g += 32) {
    const int first = __ldg(sh.all_first + g), next = __ldg(sh.all_first + g + 1);
    ordered &= first <= next;
    const long long members = static_cast<long long>(next) - first;
    unsigned tokens = static_cast<unsigned>(max(__ldg(sh.all_tokens + g), 0));
    if (a.window) tokens = min(tokens, a.window);
    if (members > 1) keys += static_cast<unsigned long long>(members - 1) * tokens;
  }
#pragma unroll
  for (int o = 16; o > 0; o /= 2) keys += __shfl_xor_sync(0xffffffffu, keys, o);
  if (!__all_sync(0xffffffffu, ordered) || keys * (a.cache.kv_heads * (a.cache.head_dim + 8u)) < sh.least) return false;
  if (!a.batch.starts) return true;
  for (uint32_t g = threadIdx.x % 32; g < sh.all_groups; g += 32)
    ordered &= groups::in_order(__ldg(sh.all_first + g), __ldg(sh.all_first + g + 1), a.batch.starts, static_cast<int>(a.batch.sequences),
                                static_cast<int>(a.batch.tokens));
  return __all_sync(0xffffffffu, ordered);
}
// How many keys sequence b has in common with its group, all of them in front of its new tokens; 0 where it is in none.
__device__ __forceinline__ int common_keys(const CacheBatch& batch, const SharedArgs& sh, uint32_t b, const Span& span) {
  uint32_t lo = 0, hi = sh.groups;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (__ldg(sh.first + mid) <= static_cast<int>(b)) lo = mid;
    else hi = mid;
  }
  const int b0 = __ldg(sh.first + lo), b1 = __ldg(sh.first + lo + 1);
  if (b0 > static_cast<int>(b) || b1 <= static_cast<int>(b)) return 0;
  // Rows that are not among the group's (starts that do not ascend) have no sums over common keys.
  if (batch.starts && (batch.starts[max(b0, 0)] > span.first || batch.starts[min(b1, static_cast<int>(batch.sequences))] < span.first + span.count)) return 0;
  return min(max(__ldcg(sh.keys + lo), 0), max(span.length - span.count, 0));
}
// By a warp: the new rows of group g's sequences (first, number), the keys that any of them has in common, the first of these that a row
// sees; every: first and last of the keys that all the rows see; lead: the member through whose row of the page table they are read, and how many
// keys the group has at most.  Members that ended or were cut back have fewer tokens than the others, so this is the first of 32 that has all
// that are said to be common, else the first that has any; what it has not is each other one's own.
__device__ __forceinline__ int4 group_of_rows(const CacheBatch& batch, const SharedArgs& sh, uint32_t g, int window, int2& every, int2& lead) {
  const groups::Range members = groups::sequences_of(__ldg(sh.first + g), __ldg(sh.first + g + 1), static_cast<int>(batch.sequences));
  const groups::Range rows = groups::rows_of(members, batch.starts, static_cast<int>(batch.tokens));
  int least = 0x7fffffff, far = 0, last = -1;
  for (int b = members.begin + static_cast<int>(threadIdx.x % 32); b < members.end; b += 32) {
    const Span s = span_of(batch, static_cast<uint32_t>(b));
    if (s.count == 0) continue;
    least = min(least, s.length - s.count);
    far = max(far, s.length - s.count);
    last = max(last, s.length - 1);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  far = __reduce_max_sync(0xffffffffu, far);
  last = __reduce_max_sync(0xffffffffu, last);
  const int common = __ldg(sh.tokens + g), looked_at = members.begin + static_cast<int>(threadIdx.x % 32);
  const int tokens = looked_at < members.end ? max(batch.lengths[looked_at], 0) : 0;
  const uint32_t any = __ballot_sync(0xffffffffu, tokens > 0), all = __ballot_sync(0xffffffffu, tokens > 0 && tokens >= common);
  const int at = max(__ffs(static_cast<int>(all ? all : any)) - 1, 0);
  lead = make_int2(members.begin + at, min(max(common, 0), __shfl_sync(0xffffffffu, tokens, at)));
  const int keys = min(lead.y, far);
  // (a window may hide all of them: one is walked over all the same, so that the rows' sums are written)
  const int from = window && least >= window ? min(least - window + 1, max(keys - 1, 0)) : 0;
  every = make_int2(window && last >= window ? last - window + 1 : 0, min(keys, max(least, 0)) - 1);
  return make_int4(rows.begin, rows.end - rows.begin, keys, from);
}

__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7FC00000); }
__device__ __forceinline__ float power_of_two(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Four of the sums of a row, not divided yet, relative to 2^m, and the sum of its weights: joined with what the row sees of the common keys,
// which is at the row's place `at`.  A place that is none (a launch in front gave up waiting, and left the row's out) gives NaN.
constexpr uint32_t kMostParts = 1024;  // CTAs that share a row's common keys: no more than there are SMs
__device__ __forceinline__ void join_common(const SharedArgs& sh, const uint4& at, int quad, float& m, float& total, float (&v)[4]) {
  // (in units of four floats, of which the scratch has 2^31 at most)
  const uint32_t last = (at.w - 1) * (at.z / 4), end = max(at.x + quad, at.y / 2) + last;
  if (at.w - 1 >= kMostParts || at.z > (1u << 20) || at.x >= sh.quads || end >= sh.quads) {
    total = quiet_nan();
    return;
  }
  const float4* const sums = reinterpret_cast<const float4*>(sh.scratch) + at.x + quad;
  const float2* const stats = reinterpret_cast<const float2*>(sh.scratch) + at.y;
  constexpr uint32_t kBatch = 12;
  for (uint32_t j0 = 0; j0 < at.w; j0 += kBatch) {
    float2 ml[kBatch];
    float4 x[kBatch];
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      const size_t part = static_cast<size_t>(min(j0 + j, at.w - 1)) * at.z;
      ml[j] = __ldcg(stats + part / 2);
      x[j] = __ldcg(sums + part / 4);
    }
    float now = m;
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      if (j0 + j >= at.w) ml[j] = make_float2(-INFINITY, 0.0f);
      now = fmaxf(now, ml[j].x);
    }
    const float before = m == -INFINITY ? 0.0f : power_of_two(m - now);
    m = now;
    total *= before;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= before;
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      const float keep = ml[j].x == -INFINITY ? 0.0f : power_of_two(ml[j].x - m);
      total = fmaf(keep, ml[j].y, total);
      v[0] = fmaf(keep, x[j].x, v[0]);
      v[1] = fmaf(keep, x[j].y, v[1]);
      v[2] = fmaf(keep, x[j].z, v[2]);
      v[3] = fmaf(keep, x[j].w, v[3]);
    }
  }
}
// Where a row's sums go that are no part, and its pair.
__device__ __forceinline__ uint4 whole_place(const SharedArgs& sh, const AttendArgs& a, size_t row) {
  const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * a.heads, dim = a.cache.head_dim;
  return make_uint4(static_cast<uint32_t>((sh.sums + row * dim) / 4), static_cast<uint32_t>((sh.sums + rows * dim) / 2 + row), 0u, 1u);
}

// ---- rows that attend to selected pages -------------------------------------------------------
// (sequence, position, keys, 0): the pages in the list's order, the last one up to the position; no keys where the row is no sequence's.
__device__ __forceinline__ int4 selected_row(const AttendArgs& a, const SelectedArgs& sel, uint32_t row) {
  const uint32_t b = sequence_of(a.batch, row);
  const Span s = span_of(a.batch, b);
  const int in = static_cast<int>(row) - s.first, position = s.length - s.count + in;
  if (in < 0 || in >= s.count || position < 0) return make_int4(static_cast<int>(b), position, 0, 0);
  const int page_tokens = static_cast<int>(a.cache.page_tokens), pages = static_cast<int>(min(sel.budget, static_cast<uint32_t>(position / page_tokens) + 1));
  return make_int4(static_cast<int>(b), position, (pages - 1) * page_tokens + position % page_tokens + 1, 0);
}
// The number of the row's index-th page for a kv head; no page's where the list or the table has none.
__device__ __forceinline__ uint32_t selected_page(const AttendArgs& a, const SelectedArgs& sel, uint32_t row, uint32_t head, int sequence, uint32_t index) {
  const uint32_t at = static_cast<uint32_t>(__ldg(sel.pages + (static_cast<size_t>(row) * a.cache.kv_heads + head) * sel.budget + index));
  return at < a.batch.width ? static_cast<uint32_t>(__ldg(a.batch.pages + static_cast<size_t>(sequence) * a.batch.width + at)) : 0xFFFFFFFFu;
}

// The rotation of one pair, every product and sum rounded to f32 (what a key is held as does not depend on the kernel).
__device__ __forceinline__ float2 rotate_pair(float x0, float x1, float2 cs) {
  return make_float2(__fsub_rn(__fmul_rn(x0, cs.x), __fmul_rn(x1, cs.y)), __fadd_rn(__fmul_rn(x1, cs.x), __fmul_rn(x0, cs.y)));
}

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
