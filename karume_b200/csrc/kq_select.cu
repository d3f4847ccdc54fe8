// Which pages of a long sequence a query attends to: a summary of each page's keys, a cheap score of it, the pages with the largest.
//
//   summary  of a page and kv head, over the page's tokens, for each channel: c = (max + min) / 2, r = (max - min) / 2 of what the keys
//            stand for; both rows as 8-bit codes with a scale, by kq_quantize_rows' rule
//   score    a query held likewise (codes a, scale s): s ((a . c) s_c + (|a| . r) s_r), about the most that s a . k can be for the page's
//            keys; the largest of the query heads that share the kv head.  An estimate: codes are rounded to the nearest, so c may be off
//            by s_c / 2 and r short by s_r / 2 in each channel, and a key be above the score by up to s (sum |a|) (s_c + s_r) / 2
//   select   the first and last pages and, up to the budget, those with the largest scores, ties to the lower page
//
// What bounds them: at few rows the trips to memory one behind the other (lengths, page numbers, summaries or keys, and the queries beside them): a
// summary 5 us, scores and selection of 128 pages 8.5, of 3126 16. Of 64 rows, 8 kv heads and 320 pages: summaries 8 us, scores and selection 23 (43 MB
// of summaries, 1.9 TB/s).
//
// The dot products are of whole numbers, up to 127 * 127 * 256, which f32 holds exactly, and each of the few roundings behind them is
// part of the definition: which pages are selected does not depend on the order of any sum.
#include <algorithm>

#include "kq_cache.cuh"
#include "kq_select_geometry.h"

namespace kq {
namespace {

constexpr float kTiny = 1.17549435e-38f;

__device__ __forceinline__ float scale_of(float largest) { return fmaxf(__fmul_rn(largest, 1.0f / 127.0f), kTiny); }
__device__ __forceinline__ int code_of(float x, float scale) { return static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.0f), 127.0f)); }
__device__ __forceinline__ uint32_t pack4(const int* v) {
  return static_cast<uint32_t>(v[0] & 255) | static_cast<uint32_t>(v[1] & 255) << 8 | static_cast<uint32_t>(v[2] & 255) << 16 | static_cast<uint32_t>(v[3]) << 24;
}

// ---- summaries ------------------------------------------------------------------------------
struct SummaryParams {
  Cache cache;
  CacheBatch batch;
  Summaries to;
  uint32_t each;  // new tokens of a block
};

// A block for each kv head and `each` new tokens: those that are the first of the call in their page, one after the other.  Its warps share
// a page's tokens, all of whose loads are under way together: one warp for a page took 11 us for what takes 6.
constexpr int kSummaryThreads = 128;

template <int D>
__global__ void __launch_bounds__(kSummaryThreads) summarize_kernel(const SummaryParams p) {
  constexpr int kLanes = D / 8, kTokens = kSummaryThreads / kLanes;  // threads of a token (eight channels each), tokens at a time
  constexpr int kWarps = kSummaryThreads / 32;
  __shared__ float ends[kWarps][2][D];
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32, heads = p.cache.kv_heads, head = blockIdx.x % heads, first_row = blockIdx.x / heads * p.each;
  const int P = static_cast<int>(p.cache.page_tokens);
  for (uint32_t row = first_row; row < min(first_row + p.each, p.batch.tokens); ++row) {  // (the same for all threads)
    const uint32_t b = sequence_of(p.batch, row);
    const Span span = span_of(p.batch, b);
    const int in = static_cast<int>(row) - span.first, position = span.length - span.count + in;
    if (in < 0 || in >= span.count || position < 0 || (in != 0 && position % P != 0)) continue;
    const uint32_t index = static_cast<uint32_t>(position / P);
    const uint8_t* const block = cache_block(p.cache, p.batch, b, index, head);
    if (!block) continue;
    const int tokens = min(P, span.length - static_cast<int>(index) * P);
    const uint32_t channel = tid % kLanes * 8;
    float low[8], high[8];
    bool lost = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      low[i] = INFINITY;
      high[i] = -INFINITY;
    }
    constexpr int kBatch = 8;
    for (int t0 = static_cast<int>(tid / kLanes); t0 < tokens; t0 += kBatch * kTokens) {
      uint32_t words[kBatch], params[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int t = min(t0 + k * kTokens, tokens - 1);  // the last one again changes nothing
        words[k] = __ldg(reinterpret_cast<const uint32_t*>(block + t * (D / 2) + channel / 2));
        params[k] = __ldg(reinterpret_cast<const uint32_t*>(block + P * D + t * 4));
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float2 so = __half22float2(*reinterpret_cast<const __half2*>(&params[k]));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          constexpr float kWhole = 8388608.0f;  // 2^23: a code in its last bits
          const float u = __uint_as_float((words[k] >> (4 * i) & 15u) | 0x4B000000u) - kWhole;
          const float x = fmaf(u, so.x, so.y);
          low[i] = fminf(low[i], x);
          high[i] = fmaxf(high[i], x);
        }
        lost |= !(fabsf(so.x) <= 65504.0f && fabsf(so.y) <= 65504.0f);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int o = kLanes; o < 32; o *= 2) {
        low[i] = fminf(low[i], __shfl_xor_sync(0xffffffffu, low[i], o));
        high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], o));
      }
    if (lane < kLanes)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ends[warp][0][channel + i] = low[i];
        ends[warp][1][channel + i] = high[i];
      }
    lost = __syncthreads_or(lost);  // a key that is NaN, or of an infinite scale: nothing can be said of the page
    if (warp == 0) {
      float most_c = 0.0f, most_r = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float least = ends[0][0][channel + i], most = ends[0][1][channel + i];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          least = fminf(least, ends[w][0][channel + i]);
          most = fmaxf(most, ends[w][1][channel + i]);
        }
        low[i] = __fmul_rn(__fadd_rn(most, least), 0.5f);
        high[i] = __fmul_rn(__fsub_rn(most, least), 0.5f);
        most_c = fmaxf(most_c, fabsf(low[i]));
        most_r = fmaxf(most_r, high[i]);
      }
#pragma unroll
      for (int o = 1; o < kLanes; o *= 2) {
        most_c = fmaxf(most_c, __shfl_xor_sync(0xffffffffu, most_c, o));
        most_r = fmaxf(most_r, __shfl_xor_sync(0xffffffffu, most_r, o));
      }
      const float scale_c = scale_of(most_c), scale_r = scale_of(most_r);
      if (lane < kLanes) {
        int c[8], r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          c[i] = lost ? 0 : code_of(low[i], scale_c);
          r[i] = lost ? 0 : code_of(high[i], scale_r);
        }
        const size_t of = (static_cast<size_t>(block - p.cache.pool) / cache_block_bytes(p.cache.page_tokens, D)) * 2;  // page * heads + head, twice
        *reinterpret_cast<uint2*>(p.to.codes + of * D + channel) = make_uint2(pack4(c), pack4(c + 4));
        *reinterpret_cast<uint2*>(p.to.codes + (of + 1) * D + channel) = make_uint2(pack4(r), pack4(r + 4));
        if (lane == 0) *reinterpret_cast<float2*>(p.to.scales + of) = lost ? make_float2(quiet_nan(), quiet_nan()) : make_float2(scale_c, scale_r);
      }
    }
    __syncthreads();  // `ends` belongs to the next page
  }
}

// ---- scores ---------------------------------------------------------------------------------
struct SelectParams {
  AttendArgs a;
  Summaries from;
  uint32_t group, budget, first, last;
  uint32_t row0, rows;  // rows of this launch
  uint32_t chunks;      // blocks that share a row's pages,
  uint32_t turns;       // kScorePages of them each, so often
  unsigned int* arrived;  // fused: [rows][kv_heads] blocks that have made their scores, zero between launches; else null
  uint32_t* keys;       // [rows][kv_heads][table width]
  int* out;             // [tokens][kv_heads][budget]
};

// ---- the largest ----------------------------------------------------------------------------
// By a block: the budget-th largest key, digit by digit, then the pages above it in order.
constexpr uint32_t kAlways = 0xFFFFFFFFu, kUnknown = 0xFFFFFFFEu;
constexpr uint32_t kFusedPages = 1024;  // a list of so many is the work of the block that made its last scores

template <int kThreads, int kKept>
struct Largest {
  uint32_t kept[kKept];  // the first keys; the others are read again
  uint32_t count[256];
  uint32_t warps[kThreads / 32], chosen[2];
};
template <int kThreads, int kKept>
__device__ __forceinline__ void select_largest(Largest<kThreads, kKept>& s, const uint32_t* keys, uint32_t pages, uint32_t budget, int* out) {
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const auto key = [&](uint32_t i) { return i < kKept ? s.kept[i] : __ldcg(keys + i); };
  for (uint32_t i = tid; i < min(pages, static_cast<uint32_t>(kKept)); i += kThreads) s.kept[i] = __ldcg(keys + i);
  uint32_t digits = 0, left = budget;  // the digits found so far; how many of the keys that begin with them are taken
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (uint32_t i = tid; i < 256; i += kThreads) s.count[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < pages; i += kThreads) {
      const uint32_t k = key(i);
      if (shift == 24 || k >> (shift + 8) == digits) atomicAdd(&s.count[k >> shift & 255u], 1u);
    }
    __syncthreads();
    // keys of larger digits: a sum from the top
    // (two digits a thread in blocks of 128)
    constexpr uint32_t kDigits = kThreads < 256 ? 256 / kThreads : 1;
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t d = 0; d < kDigits; ++d)
      if (tid < 256) mine += s.count[255 - tid * kDigits - d];
    uint32_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += v;
    }
    if (lane == 31) s.warps[warp] = upto;
    __syncthreads();
    for (uint32_t i = 0; i < min(warp, 8u); ++i) upto += s.warps[i];
    if (tid < 256 && upto - mine < left && left <= upto) {
      uint32_t above = upto - mine;
#pragma unroll
      for (uint32_t d = 0; d < kDigits; ++d) {
        const uint32_t n = s.count[255 - tid * kDigits - d];
        if (above < left && left <= above + n) {
          s.chosen[0] = 255 - tid * kDigits - d;
          s.chosen[1] = left - above;
        }
        above += n;
      }
    }
    __syncthreads();
    digits = digits << 8 | s.chosen[0];
    left = s.chosen[1];
  }
  uint32_t before = 0, equal = 0;
  for (uint32_t i0 = 0; i0 < pages; i0 += kThreads) {
    const uint32_t i = i0 + tid, k = i < pages ? key(i) : 0u;
    const bool above = i < pages && k > digits, same = i < pages && k == digits;
    // both counts of the threads in front, sixteen bits each
    const uint32_t mine = (above ? 1u : 0u) | (same ? 0x10000u : 0u);
    const uint32_t a = __ballot_sync(0xffffffffu, above), e = __ballot_sync(0xffffffffu, same), in_front = (1u << lane) - 1;
    if (lane == 0) s.warps[warp] = __popc(a) | __popc(e) << 16;
    __syncthreads();
    uint32_t sum = __popc(a & in_front) | __popc(e & in_front) << 16, upto = lane < kThreads / 32 ? s.warps[lane] : 0;
#pragma unroll
    for (int o = 1; o < kThreads / 32; o *= 2) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += v;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, upto, kThreads / 32 - 1), front = __shfl_sync(0xffffffffu, upto, warp > 0 ? warp - 1 : 0);
    if (warp > 0) sum += front;
    __syncthreads();
    const uint32_t equal_before = equal + (sum >> 16);
    if (mine) {
      const uint32_t to = before + (sum & 0xFFFFu) + min(equal_before, left);
      if (above || equal_before < left) out[to] = static_cast<int>(i);
    }
    before += all & 0xFFFFu;
    equal += all >> 16;
  }
}

// ---- and the scores' kernel ----------------------------------------------------------------------
constexpr int kScoreWarps = 4, kScorePages = 16 * kScoreWarps;  // pages that a block takes at a time: sixteen a warp

// A number that is larger where the score is; not a number: larger than any.
__device__ __forceinline__ uint32_t key_of(float score) {
  const uint32_t bits = __float_as_uint(__fadd_rn(score, 0.0f));  // one zero
  if (score != score) return kUnknown;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The pages up to a row's position, or 0 where the row is no sequence's; and the sequence.
__device__ __forceinline__ int2 pages_of_row(const AttendArgs& a, uint32_t row) {
  const uint32_t b = sequence_of(a.batch, row);
  const Span s = span_of(a.batch, b);
  const int in = static_cast<int>(row) - s.first, position = s.length - s.count + in;
  if (in < 0 || in >= s.count || position < 0) return make_int2(0, static_cast<int>(b));
  return make_int2(static_cast<int>(min(static_cast<uint32_t>(position) / a.cache.page_tokens + 1, a.batch.width)), static_cast<int>(b));
}

template <typename T, int D>
__global__ void __launch_bounds__(kScoreWarps * 32, D == 256 ? 4 : 6) score_kernel(const __grid_constant__ SelectParams p) {
  constexpr int kHeads = 8;  // columns of an MMA
  __shared__ __align__(16) uint8_t codes[2][kHeads][D + 16];  // a, |a| (rows 16 bytes apart from a multiple of 128: lanes of eight rows meet no bank twice)
  __shared__ float scales[kHeads];
  __shared__ Largest<kScoreWarps * 32, kFusedPages> largest;
  __shared__ unsigned int arrivals;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4, heads = p.a.cache.kv_heads;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t chunk = blockIdx.x % p.chunks, at = blockIdx.x / p.chunks, head = at % heads, row = p.row0 + at / heads;
  const int2 of = pages_of_row(p.a, row);
  const int pages = of.x, first = static_cast<int>(chunk * p.turns) * kScorePages;
  int* const out = p.out + (static_cast<size_t>(row) * heads + head) * p.budget;
  if (pages <= static_cast<int>(p.budget)) {  // all are taken
    if (p.arrived && chunk == 0)
      for (uint32_t i = threadIdx.x; i < p.budget; i += kScoreWarps * 32) out[i] = static_cast<int>(i) < pages ? static_cast<int>(i) : -1;
    return;
  }
  if (first >= pages) return;
  uint32_t* const keys = p.keys + static_cast<size_t>(at) * p.a.batch.width;
  const int* const table = p.a.batch.pages + static_cast<size_t>(of.y) * p.a.batch.width;
  // sixteen pages: rows g and g + 8 of the MMA, sixteen channels of 64 a lane; the order of the channels is the queries' too
  constexpr int kWide = D / 64;
  uint4 x[2][2][kWide];  // [row][c, r][channels]
  float2 by[2];
  uint32_t number[2];  // of the pages that are loaded next
  const auto look = [&](int base) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int index = base + static_cast<int>(g) + i * 8;
      number[i] = index < pages ? static_cast<uint32_t>(__ldg(table + index)) : 0xFFFFFFFFu;
    }
  };
  const auto load = [&] {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t page = number[i];
      const bool there = page < p.a.cache.pages;
      const size_t place = (static_cast<size_t>(there ? page : 0) * heads + head) * 2;
      by[i] = there ? __ldg(reinterpret_cast<const float2*>(p.from.scales + place)) : make_float2(quiet_nan(), quiet_nan());
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int j = 0; j < kWide; ++j) x[i][which][j] = __ldg(reinterpret_cast<const uint4*>(p.from.codes + (place + which) * D + t * 16 + j * 64));
    }
  };
  int base = first + static_cast<int>(warp) * 16;
  look(base);
  load();  // while the queries are worked on
  if (p.turns > 1) look(base + kScorePages);
  const int position = place_of_row(p.a.batch, row).x;
  const uint32_t blocks = (p.group + kHeads - 1) / kHeads;
  float best[2];
  bool unknown[2];
  const uint32_t turns = min(p.turns, static_cast<uint32_t>(pages - first + kScorePages - 1) / kScorePages);  // that have pages
  for (uint32_t turn = 0; turn < turns; ++turn, base += kScorePages) {
    if (turn) {
      load();
      if (turn + 1 < turns) look(base + kScorePages);
    }
    best[0] = best[1] = -INFINITY;
    unknown[0] = unknown[1] = false;
    for (uint32_t h0 = 0; h0 < p.group; h0 += kHeads) {
      if (turn == 0 || blocks > 1) {
        if (turn || h0) __syncthreads();
        for (uint32_t h = warp; h < min(static_cast<uint32_t>(kHeads), p.group - h0); h += kScoreWarps) {  // a query head a warp (other columns hold anything)
          float v[8] = {};
          if (lane < D / 8)
            load8_rotated(static_cast<const T*>(p.a.q) + static_cast<size_t>(row) * p.a.q_stride + static_cast<size_t>(head * p.group + h0 + h) * D, lane * 8, p.a.rope,
                          position, v);
          float most = 0.0f;
          bool lost = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            most = fmaxf(most, fabsf(v[i]));
            lost |= !(fabsf(v[i]) < INFINITY);
          }
#pragma unroll
          for (int o = 16; o > 0; o /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          lost = __any_sync(0xffffffffu, lost);
          const float scale = scale_of(most);
          int a[8], m[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] = lost ? 0 : code_of(v[i], scale);
            m[i] = abs(a[i]);
          }
          if (lane < D / 8) {
            *reinterpret_cast<uint2*>(&codes[0][h][lane * 8]) = make_uint2(pack4(a), pack4(a + 4));
            *reinterpret_cast<uint2*>(&codes[1][h][lane * 8]) = make_uint2(pack4(m), pack4(m + 4));
          }
          if (lane == 0) scales[h] = lost ? quiet_nan() : scale;
        }
        __syncthreads();
      }
      int acc[2][4] = {};
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int j = 0; j < kWide; ++j) {
          const uint4 q = *reinterpret_cast<const uint4*>(&codes[which][g][j * 64 + t * 16]);
          mma_s8(acc[which], x[0][which][j].x, x[1][which][j].x, x[0][which][j].y, x[1][which][j].y, q.x, q.y);
          mma_s8(acc[which], x[0][which][j].z, x[1][which][j].z, x[0][which][j].w, x[1][which][j].w, q.z, q.w);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t h = 2 * t + k;
          if (h0 + h >= p.group) continue;
          const float sum = __fadd_rn(__fmul_rn(static_cast<float>(acc[0][2 * i + k]), by[i].x), __fmul_rn(static_cast<float>(acc[1][2 * i + k]), by[i].y));
          const float score = __fmul_rn(sum, scales[h]);
          unknown[i] |= score != score;
          best[i] = fmaxf(best[i], score);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 1; o < 4; o *= 2) {
        best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], o));
        unknown[i] |= __shfl_xor_sync(0xffffffffu, static_cast<int>(unknown[i]), o) != 0;
      }
      const int index = base + static_cast<int>(g) + i * 8;
      if (t == 0 && index < pages)
        keys[index] = index < static_cast<int>(p.first) || index >= pages - static_cast<int>(p.last) ? kAlways : unknown[i] ? kUnknown : key_of(best[i]);
    }
  }
  if (!p.arrived) return;
  // the block that is the last one of the row's selects
  const unsigned int blocks_here = (static_cast<uint32_t>(pages) + p.turns * kScorePages - 1) / (p.turns * kScorePages);
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned int* const counter = p.arrived + at;
    unsigned int before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
    if (before == blocks_here - 1) *counter = 0;
    arrivals = before;
  }
  __syncthreads();
  if (arrivals == blocks_here - 1) select_largest(largest, keys, static_cast<uint32_t>(pages), p.budget, out);
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ SelectParams p) {
  __shared__ Largest<kThreads, 8192> s;
  const uint32_t heads = p.a.cache.kv_heads;
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t row = p.row0 + blockIdx.x / heads;
  const uint32_t pages = static_cast<uint32_t>(pages_of_row(p.a, row).x);
  int* const out = p.out + (static_cast<size_t>(row) * heads + blockIdx.x % heads) * p.budget;
  if (pages <= p.budget) {
    for (uint32_t i = threadIdx.x; i < p.budget; i += kThreads) out[i] = i < pages ? static_cast<int>(i) : -1;
    return;
  }
  select_largest(s, p.keys + static_cast<size_t>(blockIdx.x) * p.a.batch.width, pages, p.budget, out);
}

template <typename Kernel, typename Params>
cudaError_t launch_after(const LaunchEnv& env, Kernel kernel, uint64_t grid, int threads, const Params& p) {
  if (grid > select::kMostBlocks) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t score_as(const LaunchEnv& env, const SelectParams& p) {
  const uint64_t grid = static_cast<uint64_t>(p.rows) * p.a.cache.kv_heads * p.chunks;
  switch (p.a.cache.head_dim) {
    case 64: return launch_after(env, score_kernel<T, 64>, grid, kScoreWarps * 32, p);
    case 128: return launch_after(env, score_kernel<T, 128>, grid, kScoreWarps * 32, p);
    case 256: return launch_after(env, score_kernel<T, 256>, grid, kScoreWarps * 32, p);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_summarize(const LaunchEnv& env, const Cache& cache, const CacheBatch& batch, const Summaries& to) {
  const SummaryParams p = {cache, batch, to, select::summary_rows(batch.tokens, cache.kv_heads, !batch.starts)};
  const uint64_t grid = select::summary_blocks(batch.tokens, cache.kv_heads, p.each);
  switch (cache.head_dim) {
    case 64: return launch_after(env, summarize_kernel<64>, grid, kSummaryThreads, p);
    case 128: return launch_after(env, summarize_kernel<128>, grid, kSummaryThreads, p);
    case 256: return launch_after(env, summarize_kernel<256>, grid, kSummaryThreads, p);
    default: return cudaErrorInvalidValue;
  }
}

uint64_t select_scratch_bytes(const AttendArgs& a) { return 4ull * a.cache.kv_heads * a.batch.width; }

cudaError_t launch_select(const LaunchEnv& env, const AttendArgs& a, const Summaries& from, uint32_t budget, uint32_t first, uint32_t last, int* out, int* launches) {
  SelectParams p;
  p.a = a;
  p.from = from;
  p.group = a.heads / a.cache.kv_heads;
  p.budget = budget;
  p.first = first;
  p.last = last;
  p.keys = static_cast<uint32_t*>(env.workspace);
  p.out = out;
  // a block quantises its queries once: it takes more pages where there are blocks enough for all SMs, six each at a time (64 rows, 8 kv heads,
  // 320 pages each: two waves of blocks of eight warps 26 us, one of four warps 19)
  const uint64_t blocks = static_cast<uint64_t>(a.batch.tokens) * a.cache.kv_heads, most = (a.batch.width + kScorePages - 1) / kScorePages;
  p.turns = static_cast<uint32_t>(std::min<uint64_t>({std::max<uint64_t>((blocks * most + 6ull * env.sm_count - 1) / (6ull * env.sm_count), 1), most, 32}));
  p.chunks = static_cast<uint32_t>((most + p.turns - 1) / p.turns);
  p.turns = static_cast<uint32_t>((most + p.chunks - 1) / p.chunks);  // even shares
  *launches = 0;
  // as many rows at a time as have room in the scratch and in a grid
  const bool fused = a.batch.width <= kFusedPages;
  uint64_t room = std::min<uint64_t>(env.workspace_bytes / select_scratch_bytes(a), ((1ull << 31) - 1) / (static_cast<uint64_t>(a.cache.kv_heads) * p.chunks));
  if (fused) room = std::min<uint64_t>(room, env.counter_count / a.cache.kv_heads);
  p.arrived = fused && env.counter_count >= a.cache.kv_heads ? env.counters : nullptr;
  for (uint32_t row = 0; row < a.batch.tokens; row += p.rows) {
    p.row0 = row;
    p.rows = static_cast<uint32_t>(std::min<uint64_t>(a.batch.tokens - row, std::max<uint64_t>(room, 1)));
    cudaError_t e = a.dtype == KQ_F32 ? score_as<float>(env, p) : a.dtype == KQ_F16 ? score_as<__half>(env, p) : score_as<__nv_bfloat16>(env, p);
    *launches += 1;
    if (e != cudaSuccess) return e;
    if (p.arrived) continue;
    e = launch_after(env, select_kernel<1024>, static_cast<uint64_t>(p.rows) * a.cache.kv_heads, 1024, p);
    *launches += 1;
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace kq
