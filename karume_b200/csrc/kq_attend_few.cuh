// Attention over the paged 4-bit cache (layout in kq_cache.cuh) for few query rows a sequence: single tokens, drafts.
//
//   out = sum_j softmax_j(scale q . k_j) v_j,   k_j = u_j s_j + o_j, v_j likewise, codes u in 0..15
//
// The cache is read once, so the floor is its bytes; what the kernel is built around is that a code must cost few
// instructions on its way into the tensor cores.  (w & 0x000F000F) of a word of eight codes IS a pair of binary16 numbers,
// the subnormals u 2^-24, and (w & 0x00F000F0) the pair u 2^-20: no conversion, the powers of two are taken out of q and of
// the output.  Scores and outputs are built transposed, keys and values as the M side of mma.m16n8k16:
//
//   S^T [16 tokens, 8 columns] += K [16, 16 dims] q^T      a thread's words of a token are its A fragments
//   O^T [16 dims, 8 columns]   += V^T [16, 16 tokens] P^T  the words of two tokens, joined by two PRMTs
//
// A column is one query row (query and head of the kv head's group) for 16-bit queries; f32 queries are two binary16
// parts in neighbouring columns (fixed-point, exact sums), and so are their weights; the parts' sums are added in f32.  The weights
// get from S^T's fragment to the B fragment of P^T by one movmatrix a 8 x 8 block, nothing passes through shared memory.
//
//   score    s_j = scale log2(e) (s_j (q . u_j) + o_j sum q)            (base 2, f32; the sum of q as it is multiplied)
//   weight   p_j = 2^(s_j - M), and P = p_j s'_j (s' the value's scale) is what enters the tensor core.  M follows the
//            largest s_j + log2 of s'_j's binade, and moves only when a weight would grow past 2^8 of it: P fits binary16
//            with its full precision wherever it matters, whatever the size of the values.  16-bit queries round P to binary16
//            once (with the rotated queries, 2.9e-4 to 3.9e-4 of an f16 result; its own rounding is 2.1e-4); f32 ones keep two parts of eleven bits.
//   output   sum_j P_j (u'_j - 7.5) + sum_j p_j (o'_j + 7.5 s'_j): codes around zero, because sums of many uncentred
//            ones cancel (70001 keys: 1e-3 of the result was lost); f32 queries add each tile's sums in registers,
//            where the tensor core's own chain would truncate.
//
// Work: every (sequence, kv head, block of query rows) is a run of tiles of 32 or 64 tokens.  All runs of the call, laid end to
// end, are cut into equal ranges, one for each CTA (two to four CTAs an SM), by what the lengths say on the device: ragged batches
// and one long sequence fill the machine alike, and a recorded launch follows the lengths.  The warps of a CTA take the
// tiles in turn, each with a ring of its own that bulk copies fill (page by page: K codes, V codes, scales).  A run that
// several CTAs share leaves partial sums in the scratch; the last CTA of sixteen neighbours joins theirs in order, the last of
// those groups the groups'.
//
// What bounds it: the latency of its own instructions.  A code costs a masked shift, one operation around zero and its share of an MMA, a
// (row, key) pair an exponential and some ten more, and two warps a scheduler, which is what registers leave, do not hide how long
// they take: at 64 bfloat16 sequences of 32 heads over 8, up to 16384 tokens, 160 us (4.3 TB/s, 0.65 of the copy rate), issue slots and the
// fullest pipe are at 49 %.  16 f32 sequences up to 8190 tokens: 34 us (2.5 TB/s); one sequence of 200003, two kv heads: 29 us;
// one of 4096: 10.3 us, where the launch, the cut, the queries and the joining are most of it.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kq_cache.cuh"

namespace kq {
namespace {

constexpr uint32_t kFewWaitLimit = 1u << 22;
constexpr int kFewTimeout = 40;      // status word: a copy of the cache did not arrive

// What a run of the list is.
//   kWhole     a sequence's new rows and all keys they see
//   kShared    prefix: the new rows of a group of sequences and the keys that the group has in common, read through one member's
//              pages; the sums go to `sh`.  Rest: a sequence's new rows and the keys behind those, joined with the sums
//   kSelected  one new row and the tokens of the pages selected for it (and a kv head), in the order of the list, as if they were a sequence
enum FewMode { kWhole, kShared, kSelected };

// ---- shapes of one instance -------------------------------------------------------------------
// kPair: a query row has two neighbouring columns of an n-tile, so that a thread works on one row: the parts of f32 queries,
// or one 16-bit query and nothing (four rows or fewer: half the softmax work of two rows a thread).  Otherwise a column each.
template <typename T, int D, int NT, bool kPair, int kMode>
struct Few {
  static constexpr bool kSplit = sizeof(T) == 4;
  static_assert(kPair || !kSplit, "f32 queries are pairs of parts");
  // Tokens a warp takes at a time.  What a tile costs whatever its size (the wait, the next copies, the check of M) is a third
  // of 32 tokens' instructions: 64 of them gain 10 % where registers and shared memory leave room (64 sequences, bf16: 169 -> 152 us),
  // and lose as much on the wide forms.
  static constexpr int kTile = NT == 1 && D <= 128 ? 64 : 32;
  static constexpr int kSubs = kTile / 16;
  static constexpr int kOf = kPair ? 4 : 8;          // query rows of an n-tile
  static constexpr int kRows = kOf * NT;             // ... and of a block
  static constexpr int kWarps = 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = 2;
  static constexpr int kSteps = D / 16;              // k-steps of S^T
  static constexpr int kWords = D / 32;              // words of a token in a thread (keys)
  static constexpr int kVWords = D / 64;             // ... (values)
  static constexpr int kTileBytes = kTile * (D + 8);
  static constexpr bool kQInRegisters = NT * kSteps <= 16;
  static constexpr int kPartFloats = kRows * (D + 2);  // a partial result in the scratch: sums, M, l
  static constexpr int kShort = 512 / kTile;                    // tiles of a run that is not shared by CTAs
  // What a run costs whatever its length (its queries, joining its warps, what it has in common: 5 to 6 us), in tiles: a range of the list is
  // cut by both.  (64 sequences of up to 1024 tokens behind common ones, by tiles alone: the last CTA ended after 45 us, the mean one after 26.
  // Two whole f32 sequences of 1100: 11.9 us, by tiles alone 16.3, where short ranges reach from one run into the next.)
  // Whole sequences are cut by tiles, and selections, which are alike.
  static constexpr int kHead = kMode == kShared ? 640 / kTile : 0;
  static constexpr int kSpans = 128;                   // sequences whose lengths are kept in shared memory
  static_assert(kMode != kShared || kSpans >= static_cast<int>(groups::kAtOnce), "a place for every group of a launch");

  static constexpr int kRing = 0;
  static constexpr int kMerge = kRing + kWarps * kStages * kTileBytes;
  static constexpr int kQFrag = kMerge + kWarps * kRows * D * 4;       // [NT][kSteps][32] x 8 B
  static constexpr int kRowConst = kQFrag + NT * kSteps * 32 * 8;      // factor, offset, last key, first key of each row
  static constexpr int kWarpStat = kRowConst + kRows * 16;             // [kWarps][kRows] x (M, l, centre sum)
  static constexpr int kScan = kWarpStat + (kWarps * kRows * 12 + 15) / 16 * 16;  // sums of the warps, what the scan found
  static constexpr int kSpan = kScan + kWarps * 8 + 32 + kWarps * 8;
  static constexpr int kAll = kSpan + kSpans * 16;     // kShared: keys that every row of a group sees
  static constexpr int kLead = kAll + (kMode == kShared ? kSpans * 8 : 0);  // ... and through whose pages they are read
  static constexpr int kBars = kLead + (kMode == kShared ? kSpans * 4 : 0);
  static constexpr int kMisc = kBars + kWarps * kStages * 8;
  static constexpr int kSmem = kMisc + 16;
  // CTAs of an SM: what waits in one is hidden by the others; as many as registers and shared memory allow
  static constexpr int kFit = 228 * 1024 / (kSmem + 1024);
  static constexpr int kCtas = NT == 1 && D <= 128 ? (kFit < 4 ? kFit : 4) : (kFit < 2 ? kFit : 2);
};

struct FewParams {
  AttendArgs a;
  uint32_t group;          // query heads of a kv head
  uint32_t page_shift;     // log2 of a page's tokens
  float* parts;            // [4 * grid][kPartFloats]: two of a CTA, and two of the groups that begin with it
  unsigned int* counters;  // [3 * grid], zero between launches
  int* status;
  uint32_t beyond;         // sequences of more query rows a kv head are another kernel's
  bool prefix;             // kShared: the groups' common keys, else the sequences' own
  SharedArgs sh;
  SelectedArgs sel;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(__half lo, __half hi) {
  return static_cast<uint32_t>(__half_as_ushort(lo)) | (static_cast<uint32_t>(__half_as_ushort(hi)) << 16);
}
__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hadd2_u(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]);
template <>
__device__ __forceinline__ void store4<float>(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
template <>
__device__ __forceinline__ void store4<__half>(__half* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_half2(__float2half_rn(v[0]), __float2half_rn(v[1])), pack_half2(__float2half_rn(v[2]), __float2half_rn(v[3])));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[4]) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// ---- the work list --------------------------------------------------------------------------
// A sequence's runs: `units` = kv heads x blocks of rows, each of `tiles` tiles from tile_lo on.
// Its row of the list, in shared memory too: first row and number of them, keys, and
//   kShared  rest: how many keys it has in common; prefix: the first key that one of its rows sees
//   kSelected  (sequence, position, keys, -): the row's own number is that in the list
struct Runs {
  Span span;
  int low;                    // the list's fourth number
  int sequence, position;     // kSelected
  int tile_lo, tiles;
  uint32_t blocks, units;
};
template <int kMode>
__device__ __forceinline__ Runs runs_of(const FewParams& p, const int4& item, uint32_t number, int rows, int tile) {
  Runs r;
  r.span = Span{item.x, item.y, item.z};
  r.low = kMode == kWhole ? 0 : item.w;
  if constexpr (kMode == kSelected) {
    r.span = Span{static_cast<int>(number), 1, item.z};
    r.sequence = item.x;
    r.position = item.y;
  }
  int from = 0;
  if (kMode == kShared && p.prefix) {
    from = r.low;
  } else if constexpr (kMode != kSelected) {
    const int first = r.span.length - r.span.count;  // position of the first query
    const int window = static_cast<int>(min(p.a.window, 0x7fffffffu));
    from = window && first + 1 > window ? first + 1 - window : 0;
    if constexpr (kMode == kShared) from = max(from, r.low);
  }
  r.tile_lo = from / tile;
  r.tiles = (r.span.length - 1) / tile + 1 - r.tile_lo;
  const uint64_t query_rows = static_cast<uint64_t>(r.span.count) * p.group;
  r.blocks = r.span.length > 0 && query_rows <= p.beyond ? static_cast<uint32_t>((query_rows + rows - 1) / rows) : 0;  // idle: no work
  r.units = r.blocks * p.a.cache.kv_heads;
  return r;
}

// Keys that the rows of a block see: from the first row's first to the last row's last.
struct Keys {
  int first, last;          // of any row
  int first_all, last_all;  // of all rows
};
template <int kMode>
__device__ __forceinline__ Keys keys_of(const FewParams& p, const Runs& r, uint32_t number, uint32_t block, int rows, const int2* all) {
  Keys k;
  if constexpr (kMode == kSelected) {
    k.first = k.first_all = 0;
    k.last = k.last_all = r.span.length - 1;
    return k;
  }
  if (kMode == kShared && p.prefix) {
    k.first = r.low;
    k.last = r.span.length - 1;
    k.first_all = all[number].x;
    k.last_all = all[number].y;
    return k;
  }
  const int q0 = static_cast<int>(block * rows / p.group);
  const int q1 = min(static_cast<int>(((block + 1) * rows - 1) / p.group), r.span.count - 1);
  const int base = r.span.length - r.span.count, window = static_cast<int>(min(p.a.window, 0x7fffffffu));
  k.last = base + q1;
  k.last_all = base + q0;
  k.first = window && base + q0 + 1 > window ? base + q0 + 1 - window : 0;
  k.first_all = window && base + q1 + 1 > window ? base + q1 + 1 - window : 0;
  if constexpr (kMode == kShared) {
    k.first = max(k.first, r.low);
    k.first_all = max(k.first_all, r.low);
  }
  return k;
}

// A place in the list: tile `tile` (counted from the sequence's first) of a run.
struct Walk {
  uint32_t b, head, block;
  int tile;
  Runs runs;
  Keys keys;
};
// Carries a tile number beyond the run's end into the following runs; false behind the last one.
template <int kMode, typename ItemAt>
__device__ __forceinline__ bool settle(Walk& w, const FewParams& p, uint32_t items, int rows, int tile, const int2* all, ItemAt item_at) {
  while (w.tile >= w.runs.tile_lo + w.runs.tiles || w.runs.units == 0) {
    if (w.runs.units != 0) w.tile -= w.runs.tiles;
    if (w.runs.units == 0 || (++w.block == w.runs.blocks && ++w.head == p.a.cache.kv_heads)) {
      if (++w.b >= items) return false;
      w.tile -= w.runs.units != 0 ? w.runs.tile_lo : 0;
      w.runs = runs_of<kMode>(p, item_at(w.b), w.b, rows, tile);
      w.tile += w.runs.units != 0 ? w.runs.tile_lo : 0;
      w.head = w.block = 0;
    } else if (w.block == w.runs.blocks) {
      w.block = 0;
    }
    if (w.runs.units != 0) w.keys = keys_of<kMode>(p, w.runs, w.b, w.block, rows, all);
  }
  return true;
}

template <typename T, int D, int NT, bool kPair, int kMode>
__global__ void __launch_bounds__(Few<T, D, NT, kPair, kMode>::kThreads, Few<T, D, NT, kPair, kMode>::kCtas) attend_few_kernel(const __grid_constant__ FewParams p) {
  using F = Few<T, D, NT, kPair, kMode>;
  constexpr int kRows = F::kRows, kOf = F::kOf, kWarps = F::kWarps, kStages = F::kStages, kTile = F::kTile, kSubs = F::kSubs;
  constexpr bool kSplit = F::kSplit;
  constexpr int kPer = kPair ? 1 : 2;  // query rows of a thread in one n-tile
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  float* merge = reinterpret_cast<float*>(smem + F::kMerge);
  uint2* q_frag = reinterpret_cast<uint2*>(smem + F::kQFrag);
  float4* row_const = reinterpret_cast<float4*>(smem + F::kRowConst);
  float* warp_stat = reinterpret_cast<float*>(smem + F::kWarpStat);
  unsigned long long* scan = reinterpret_cast<unsigned long long*>(smem + F::kScan);
  unsigned long long* found = scan + kWarps;  // sequence and tiles in front of it, of both cuts; runs of each warp's sequences
  int4* spans = reinterpret_cast<int4*>(smem + F::kSpan);
  int2* all = reinterpret_cast<int2*>(smem + F::kAll);
  int* leads = reinterpret_cast<int*>(smem + F::kLead);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + F::kMisc);
  volatile unsigned int* arrived = reinterpret_cast<volatile unsigned int*>(smem + F::kMisc + 4);
  const uint32_t bars = smem_u32(smem + F::kBars) + warp * kStages * 8;
  if (lane < kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + lane * 8) : "memory");
  if (tid == 0) *abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  pdl_launch_dependents();
  pdl_wait_prior_grid();

  // ---- this CTA's range of the list --------------------------------------------------------------
  const bool prefix = kMode == kShared && p.prefix;
  const bool sharing = kMode != kShared || worth_sharing(p.a, p.sh);
  if (prefix && !sharing) return;
  const uint32_t items = kMode == kSelected ? p.a.batch.tokens : prefix ? p.sh.groups : p.a.batch.sequences, each = (items + F::kThreads - 1) / F::kThreads;
  const bool kept = items <= F::kSpans;
  if constexpr (kMode == kShared) {
    if (prefix) {  // (no more groups than are kept)
      for (uint32_t g_at = warp; g_at < items; g_at += kWarps) {
        int2 every, lead;
        const int4 item = group_of_rows(p.a.batch, p.sh, g_at, static_cast<int>(min(p.a.window, 0x7fffffffu)), every, lead);
        if (lane == 0) {
          spans[g_at] = item;
          all[g_at] = every;
          leads[g_at] = lead.x;
          if (blockIdx.x == 0) p.sh.keys[g_at] = lead.y;
        }
      }
      __syncthreads();
    }
  }
  auto make_item = [&](uint32_t b) {
    if constexpr (kMode == kSelected) return selected_row(p.a, p.sel, b);
    const Span span = span_of(p.a.batch, b);
    return make_int4(span.first, span.count, span.length, kMode == kShared && sharing ? common_keys(p.a.batch, p.sh, b, span) : 0);
  };
  auto item_at = [&](uint32_t b) { return kept ? spans[b] : make_item(b); };
  unsigned long long mine = 0;
  uint32_t mine_runs = 0;
  for (uint32_t b = tid * each; b < min((tid + 1) * each, items); ++b) {
    const int4 item = prefix ? spans[b] : make_item(b);
    if (kept && !prefix) spans[b] = item;
    const Runs r = runs_of<kMode>(p, item, b, kRows, kTile);
    const Span span = r.span;
    mine += static_cast<unsigned long long>(r.units) * static_cast<unsigned>(r.tiles + F::kHead);
    mine_runs += r.units;
    if (!prefix && span.length == 0 && blockIdx.x == b % gridDim.x)  // an idle sequence's rows are zero
      for (int i = 0; i < span.count; ++i)
        for (uint32_t d = 0; d < p.a.heads * D; d += 4) {
          const float zero[4] = {};
          store4(static_cast<T*>(p.a.out) + static_cast<size_t>(span.first + i) * p.a.out_stride + d, zero);
        }
  }
  unsigned long long upto = mine;  // inclusive sum over the threads
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= static_cast<uint32_t>(o)) upto += v;
  }
  const uint32_t warp_runs = __reduce_add_sync(0xffffffffu, mine_runs);
  if (lane == 31) scan[warp] = upto;
  if (lane == 30) found[4 + warp] = warp_runs;
  __syncthreads();
  unsigned long long total = 0, runs = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (static_cast<uint32_t>(i) < warp) upto += scan[i];
    total += scan[i];
    runs += found[4 + i];
  }
  // rows that belong to no sequence are zero
  if (kMode != kSelected && !prefix && p.a.batch.starts) {
    const int tokens = static_cast<int>(p.a.batch.tokens);
    const int head_rows = min(max(p.a.batch.starts[0], 0), tokens), tail = max(min(p.a.batch.starts[items], tokens), head_rows);
    for (int i = blockIdx.x; i < head_rows + tokens - tail; i += gridDim.x) {
      T* out = static_cast<T*>(p.a.out) + static_cast<size_t>(i < head_rows ? i : tail + i - head_rows) * p.a.out_stride;
      const float zero[4] = {};
      for (uint32_t d = tid * 4; d < p.a.heads * D; d += F::kThreads * 4) store4(out + d, zero);
    }
  }
  if (total == 0) return;
  // equal ranges, of 256 tokens at least, or of a run's where those are shorter: then as many CTAs as runs share the work
  const unsigned long long per = max((total + gridDim.x - 1) / gridDim.x, min(256ull / kTile, (total + runs - 1) / runs));
  const unsigned long long cut[2] = {blockIdx.x * per, min(blockIdx.x * per + per, total)};
  if (cut[0] >= total) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (upto - mine <= cut[i] && cut[i] < upto) {
      found[2 * i] = tid * each;
      found[2 * i + 1] = upto - mine;
    }
  __syncthreads();
  // Walk to tile number x; a run of up to kShort tiles is not cut: a cut inside it moves to its beginning, so it is the later range's
  auto locate = [&](unsigned long long& x, int i) {
    Walk w;
    w.b = static_cast<uint32_t>(found[2 * i]);
    w.runs = runs_of<kMode>(p, item_at(w.b), w.b, kRows, kTile);
    unsigned long long skip = x - found[2 * i + 1];
    while (skip >= static_cast<unsigned long long>(w.runs.units) * static_cast<unsigned>(w.runs.tiles + F::kHead)) {  // sequences of one thread's share
      skip -= static_cast<unsigned long long>(w.runs.units) * static_cast<unsigned>(w.runs.tiles + F::kHead);
      ++w.b;
      w.runs = runs_of<kMode>(p, item_at(w.b), w.b, kRows, kTile);
    }
    const uint32_t unit = static_cast<uint32_t>(skip / static_cast<unsigned>(w.runs.tiles + F::kHead));
    int in = static_cast<int>(skip % static_cast<unsigned>(w.runs.tiles + F::kHead));
    if (w.runs.tiles <= F::kShort || in <= F::kHead) {
      x -= static_cast<unsigned>(in);
      in = F::kHead;
    }
    in -= F::kHead;
    w.head = unit / w.runs.blocks;
    w.block = unit % w.runs.blocks;
    w.tile = w.runs.tile_lo + in;
    w.keys = keys_of<kMode>(p, w.runs, w.b, w.block, kRows, all);
    return w;
  };
  unsigned long long begin = cut[0], end = cut[1];
  Walk at = locate(begin, 0);
  if (end < total) locate(end, 1);
  if (begin >= end) return;

  // ---- copies: the warp's tiles, a ring's length ahead --------------------------------------------
  const uint32_t ring = smem_u32(smem + F::kRing) + warp * kStages * F::kTileBytes;
  uint8_t* const ring_ptr = smem + F::kRing + warp * kStages * F::kTileBytes;
  // lane 4 i + j copies array j (K codes, V codes, K scales, V scales) of the tile's i-th piece, a run of tokens in one page
  const uint32_t P = p.a.cache.page_tokens, run = min(P, static_cast<uint32_t>(kTile));
  const uint32_t piece = lane / 4, array = lane % 4, token_bytes = array < 2 ? D / 2 : 4;
  const bool copies = piece * run < kTile;
  const uint32_t from_block = (array >= 2 ? P * D : 0u) + (array & 1 ? P * token_bytes : 0u);
  const uint32_t to_stage = (array >= 2 ? kTile * D : 0) + ((array & 1 ? kTile : 0) + piece * run) * token_bytes;
  const uint32_t block_bytes = static_cast<uint32_t>(cache_block_bytes(P, D)), page_bytes = block_bytes * p.a.cache.kv_heads;  // 1024 heads: 70 MB at most
  Walk ahead = at;
  ahead.tile += static_cast<int>(warp);
  unsigned long long range = end - begin;  // tiles of the range: without what runs cost
  if constexpr (F::kHead > 0) {
    Walk w = at;
    range = 0;
    for (unsigned long long pos = begin; pos < end;) {
      const unsigned head = w.tile == w.runs.tile_lo ? F::kHead : 0;
      const unsigned in_run = min(static_cast<unsigned>(w.runs.tile_lo + w.runs.tiles - w.tile), static_cast<unsigned>(end - pos - head));
      range += in_run;
      pos += head + in_run;
      w.tile += static_cast<int>(in_run);
      if (pos < end) settle<kMode>(w, p, items, kRows, kTile, all, item_at);
    }
  }
  int to_issue = range > warp ? static_cast<int>((range - warp + kWarps - 1) / kWarps) : 0;  // tiles of this warp not passed yet
  uint32_t issued = 0, used = 0;
  // the next tile to copy: its page number is loaded a tile's time before it is needed
  bool wanted = false;
  uint32_t page = 0, in_page = 0;
  bool waiting = false;
  auto look_ahead = [&]() {
    waiting = false;
    for (; to_issue > 0 && !waiting; ahead.tile += kWarps, --to_issue) {
      settle<kMode>(ahead, p, items, kRows, kTile, all, item_at);
      const int first = ahead.tile * kTile;
      if (first > ahead.keys.last || first + kTile <= ahead.keys.first) continue;
      const uint32_t key = static_cast<uint32_t>(first) + piece * run;
      in_page = ahead.head * block_bytes + from_block + (key & (P - 1)) * token_bytes;
      const uint32_t index = key >> p.page_shift;
      wanted = copies && static_cast<int>(key) <= ahead.keys.last;
      page = 0xFFFFFFFFu;
      if constexpr (kMode == kSelected) {
        if (wanted) page = selected_page(p.a, p.sel, ahead.b, ahead.head, ahead.runs.sequence, index);
      } else {
        const uint32_t of = prefix ? static_cast<uint32_t>(leads[ahead.b]) : ahead.b;
        if (wanted && index < p.a.batch.width) page = static_cast<uint32_t>(__ldg(p.a.batch.pages + static_cast<size_t>(of) * p.a.batch.width + index));
      }
      waiting = true;
    }
  };
  auto issue_next = [&]() {
    if (waiting) {
      const uint32_t stage = issued % kStages, bar = bars + stage * 8;
      const bool have = page < p.a.cache.pages;  // a negative number is not
      const uint32_t all = __ballot_sync(0xffffffffu, have), lost = __ballot_sync(0xffffffffu, wanted && !have);
      if (lost) {  // no such page: what it would hold is NaN
        uint32_t* params = reinterpret_cast<uint32_t*>(ring_ptr + stage * F::kTileBytes + kTile * D);
        for (uint32_t i = lane; i < kTile; i += 32)
          if (lost >> (i / run * 4) & 1) params[i] = params[kTile + i] = 0x7E007E00u;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (lane == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(__popc(all) / 4 * run * (D + 8)) : "memory");
      __syncwarp();
      if (have) {
        const uint8_t* from = p.a.cache.pool + static_cast<uint64_t>(page) * page_bytes + in_page;
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(ring + stage * F::kTileBytes + to_stage), "l"(from), "r"(run * token_bytes), "r"(bar) : "memory");
      }
      ++issued;
      look_ahead();
    }
  };
  __syncwarp();
  look_ahead();
  for (int i = 0; i < kStages; ++i) issue_next();

  const uint32_t odd = t & 1;  // the order of a thread's tokens in a pair of rows: neighbouring rows fall into different banks
  const uint32_t token_g = g ^ ((g >> 1) & 1);
  const uint32_t token_t0 = 2 * t + odd, token_t1 = 2 * t + 1 - odd;
  constexpr uint32_t kCentre0 = 0x800F800Fu;  // -15 2^-24, twice: 2 u - 15
  constexpr uint32_t kCentre1 = 0x80788078u;  // -7.5 2^-20, twice

  // ---- run by run --------------------------------------------------------------------------------
  unsigned long long passed = 0;  // tiles of the range
  for (unsigned long long pos = begin; pos < end;) {
    const int run_end = at.runs.tile_lo + at.runs.tiles;
    const unsigned head_of_run = at.tile == at.runs.tile_lo ? F::kHead : 0;  // at a run's beginning
    const int stop = static_cast<int>(min(static_cast<unsigned long long>(run_end), at.tile + (end - pos - head_of_run)));
    const int q_rows = at.runs.span.count * static_cast<int>(p.group);
    const int base = kMode == kSelected ? at.runs.position : at.runs.span.length - at.runs.span.count;
    const Keys keys = at.keys;
    auto position_of = [&](int query) {
      if (prefix) return place_of_row(p.a.batch, static_cast<uint32_t>(at.runs.span.first + query)).x;
      return base + query;
    };

    // queries: rotated, scaled to binary16's range by a power of two, in the order of the B fragments
    // (all of a warp's rows asked for before the first is worked on)
    float loaded[kRows / kWarps][8];
#pragma unroll
    for (int i = 0; i < kRows / kWarps; ++i) {
      const int row = static_cast<int>(at.block) * kRows + static_cast<int>(warp) + i * kWarps, query = row / static_cast<int>(p.group);
      const int head = static_cast<int>(at.head * p.group) + row - query * static_cast<int>(p.group);
#pragma unroll
      for (int e = 0; e < 8; ++e) loaded[i][e] = 0.0f;
      if (row < q_rows && lane < D / 8)
        load8_rotated(static_cast<const T*>(p.a.q) + static_cast<size_t>(at.runs.span.first + query) * p.a.q_stride + static_cast<size_t>(head) * D,
                      lane * 8, p.a.rope, position_of(query), loaded[i]);
    }
#pragma unroll
    for (int i_row = 0; i_row < kRows / kWarps; ++i_row) {
      const int r = static_cast<int>(warp) + i_row * kWarps;
      const int query = (static_cast<int>(at.block) * kRows + r) / static_cast<int>(p.group);
      const bool there = static_cast<int>(at.block) * kRows + r < q_rows;
      const float (&v)[8] = loaded[i_row];
      float big = 0.0f, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(v[i]));
#pragma unroll
      for (int o = 16; o > 0; o /= 2) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      // 2^(13 - exponent of the largest): all below 2^14
      const int e = static_cast<int>(__float_as_uint(big) >> 23);
      const int up = big > 0.0f && e < 255 ? min(max(140 - e, -100), 120) : 0;
      const float lift = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
      __half hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = v[i] * lift, down = (i & 1) ? 0.0625f : 1.0f;
        // f32: fixed-point parts, multiples of 8 and of 2^-8.  Their products with codes are whole multiples too, 22 bits in
        // all of a row, so that the tensor core (which cuts each product at a place set by the largest) adds them exactly
        const float top = kSplit ? rintf(x * 0.125f) * 8.0f : x;
        hi[i] = __float2half_rn(top * down);
        lo[i] = kSplit ? __float2half_rn(rintf((x - top) * 256.0f) * (0.00390625f * down)) : __ushort_as_half(0);
        // The offsets meet the queries as they were rounded, like the codes: a rounding then weighs as much as the key, not as the code
        // times its scale, which in a row with one large value is large everywhere.
        sum = fmaf(__half2float(hi[i]) + __half2float(lo[i]), (i & 1) ? 16.0f : 1.0f, sum);
      }
      sum = warp_sum(sum) * __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
      if (lane < D / 8) {
        // word W = lane of a key lies with thread tt as its word ww
        const uint32_t tt = D == 64 ? lane / 2 : lane % 16 / 4, ww = D == 64 ? lane % 2 : lane / 16 * 4 + lane % 4;
#pragma unroll
        for (int part = 0; part < (kPair ? 2 : 1); ++part) {
          const uint32_t col = r * (kPair ? 2 : 1) + part, n = col / 8, c = col % 8;
          const __half* h = part ? lo : hi;
#pragma unroll
          for (int half = 0; half < 2; ++half)
            q_frag[(n * F::kSteps + 2 * ww + half) * 32 + c * 4 + tt] =
                make_uint2(pack_half2(h[2 * half], h[2 * half + 4]), pack_half2(h[2 * half + 1], h[2 * half + 5]));
        }
      }
      if (lane == 0) {
        const float factor = p.a.scale * 1.4426950408889634f;
        int last = there ? base + query : -1;
        const int window = static_cast<int>(min(p.a.window, 0x7fffffffu));
        int from = 0;
        if (kMode == kSelected) {
          last = there ? at.runs.span.length - 1 : -1;
        } else if (prefix) {
          const int2 place = there ? place_of_row(p.a.batch, static_cast<uint32_t>(at.runs.span.first + query)) : make_int2(0, 0);
          from = window && place.x + 1 > window ? place.x + 1 - window : 0;
          last = min(place.y, at.runs.span.length) - 1;
        } else {
          from = window && last + 1 > window ? last + 1 - window : 0;
          if constexpr (kMode == kShared) from = max(from, at.runs.low);
        }
        // the accumulators hold 2^(up - 24) q . u
        row_const[r] = make_float4(factor * exp2f(static_cast<float>(24 - up)), factor * sum, __int_as_float(last), __int_as_float(from));
      }
    }
    __syncthreads();
    uint2 bq[F::kQInRegisters ? NT : 1][F::kQInRegisters ? F::kSteps : 1];
    if constexpr (F::kQInRegisters) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int s = 0; s < F::kSteps; ++s) bq[n][s] = q_frag[(n * F::kSteps + s) * 32 + lane];
    }
    // a thread's query rows in n-tile n: n * kOf + t * kPer + i
    float factor[NT][kPer], offset[NT][kPer];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float4 c = row_const[n * kOf + t * kPer + i];
        factor[n][i] = c.x;
        offset[n][i] = c.y;
      }
    // what the one row of a thread has in common: its place is there when the row is finished
    uint4 place_ahead = {};
    if constexpr (kMode == kShared && kRows * D / 4 <= F::kThreads) {
      const int row = static_cast<int>(at.block) * kRows + static_cast<int>(tid) / (D / 4);
      if (!prefix && at.runs.low > 0 && static_cast<int>(tid) < kRows * D / 4 && row < q_rows) {
        const int query = row / static_cast<int>(p.group);
        place_ahead = __ldcg(p.sh.places + static_cast<size_t>(at.runs.span.first + query) * p.a.heads + at.head * p.group + static_cast<uint32_t>(row - query * static_cast<int>(p.group)));
      }
    }
    float M[NT][kPer], l[NT][kPer] = {}, centre[NT][kPer] = {};
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < kPer; ++i) M[n][i] = -INFINITY;
    // f32 queries: sums of a thread's two dims an MMA for its one row; 16-bit ones: the accumulators of two columns
    constexpr int kHold = kSplit ? 2 : 4, kSide = kSplit ? 1 : 2;  // row i's dims are [i] and [kSide + i]
    float O[NT][F::kVWords * 4][kHold] = {};

    const int ahead_of = static_cast<int>((F::kHead > 0 ? passed : pos - begin) % kWarps);
    for (int tile_at = at.tile + (static_cast<int>(warp) + kWarps - ahead_of) % kWarps; tile_at < stop; tile_at += kWarps) {
      const int first = tile_at * kTile;
      if (first > keys.last || first + kTile <= keys.first) continue;
      const uint32_t stage = used % kStages, parity = used / kStages & 1;
      {
        const uint32_t bar = bars + stage * 8;
        uint32_t done = 0;
        for (uint32_t spin = 0; spin < kFewWaitLimit && !done; ++spin) {
          asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                       : "=r"(done) : "r"(bar), "r"(parity) : "memory");
          if (!done && (spin & 1023u) == 1023u && *abort_flag) break;
        }
        if (!__all_sync(0xffffffffu, done)) {
          *abort_flag = 1;
          *reinterpret_cast<volatile int*>(p.status) = kFewTimeout;
          waiting = false;  // nothing more is copied: the barrier's phase is not over, and may not be arrived on again
          to_issue = 0;
        }
      }
      const uint8_t* tile = ring_ptr + stage * F::kTileBytes;
      const bool whole = first >= keys.first_all && first + kTile - 1 <= keys.last_all;
      float s[kSubs][NT][kPer][2];  // [subtile][..][row][token half]
      uint32_t vp[kSubs][2];        // the values' (scale, offset) of the thread's tokens
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        float acc[NT][4] = {};
        const uint8_t* row0 = tile + (sub * 16 + token_g) * (D / 2);
        const uint8_t* row1 = row0 + 8 * (D / 2);
        uint32_t x0[F::kWords], x1[F::kWords];
        if constexpr (D == 64) {
          *reinterpret_cast<uint2*>(x0) = *reinterpret_cast<const uint2*>(row0 + t * 8);
          *reinterpret_cast<uint2*>(x1) = *reinterpret_cast<const uint2*>(row1 + t * 8);
        } else {
#pragma unroll
          for (int i = 0; i < F::kWords / 4; ++i) {
            *reinterpret_cast<uint4*>(x0 + 4 * i) = *reinterpret_cast<const uint4*>(row0 + i * 64 + t * 16);
            *reinterpret_cast<uint4*>(x1 + 4 * i) = *reinterpret_cast<const uint4*>(row1 + i * 64 + t * 16);
          }
        }
#pragma unroll
        for (int w = 0; w < F::kWords; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t a = half ? x0[w] >> 8 : x0[w], b = half ? x1[w] >> 8 : x1[w];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 bb = F::kQInRegisters ? bq[F::kQInRegisters ? n : 0][F::kQInRegisters ? 2 * w + half : 0]
                                                : q_frag[(n * F::kSteps + 2 * w + half) * 32 + lane];
              mma16816(acc[n], a & 0x000F000Fu, b & 0x000F000Fu, a & 0x00F000F0u, b & 0x00F000F0u, bb.x, bb.y);
            }
          }
        const uint32_t* params = reinterpret_cast<const uint32_t*>(tile + kTile * D) + sub * 16 + token_g;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t kp = params[half * 8];
          vp[sub][half] = params[kTile + half * 8];
          const float2 so = __half22float2(*reinterpret_cast<const __half2*>(&kp));
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              const float dot = kSplit ? acc[n][2 * half] + acc[n][2 * half + 1] : acc[n][2 * half + i];
              s[sub][n][i][half] = fmaf(dot, so.x * factor[n][i], so.y * offset[n][i]);
            }
        }
      }
      // the largest binade of the values' scales that a row sees (at least log2 of a scale)
      auto binade_of = [](uint32_t bits) { return static_cast<float>(max(static_cast<int>(bits >> 10), 1) - 14); };
      float binade[NT][kPer];
      if (whole) {
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < 2 * kSubs; ++j) big = max(big, vp[j / 2][j % 2] & 0x7C00u);
        const float common = binade_of(big);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < kPer; ++i) binade[n][i] = common;
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const float4 c = row_const[n * kOf + t * kPer + i];
            uint32_t big = 0;
#pragma unroll
            for (int j = 0; j < 2 * kSubs; ++j) {
              const int key = first + j * 8 + static_cast<int>(token_g);
              if (key > __float_as_int(c.z) || key < __float_as_int(c.w)) s[j / 2][n][i][j % 2] = -INFINITY;
              else big = max(big, vp[j / 2][j % 2] & 0x7C00u);
            }
            binade[n][i] = binade_of(big);
          }
      }
      // M: the largest score with its binade
      bool more = false;
      float top[NT][kPer];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          top[n][i] = fmaxf(s[0][n][i][0], s[0][n][i][1]);
#pragma unroll
          for (int sub = 1; sub < kSubs; ++sub) top[n][i] = fmaxf(top[n][i], fmaxf(s[sub][n][i][0], s[sub][n][i][1]));
          top[n][i] += binade[n][i];
          if constexpr (kSplit) {  // the tile's largest
#pragma unroll
            for (int o = 4; o < 32; o *= 2) top[n][i] = fmaxf(top[n][i], __shfl_xor_sync(0xffffffffu, top[n][i], o));
          }
          more |= top[n][i] > M[n][i] + 8.0f;
        }
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            float m = top[n][i];
            if constexpr (!kSplit) {
#pragma unroll
              for (int o = 4; o < 32; o *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            }
            m = fmaxf(m, M[n][i]);
            const float keep = m == -INFINITY ? 1.0f : exp2_fast(M[n][i] - m);
            M[n][i] = m;
            l[n][i] *= keep;
            centre[n][i] *= keep;
#pragma unroll
            for (int d = 0; d < F::kVWords * 4; ++d) {
              O[n][d][i] *= keep;
              O[n][d][kSide + i] *= keep;
            }
          }
      }
      float shift[NT][kPer], lift[NT], drop[NT];  // f32: P is lifted to just below 2^14 in each tile, and back when its sums are added
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) shift[n][i] = M[n][i] == -INFINITY ? 0.0f : -M[n][i];
        // as numbers: a tile in which the row sees nothing has a largest score of -inf
        const int up = kSplit ? static_cast<int>(fminf(fmaxf(14.0f - ceilf(top[n][0] + shift[n][0]), 0.0f), 120.0f)) : 6;
        lift[n] = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
        drop[n] = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
      }
      uint32_t bp[kSubs][NT][2];
      auto weigh = [&](auto all_seen) {
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float2 so = __half22float2(*reinterpret_cast<const __half2*>(&vp[sub][half]));
            const float mid = fmaf(7.5f, so.x, so.y);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float pv[kPer];
#pragma unroll
              for (int i = 0; i < kPer; ++i) {
                const float sc = s[sub][n][i][half], w = exp2_fast(sc + shift[n][i]);
                l[n][i] += w;
                if (decltype(all_seen)::value || sc != -INFINITY) {
                  centre[n][i] = fmaf(w, mid, centre[n][i]);
                  pv[i] = w * so.x;
                } else {
                  pv[i] = 0.0f;  // what is not seen may hold anything
                }
                pv[i] *= lift[n];
              }
              uint32_t both;
              if constexpr (kSplit) {  // the high part: whole numbers (their sums are exact) of eleven bits, so that small weights keep 22 too
                const float hi = __uint_as_float(__float_as_uint(rintf(pv[0])) & 0xFFFFE000u);
                both = pack_half2(__float2half_rn(hi), __float2half_rn(pv[0] - hi));
              } else {
                const __half2 h = __floats2half2_rn(pv[0], kPair ? 0.0f : pv[kPer - 1]);
                both = *reinterpret_cast<const uint32_t*>(&h);
              }
              bp[sub][n][half] = transposed(both);
            }
          }
      };
      if (whole) weigh(std::true_type());
      else weigh(std::false_type());
      float tile_acc[kSplit ? NT : 1][kSplit ? F::kVWords * 4 : 1][4] = {};
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        const uint8_t* v0 = tile + kTile * (D / 2) + sub * 16 * (D / 2) + g * (D / 16);
        uint32_t xa[F::kVWords], xb[F::kVWords], xc[F::kVWords], xd[F::kVWords];
        auto load_v = [&](uint32_t (&x)[F::kVWords], uint32_t token) {
          const uint8_t* from_v = v0 + token * (D / 2);
          if constexpr (D == 64) x[0] = *reinterpret_cast<const uint32_t*>(from_v);
          else if constexpr (D == 128) *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(from_v);
          else *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(from_v);
        };
        load_v(xa, token_t0);
        load_v(xb, token_t1);
        load_v(xc, token_t0 + 8);
        load_v(xd, token_t1 + 8);
#pragma unroll
        for (int w = 0; w < F::kVWords; ++w) {
          const uint32_t lo01 = __byte_perm(xa[w], xb[w], 0x5410), hi01 = __byte_perm(xa[w], xb[w], 0x7632);
          const uint32_t lo23 = __byte_perm(xc[w], xd[w], 0x5410), hi23 = __byte_perm(xc[w], xd[w], 0x7632);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // dims i (rows g) and i + 4 (rows g + 8) of the word
            uint32_t a[4] = {lo01, hi01, lo23, hi23};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t x = i >= 2 ? a[j] >> 8 : a[j];
              a[j] = (i & 1) ? hadd2_u(x & 0x00F000F0u, kCentre1) : hfma2_u(x & 0x000F000Fu, 0x40004000u, kCentre0);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (kSplit) mma16816(tile_acc[n][w * 4 + i], a[0], a[1], a[2], a[3], bp[sub][n][0], bp[sub][n][1]);
              else mma16816(O[n][w * 4 + i], a[0], a[1], a[2], a[3], bp[sub][n][0], bp[sub][n][1]);
            }
          }
        }
      }
      if constexpr (kSplit) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int d = 0; d < F::kVWords * 4; ++d) {
            O[n][d][0] = fmaf(tile_acc[n][d][0] + tile_acc[n][d][1], drop[n], O[n][d][0]);
            O[n][d][1] = fmaf(tile_acc[n][d][2] + tile_acc[n][d][3], drop[n], O[n][d][1]);
          }
      }
      ++used;
      __syncwarp();
      issue_next();
    }

    // ---- the warps' sums, joined ---------------------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int o = 4; o < 32; o *= 2) {
          l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], o);
          centre[n][i] += __shfl_xor_sync(0xffffffffu, centre[n][i], o);
        }
    if (g == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          float* st = warp_stat + (warp * kRows + n * kOf + t * kPer + i) * 3;
          st[0] = M[n][i];
          st[1] = l[n][i];
          st[2] = centre[n][i];
        }
    }
    // the codes' powers of two, even dims (2 u - 15) 2^-24, odd ones (u - 7.5) 2^-20, and the 16-bit weights' 2^6
    constexpr float kEven = kSplit ? 8388608.0f : 131072.0f, kOdd = kSplit ? 1048576.0f : 16384.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int w = 0; w < F::kVWords; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // dims 0..3, then 4..7 of the thread's word
            const int e = half * kSide + i;
            *reinterpret_cast<float4*>(merge + (warp * kRows + n * kOf + t * kPer + i) * D + g * (D / 8) + w * 8 + half * 4) =
                make_float4(O[n][w * 4][e] * kEven, O[n][w * 4 + 1][e] * kOdd, O[n][w * 4 + 2][e] * kEven, O[n][w * 4 + 3][e] * kOdd);
          }
    __syncthreads();
    constexpr int kQuads = kRows * D / 4;  // outputs of the block, by four
    constexpr int kLoops = (kQuads + F::kThreads - 1) / F::kThreads;
    const bool complete = at.tile == at.runs.tile_lo && stop == run_end;
    const unsigned long long run_begin = pos + head_of_run - static_cast<unsigned>(at.tile - at.runs.tile_lo);  // its first tile's place
    const uint32_t c0 = static_cast<uint32_t>(run_begin / per), c1 = static_cast<uint32_t>((run_begin + static_cast<unsigned>(at.runs.tiles) - 1) / per);
    auto slot_of = [&](uint32_t c) { return c == c0 ? 2 * c0 + 1 : 2 * c; };  // a CTA's last run goes on, or its first came from before
    float* part = p.parts + static_cast<size_t>(slot_of(blockIdx.x)) * F::kPartFloats;
    auto store_row = [&](int quad, const float (&v)[4], float total_l, float m) {
      const int row = static_cast<int>(at.block) * kRows + quad / (D / 4), query = row / static_cast<int>(p.group);
      if (row >= q_rows) return;
      const int head = static_cast<int>(at.head * p.group) + row - query * static_cast<int>(p.group);
      if constexpr (kMode == kShared) {
        const size_t of = static_cast<size_t>(at.runs.span.first + query) * p.a.heads + static_cast<size_t>(head);
        if (prefix) {
          const uint4 place = whole_place(p.sh, p.a, of);
          __stcg(reinterpret_cast<float4*>(p.sh.scratch) + place.x + quad % (D / 4), make_float4(v[0], v[1], v[2], v[3]));
          if (quad % (D / 4) == 0) {
            __stcg(reinterpret_cast<float2*>(p.sh.scratch) + place.y, make_float2(m, total_l));
            __stcg(p.sh.places + of, place);
          }
          return;
        }
        if (at.runs.low > 0) {  // with what the row sees of the common keys
          float all[4] = {v[0], v[1], v[2], v[3]};
          join_common(p.sh, kLoops == 1 ? place_ahead : __ldcg(p.sh.places + of), quad % (D / 4), m, total_l, all);
          const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
          const float o[4] = {all[0] * inv, all[1] * inv, all[2] * inv, all[3] * inv};
          store4(static_cast<T*>(p.a.out) + static_cast<size_t>(at.runs.span.first + query) * p.a.out_stride + static_cast<size_t>(head) * D + quad % (D / 4) * 4, o);
          return;
        }
      }
      const float inv = total_l == 0.0f ? 0.0f : 1.0f / total_l;
      const float o[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
      store4(static_cast<T*>(p.a.out) + static_cast<size_t>(at.runs.span.first + query) * p.a.out_stride + static_cast<size_t>(head) * D + quad % (D / 4) * 4, o);
    };
#pragma unroll
    for (int k = 0; k < kLoops; ++k) {
      const int quad = static_cast<int>(tid) + k * F::kThreads;
      if (quad >= kQuads) break;
      const int row = quad / (D / 4);
      float m = -INFINITY, total_l = 0.0f, mid = 0.0f, sum[4] = {};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_stat[(w * kRows + row) * 3]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* st = warp_stat + (w * kRows + row) * 3;
        const float keep = st[0] == -INFINITY ? 0.0f : exp2_fast(st[0] - m);
        const float4 v = reinterpret_cast<const float4*>(merge + w * kRows * D)[quad];
        total_l = fmaf(keep, st[1], total_l);
        mid = fmaf(keep, st[2], mid);
        sum[0] = fmaf(keep, v.x, sum[0]);
        sum[1] = fmaf(keep, v.y, sum[1]);
        sum[2] = fmaf(keep, v.z, sum[2]);
        sum[3] = fmaf(keep, v.w, sum[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += mid;
      if (complete) {
        store_row(quad, sum, total_l, m);
      } else {
        __stcg(reinterpret_cast<float4*>(part) + quad, make_float4(sum[0], sum[1], sum[2], sum[3]));
        if (quad % (D / 4) == 0) __stcg(reinterpret_cast<float2*>(part + kRows * D) + row, make_float2(m, total_l));
      }
    }
    if (!complete) {
      // the last CTA of sixteen neighbours joins their parts, the last of these groups the groups'
      constexpr uint32_t kGroup = 16;
      const uint32_t group0 = max(c0, blockIdx.x / kGroup * kGroup), group1 = min(c1, blockIdx.x / kGroup * kGroup + kGroup - 1);
      const uint32_t groups = c1 / kGroup - c0 / kGroup + 1;
      auto last_of = [&](unsigned int* counter, uint32_t count) {
        __syncthreads();
        if (tid == 0) {
          unsigned int before;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
          if (before == count - 1) *counter = 0;
          *arrived = before;
        }
        __syncthreads();
        return *arrived == count - 1;
      };
      // joins the parts in slots slot(0 .. count), in order; into `to`, or (null) the output
      auto join = [&](auto slot, uint32_t count, float* to) {
#pragma unroll
        for (int k = 0; k < kLoops; ++k) {
          const int quad = static_cast<int>(tid) + k * F::kThreads;
          if (quad >= kQuads) break;
          const int row = quad / (D / 4);
          float m = -INFINITY, total_l = 0.0f, v[4] = {};
          constexpr uint32_t kBatch = 8;
          for (uint32_t j0 = 0; j0 < count; j0 += kBatch) {
            float2 ml[kBatch];
            float4 x[kBatch];
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
              const float* from_part = p.parts + static_cast<size_t>(slot(min(j0 + j, count - 1))) * F::kPartFloats;
              ml[j] = __ldcg(reinterpret_cast<const float2*>(from_part + kRows * D) + row);
              x[j] = __ldcg(reinterpret_cast<const float4*>(from_part) + quad);
            }
            float now = m;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
              if (j0 + j >= count) ml[j] = make_float2(-INFINITY, 0.0f);
              now = fmaxf(now, ml[j].x);
            }
            const float before = m == -INFINITY ? 0.0f : exp2_fast(m - now);
            m = now;
            total_l *= before;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= before;
#pragma unroll
            for (uint32_t j = 0; j < kBatch; ++j) {
              const float keep = ml[j].x == -INFINITY ? 0.0f : exp2_fast(ml[j].x - m);
              total_l = fmaf(keep, ml[j].y, total_l);
              v[0] = fmaf(keep, x[j].x, v[0]);
              v[1] = fmaf(keep, x[j].y, v[1]);
              v[2] = fmaf(keep, x[j].z, v[2]);
              v[3] = fmaf(keep, x[j].w, v[3]);
            }
          }
          if (!to) {
            store_row(quad, v, total_l, m);
          } else {
            __stcg(reinterpret_cast<float4*>(to) + quad, make_float4(v[0], v[1], v[2], v[3]));
            if (quad % (D / 4) == 0) __stcg(reinterpret_cast<float2*>(to + kRows * D) + row, make_float2(m, total_l));
          }
        }
      };
      if (last_of(p.counters + slot_of(group0), group1 - group0 + 1)) {
        if (groups == 1) {
          join([&](uint32_t j) { return slot_of(group0 + j); }, group1 - group0 + 1, nullptr);
        } else {
          join([&](uint32_t j) { return slot_of(group0 + j); }, group1 - group0 + 1, p.parts + static_cast<size_t>(2 * gridDim.x + slot_of(group0)) * F::kPartFloats);
          if (last_of(p.counters + 2 * gridDim.x + c0, groups))
            join([&](uint32_t j) { return 2 * gridDim.x + slot_of(j == 0 ? c0 : (c0 / kGroup + j) * kGroup); }, groups, nullptr);
        }
      }
    }
    __syncthreads();  // q_frag, row_const, merge and warp_stat belong to the next run
    pos += head_of_run + static_cast<unsigned>(stop - at.tile);
    passed += static_cast<unsigned>(stop - at.tile);
    at.tile = stop;
    if (pos < end) settle<kMode>(at, p, items, kRows, kTile, all, item_at);
  }
}

// The call's common part; kMode's own numbers are the caller's.
inline FewParams few_params(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond) {
  FewParams p = {};
  p.a = a;
  p.group = a.heads / a.cache.kv_heads;
  while ((1u << p.page_shift) < a.cache.page_tokens) ++p.page_shift;
  p.parts = static_cast<float*>(env.workspace);
  p.counters = env.counters;
  p.status = env.status;
  p.beyond = beyond;
  return p;
}

template <typename T, int D, int NT, bool kPair, int kMode>
cudaError_t few_as(const LaunchEnv& env, const FewParams& p) {
  using F = Few<T, D, NT, kPair, kMode>;
  static_assert(F::kCtas >= 1, "shared memory");
  static_assert(F::kMerge % 16 == 0 && F::kQFrag % 16 == 0 && F::kRowConst % 16 == 0 && F::kScan % 16 == 0 && F::kSpan % 16 == 0 && F::kBars % 8 == 0 &&
                    F::kPartFloats % 4 == 0, "alignment of the shared arrays and of the parts");
  static OncePerDevice once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(attend_few_kernel<T, D, NT, kPair, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem); });
  if (e != cudaSuccess) return e;
  // a CTA's two parts and those of its groups must fit the scratch; one CTA alone shares no run
  const uint64_t fit = env.workspace ? env.workspace_bytes / (4ull * F::kPartFloats * sizeof(float)) : 0;
  const unsigned grid = static_cast<unsigned>(
      std::max<uint64_t>(1, std::min<uint64_t>({static_cast<uint64_t>(env.sm_count) * F::kCtas, fit, env.counter_count / 3})));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(F::kThreads);
  cfg.dynamicSmemBytes = F::kSmem;
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attend_few_kernel<T, D, NT, kPair, kMode>, p);
}

// By the rows that a sequence's new tokens make with one kv head; beyond the widest block, blocks of it.
template <typename T, int D, int kMode>
cudaError_t few_of(const LaunchEnv& env, const FewParams& p, uint64_t rows) {
  if (rows <= 4) return few_as<T, D, 1, true, kMode>(env, p);
  if constexpr (sizeof(T) == 4) {
    if (rows <= 8 || D > 128) return few_as<T, D, 2, true, kMode>(env, p);
    if constexpr (D <= 128) return few_as<T, D, 4, true, kMode>(env, p);
  } else {
    if (rows <= 8) return few_as<T, D, 1, false, kMode>(env, p);
    if (rows <= 16 || D > 128) return few_as<T, D, 2, false, kMode>(env, p);
    if constexpr (D <= 128) return few_as<T, D, 4, false, kMode>(env, p);
  }
  return cudaErrorInvalidValue;
}

template <typename T, int kMode>
cudaError_t few_in(const LaunchEnv& env, const FewParams& p, uint64_t rows) {
  switch (p.a.cache.head_dim) {
    case 64: return few_of<T, 64, kMode>(env, p, rows);
    case 128: return few_of<T, 128, kMode>(env, p, rows);
    case 256: return few_of<T, 256, kMode>(env, p, rows);
    default: return cudaErrorInvalidValue;
  }
}

template <int kMode>
cudaError_t launch_few(const LaunchEnv& env, const FewParams& p, uint64_t rows) {
  if (p.a.dtype == KQ_F32) return few_in<float, kMode>(env, p, rows);
  if (p.a.dtype == KQ_F16) return few_in<__half, kMode>(env, p, rows);
  return few_in<__nv_bfloat16, kMode>(env, p, rows);
}

// Over common keys (prefix) or behind them.
template <typename T>
cudaError_t few_shared(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, bool prefix, const SharedArgs& sh, uint64_t rows) {
  FewParams p = few_params(env, a, beyond);
  p.prefix = prefix;
  p.sh = sh;
  return few_in<T, kShared>(env, p, rows);
}

// Query rows (of a sequence and kv head) up to which this kernel is faster than 128-row MMAs.  16 sequences of 4096 tokens, 8 kv heads,
// this one / the other: bfloat16 16 rows 43 / 95 us, 32 rows 88 / 96, 48 rows 141 / 97; f32 32 rows 104 / 148, 48 rows 147 / 148.
constexpr uint32_t kFewRows = 32;

}  // namespace
}  // namespace kq
