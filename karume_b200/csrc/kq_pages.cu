// Pages of a paged cache that sequences share: which page belongs to whom, and copies of pages.
//
//   grow     every sequence gets the pages that its next tokens need
//   fork     every sequence becomes the beginning of a sequence, all at once; pages are shared, one that is not full has one owner
//   compact  the pages in use move to the lowest numbers
//   copy     the content of pages, in any number of pools
//
// The first three work on small arrays of whole numbers, so what bounds them is latency: loads that depend on one another, atomic
// operations and the barriers between the steps, each of which sees all of the step in front.  One cluster of CTAs does all of a call:
// its barrier costs a fraction of a launch.  Free pages are those without a name in `refs`, the lowest first: nothing else has to be
// kept, and which page a call takes does not depend on the order in which its threads run.
#include <algorithm>

#include "kq_cache.cuh"

namespace kq {
namespace {

constexpr int kBookThreads = 1024;
constexpr int kPagesAThread = 4;    // neighbours that a thread looks at when pages are counted
constexpr uint32_t kMaxCluster = 8;
constexpr int kFew = 8;             // table entries that a thread takes
constexpr int kOneThreads = 1 << 30;  // beside a row's pages: such a one
constexpr uint32_t kChunk = 128;    // table entries that a warp takes at a time
constexpr int kLowest = -0x7fffffff;

struct BookParams {
  PageBook book;
  const int* news;     // grow
  const int* parents;  // fork
  const int* keep;     // ... null: all
  int* pairs;          // fork [sequences][2], compact [pages][2]
  int* list;           // scratch [pages]: free pages in order
  int* moves;          // scratch [pages]: compact: pages that move, in order
  int* place;          // scratch [pages]: compact: a moving page's place in `moves`
  int4* state;         // scratch [sequences]: what a step found, for the steps behind it
  int* stage;          // scratch [sequences][width]: fork: new rows, until every old one has been read
};

constexpr uint32_t kKept = 1024;  // sequences whose numbers are kept in shared memory

struct Shared {
  int4 kept[kKept];   // what a sequence becomes,
  int tail[kKept];    // its last page where that is not full,
  int4 state[kKept];  // what a step found, for the steps behind it (beyond kKept: in the scratch)
  int totals[2][kMaxCluster];  // of the CTAs, turn about
  long long warps[32];
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cta_count() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
// All of the call's threads have come here, and see what the others wrote (read past L1, which others' writes do not reach).
__device__ __forceinline__ void sync_all(uint32_t ctas) {
  if (ctas == 1) __syncthreads();
  else cluster_sync_all();
}
// In front of the first write into another CTA's shared memory: all of them have begun.
__device__ __forceinline__ void begin_all(uint32_t ctas) {
  if (ctas > 1) cluster_sync_all();
}
__device__ __forceinline__ int fresh(const int* p) { return __ldcg(p); }
__device__ __forceinline__ void put_remote(int* local, uint32_t rank, int value) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(local))), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(value) : "memory");
}

// Sum of the values of the block's threads in front of the calling one; `total`: of all of them.
template <typename T>
__device__ __forceinline__ T block_before(Shared& s, T value, T& total) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const auto upto_of = [&](T v) {
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const T other = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= static_cast<uint32_t>(o)) v += other;
    }
    return v;
  };
  const T upto = upto_of(value);
  if (lane == 31) s.warps[warp] = upto;
  __syncthreads();
  const T mine = static_cast<T>(s.warps[lane]), sum = upto_of(mine);
  total = __shfl_sync(0xffffffffu, sum, 31);
  const T before = __shfl_sync(0xffffffffu, sum - mine, warp);
  __syncthreads();  // s.warps belongs to the next sum
  return before + upto - value;
}
__device__ __forceinline__ int block_most(Shared& s, int value) {
  const int of_warp = __reduce_max_sync(0xffffffffu, value);
  if (threadIdx.x % 32 == 0) s.warps[threadIdx.x / 32] = of_warp;
  __syncthreads();
  const int most = __reduce_max_sync(0xffffffffu, static_cast<int>(s.warps[threadIdx.x % 32]));
  __syncthreads();
  return most;
}

// The cluster's CTAs' totals: those in front of the calling CTA, and of all.  `turn` counts the calls.
__device__ __forceinline__ int2 cluster_before(Shared& s, int total, uint32_t rank, uint32_t ctas, uint32_t& turn) {
  if (ctas == 1) {
    __syncthreads();
    return make_int2(0, total);
  }
  int* const of = s.totals[turn++ & 1];
  if (threadIdx.x < ctas) put_remote(of + rank, threadIdx.x, total);
  cluster_sync_all();
  int2 r = make_int2(0, 0);
  for (uint32_t i = 0; i < ctas; ++i) {
    if (i < rank) r.x += of[i];
    r.y += of[i];
  }
  return r;
}

// Pages of from .. to that are `used` (or not), in order, into list[0 .. limit); returns how many were found (the scan ends with the
// step that reaches the limit).
__device__ __forceinline__ int ranked(const BookParams& p, Shared& s, bool used, uint32_t from, uint32_t to, int limit, int* list, uint32_t rank, uint32_t ctas,
                                      uint32_t& turn) {
  int found = 0;
  for (uint32_t base = from; base < to && found < limit; base += ctas * kBookThreads * kPagesAThread) {
    const uint32_t at = base + (rank * kBookThreads + threadIdx.x) * kPagesAThread;
    uint32_t is = 0;
#pragma unroll
    for (int i = 0; i < kPagesAThread; ++i)
      if (at + i < to && (fresh(p.book.refs + at + i) != 0) == used) is |= 1u << i;
    int total;
    int before = block_before(s, __popc(is), total);
    const int2 all = cluster_before(s, total, rank, ctas, turn);
    before += found + all.x;
    found += all.y;
#pragma unroll
    for (int i = 0; i < kPagesAThread; ++i)
      if (is >> i & 1) {
        if (before < limit) list[before] = static_cast<int>(at + i);
        ++before;
      }
  }
  return found;
}

__device__ __forceinline__ int pages_of(int tokens, uint32_t shift) { return static_cast<int>((static_cast<uint32_t>(tokens) + (1u << shift) - 1) >> shift); }
// A sequence's tokens, as many as its row has room for.
__device__ __forceinline__ int length_of(const PageBook& k, uint32_t b) {
  const uint64_t room = static_cast<uint64_t>(k.width) << k.shift;
  return static_cast<int>(min(static_cast<uint64_t>(max(k.lengths[b], 0)), min(room, static_cast<uint64_t>(0x7fffffff))));
}
__device__ __forceinline__ bool a_page(const PageBook& k, int page) { return static_cast<uint32_t>(page) < k.pages; }

__device__ __forceinline__ void tell(const BookParams& p, int missing, int pages, int pairs) {
  if (cta_rank() == 0 && threadIdx.x == 0) {
    p.book.report[0] = missing;
    p.book.report[1] = pages;
    p.book.report[2] = pairs;
    p.book.report[3] = 0;
  }
}
// Every (sequence, chunk of its row up to `entries`) once over the cluster's warps.
__device__ __forceinline__ void put_state(const BookParams& p, Shared& s, uint32_t b, bool mine, const int4& v) {
  if (b < kKept) s.state[b] = v;  // every CTA for itself
  else if (mine) p.state[b] = v;
}
__device__ __forceinline__ int4 state_of(const BookParams& p, const Shared& s, uint32_t b) { return b < kKept ? s.state[b] : __ldcg(p.state + b); }
template <typename Use>
__device__ __forceinline__ void each_chunk(const PageBook& k, uint32_t entries, uint32_t rank, uint32_t ctas, Use use) {
  const uint32_t chunks = (entries + kChunk - 1) / kChunk, warps = ctas * (kBookThreads / 32);
  const uint64_t all = static_cast<uint64_t>(k.sequences) * chunks;
  for (uint64_t u = rank * (kBookThreads / 32) + threadIdx.x / 32; u < all; u += warps) use(static_cast<uint32_t>(u / chunks), static_cast<uint32_t>(u % chunks) * kChunk);
}

__global__ void __launch_bounds__(kBookThreads, 1) pages_grow_kernel(const BookParams p) {
  __shared__ Shared s;
  const uint32_t rank = cta_rank(), ctas = cta_count(), lane = threadIdx.x % 32;
  uint32_t turn = 0;
  pdl_launch_dependents();
  begin_all(ctas);
  pdl_wait_prior_grid();
  const PageBook& k = p.book;
  const uint64_t room = static_cast<uint64_t>(k.width) << k.shift;
  // what each sequence needs, every CTA for itself
  long long need = 0;
  int most = 0;
  bool bad = false;
  for (uint32_t b0 = 0; b0 < k.sequences; b0 += kBookThreads) {
    const uint32_t b = b0 + threadIdx.x;
    int length = 0, news = 0, held = 0, more = 0;
    if (b < k.sequences) {
      length = length_of(k, b);
      news = max(p.news[b], 0);
      const uint64_t wanted = static_cast<uint64_t>(length) + static_cast<uint64_t>(news);
      if (wanted > room || wanted > 0x7fffffffull) bad = true;
      held = pages_of(length, k.shift);
      more = bad ? 0 : pages_of(length + news, k.shift) - held;
    }
    long long total;
    const long long before = need + block_before(s, static_cast<long long>(more), total);
    // (numbers beyond 31 bits are of a call that has too few pages)
    if (b < k.sequences) put_state(p, s, b, b0 / kBookThreads % ctas == rank, make_int4(length + (bad ? 0 : news), held, more, static_cast<int>(min(before, 0x7fffffffll))));
    need += total;
    most = max(most, more);
  }
  bad = __syncthreads_or(bad);
  most = block_most(s, most);
  if (bad) {
    tell(p, -1, 0, 0);
    return;
  }
  const int limit = static_cast<int>(min(need, static_cast<long long>(k.pages) + 1));
  const int found = need ? ranked(p, s, false, 0, k.pages, limit, p.list, rank, ctas, turn) : 0;
  if (found < need) {
    tell(p, static_cast<int>(min(need - found, 0x7fffffffll)), 0, 0);
    return;
  }
  sync_all(ctas);  // the list and the states
  each_chunk(k, static_cast<uint32_t>(most), rank, ctas, [&](uint32_t b, uint32_t from) {
    const int4 st = state_of(p, s, b);
    for (uint32_t i = from + lane; i < from + kChunk && static_cast<int>(i) < st.z; i += 32) {
      const int page = fresh(p.list + st.w + i);
      k.table[static_cast<size_t>(b) * k.width + st.y + i] = page;
      k.refs[page] = 1;
    }
  });
  for (uint32_t b = rank * kBookThreads + threadIdx.x; b < k.sequences; b += ctas * kBookThreads) k.lengths[b] = state_of(p, s, b).x;
  tell(p, 0, static_cast<int>(need), 0);
}

// What sequence b becomes: the first n tokens of its parent.
struct Becomes {
  int parent, n, old;
  bool changes;
};
__device__ __forceinline__ Becomes becomes(const BookParams& p, uint32_t b) {
  Becomes r;
  r.parent = p.parents[b];
  r.old = length_of(p.book, b);
  r.n = 0;
  if (r.parent >= 0) {
    r.n = static_cast<uint32_t>(r.parent) == b ? r.old : length_of(p.book, static_cast<uint32_t>(r.parent));
    if (p.keep) r.n = min(r.n, max(p.keep[b], 0));
  }
  r.changes = r.parent < 0 ? r.old > 0 : static_cast<uint32_t>(r.parent) != b || r.n < r.old;
  return r;
}

// (for the first kKept sequences, from where the block has put it)
__device__ __forceinline__ Becomes becomes_again(const BookParams& p, const Shared& s, uint32_t b) {
  if (b >= kKept) return becomes(p, b);
  const int4 v = s.kept[b];
  return Becomes{v.x, v.y, v.z, v.w != 0};
}

__global__ void __launch_bounds__(kBookThreads, 1) pages_fork_kernel(const BookParams p) {
  __shared__ Shared s;
  const uint32_t rank = cta_rank(), ctas = cta_count(), lane = threadIdx.x % 32;
  uint32_t turn = 0;
  pdl_launch_dependents();
  begin_all(ctas);
  pdl_wait_prior_grid();
  const PageBook& k = p.book;
  const auto no_pairs = [&](uint32_t from) {
    for (uint32_t i = 2 * from + rank * kBookThreads + threadIdx.x; i < 2 * k.sequences; i += ctas * kBookThreads) p.pairs[i] = -1;
  };
  bool bad = false;
  int entries = 0;  // of any row that changes, old or new
  for (uint32_t b = threadIdx.x; b < k.sequences; b += kBookThreads) {
    if (p.parents[b] >= static_cast<int>(k.sequences)) {
      bad = true;
    } else {
      const Becomes w = becomes(p, b);
      if (b < kKept) s.kept[b] = make_int4(w.parent, w.n, w.old, w.changes);
      const bool cut = w.parent >= 0 && static_cast<uint32_t>(w.parent) == b && pages_of(w.old, k.shift) - (w.n >> k.shift) <= kFew;
      if (w.changes && !cut) entries = max(entries, pages_of(max(w.n, w.old), k.shift));
    }
  }
  bad = __syncthreads_or(bad);
  entries = block_most(s, entries);
  if (bad) {
    tell(p, -1, 0, 0);
    no_pairs(0);
    return;
  }
  // ---- the names that rows give up, and those of whole pages that they take -------------------------
  // A row that gives up its last few pages only is one thread's (a warp looks at all of a row: 256 rows of 500 pages, cut by one each, took
  // 5 us more); `entries` is of the others.
  const auto few_given = [&](const Becomes& w, uint32_t b) {
    return w.changes && w.parent >= 0 && static_cast<uint32_t>(w.parent) == b && pages_of(w.old, k.shift) - (w.n >> k.shift) <= kFew;
  };
  const auto names = [&](int by) {
    for (uint32_t b = rank * kBookThreads + threadIdx.x; b < k.sequences; b += ctas * kBookThreads) {
      const Becomes w = becomes_again(p, s, b);
      if (!few_given(w, b)) continue;
      const int whole = w.n >> k.shift, held = pages_of(w.old, k.shift);
      for (int i = whole; i < held; ++i) {
        const int page = k.table[static_cast<size_t>(b) * k.width + i];
        if (a_page(k, page)) atomicSub(k.refs + page, by);
      }
    }
    each_chunk(k, static_cast<uint32_t>(entries), rank, ctas, [&](uint32_t b, uint32_t from) {
      const Becomes w = becomes_again(p, s, b);
      if (!w.changes || few_given(w, b) || static_cast<int>(from) >= pages_of(max(w.n, w.old), k.shift)) return;
      const bool same = w.parent >= 0 && static_cast<uint32_t>(w.parent) == b;
      const int whole = w.n >> k.shift, held = pages_of(w.old, k.shift);
      const int* const mine = k.table + static_cast<size_t>(b) * k.width;
      const int* const theirs = k.table + static_cast<size_t>(max(w.parent, 0)) * k.width;
      constexpr int kEach = kChunk / 32;
      int given[kEach], taken[kEach];  // all loads first
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = static_cast<int>(from + lane) + 32 * j;
        given[j] = i < held && !(same && i < whole) ? mine[i] : -1;
        taken[j] = i < whole && !same ? theirs[i] : -1;
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = static_cast<int>(from + lane) + 32 * j;
        if (a_page(k, given[j])) atomicSub(k.refs + given[j], by);
        if (a_page(k, taken[j])) atomicAdd(k.refs + taken[j], by);
        if (i < whole && !same) p.stage[static_cast<size_t>(b) * k.width + i] = taken[j];
      }
    });
  };
  names(1);
  sync_all(ctas);
  // ---- last pages that are not full: one that nobody names goes to the lowest sequence ----------------
  const auto tail_of = [&](const Becomes& w) {
    return w.changes && (w.n & ((1 << k.shift) - 1)) ? k.table[static_cast<size_t>(w.parent) * k.width + (w.n >> k.shift)] : -1;
  };
  for (uint32_t b = threadIdx.x; b < min(k.sequences, kKept); b += kBookThreads) s.tail[b] = tail_of(becomes_again(p, s, b));
  __syncthreads();
  for (uint32_t b = rank * kBookThreads + threadIdx.x; b < k.sequences; b += ctas * kBookThreads) {
    const int page = b < kKept ? s.tail[b] : tail_of(becomes_again(p, s, b));
    if (a_page(k, page) && fresh(k.refs + page) <= 0) atomicMin(k.refs + page, kLowest + static_cast<int>(b));
  }
  sync_all(ctas);
  int need = 0;
  for (uint32_t b0 = 0; b0 < k.sequences; b0 += kBookThreads) {
    const uint32_t b = b0 + threadIdx.x;
    Becomes w = {};
    int page = -1, place = -1;
    if (b < k.sequences) {
      w = becomes_again(p, s, b);
      page = b < kKept ? s.tail[b] : tail_of(w);
      if (a_page(k, page)) place = fresh(k.refs + page) == kLowest + static_cast<int>(b) ? -2 : 0;  // takes it over, or needs another
    }
    int total;
    const int before = block_before(s, place == 0 ? 1 : 0, total);
    if (place == 0) place = need + before;
    need += total;
    if (b < k.sequences)
      put_state(p, s, b, b0 / kBookThreads % ctas == rank, make_int4(w.changes ? w.n : -1, pages_of(w.old, k.shift) | (few_given(w, b) ? kOneThreads : 0), page, place));
  }
  const int found = need ? ranked(p, s, false, 0, k.pages, need, p.list, rank, ctas, turn) : 0;
  sync_all(ctas);  // the list, the states; every look at `refs`
  const bool enough = found >= need;
  for (uint32_t b = rank * kBookThreads + threadIdx.x; b < k.sequences; b += ctas * kBookThreads) {
    const int4 st = state_of(p, s, b);
    if (st.w == -2) k.refs[st.z] = enough ? 1 : 0;
  }
  if (!enough) {  // all as it was
    sync_all(ctas);
    names(-1);
    tell(p, need - found, 0, 0);
    no_pairs(0);
    return;
  }
  // ---- the new rows ---------------------------------------------------------------------------------
  each_chunk(k, static_cast<uint32_t>(entries), rank, ctas, [&](uint32_t b, uint32_t from) {
    const int4 st = state_of(p, s, b);
    if (st.x < 0) return;
    const int whole = st.x >> k.shift, all = pages_of(st.x, k.shift);
    if ((st.y & kOneThreads) || static_cast<int>(from) >= max(all, st.y)) return;
    const bool same = (b < kKept ? s.kept[b].x : p.parents[b]) == static_cast<int>(b);
    for (int i = static_cast<int>(from + lane); i < static_cast<int>(from + kChunk); i += 32) {
      int* const entry = k.table + static_cast<size_t>(b) * k.width + i;
      if (i < whole) {
        if (!same) *entry = fresh(p.stage + static_cast<size_t>(b) * k.width + i);
      } else if (i < all) {
        *entry = st.w >= 0 ? fresh(p.list + st.w) : st.z;
      } else if (i < st.y) {
        *entry = -1;
      }
    }
  });
  for (uint32_t b = rank * kBookThreads + threadIdx.x; b < k.sequences; b += ctas * kBookThreads) {
    const int4 st = state_of(p, s, b);
    if (st.x >= 0 && (st.y & kOneThreads)) {
      for (int i = st.x >> k.shift; i < (st.y & ~kOneThreads); ++i)
        k.table[static_cast<size_t>(b) * k.width + i] = i < pages_of(st.x, k.shift) ? (st.w >= 0 ? fresh(p.list + st.w) : st.z) : -1;
    }
    if (st.x >= 0) k.lengths[b] = st.x;
    if (st.w >= 0) {
      const int page = fresh(p.list + st.w);
      k.refs[page] = 1;
      p.pairs[2 * st.w] = st.z;
      p.pairs[2 * st.w + 1] = page;
    }
  }
  no_pairs(static_cast<uint32_t>(need));
  tell(p, 0, need, need);
}

__global__ void __launch_bounds__(kBookThreads, 1) pages_compact_kernel(const BookParams p) {
  __shared__ Shared s;
  const uint32_t rank = cta_rank(), ctas = cta_count(), lane = threadIdx.x % 32;
  uint32_t turn = 0;
  pdl_launch_dependents();
  begin_all(ctas);
  pdl_wait_prior_grid();
  const PageBook& k = p.book;
  int mine = 0;
  for (uint32_t i = rank * kBookThreads + threadIdx.x; i < k.pages; i += ctas * kBookThreads) mine += k.refs[i] != 0;
  int total;
  block_before(s, mine, total);
  const uint32_t used = static_cast<uint32_t>(cluster_before(s, total, rank, ctas, turn).y);
  const int holes = ranked(p, s, false, 0, used, static_cast<int>(used), p.list, rank, ctas, turn);
  ranked(p, s, true, used, k.pages, holes, p.moves, rank, ctas, turn);  // as many
  sync_all(ctas);
  for (uint32_t i = rank * kBookThreads + threadIdx.x; i < k.pages; i += ctas * kBookThreads) {
    int from = -1, to = -1;
    if (static_cast<int>(i) < holes) {
      from = fresh(p.moves + i);
      to = fresh(p.list + i);
      k.refs[to] = fresh(k.refs + from);
      k.refs[from] = 0;
      p.place[from] = static_cast<int>(i);
    }
    p.pairs[2 * i] = from;
    p.pairs[2 * i + 1] = to;
  }
  sync_all(ctas);
  each_chunk(k, k.width, rank, ctas, [&](uint32_t b, uint32_t first) {
    const int held = pages_of(length_of(k, b), k.shift);
    for (int i = static_cast<int>(first + lane); i < static_cast<int>(first + kChunk) && i < held; i += 32) {
      int* const entry = k.table + static_cast<size_t>(b) * k.width + i;
      const int page = *entry;
      if (!a_page(k, page) || static_cast<uint32_t>(page) < used) continue;
      const int place = fresh(p.place + page);  // a page that the counts do not know has none: anything is there
      if (static_cast<uint32_t>(place) < static_cast<uint32_t>(holes) && fresh(p.moves + place) == page) *entry = fresh(p.list + place);
    }
  });
  tell(p, 0, static_cast<int>(used), holes);
}

// ---- copies -----------------------------------------------------------------------------------------
// Bulk copies into shared memory and out of it, a warp with a ring of stages: no registers, and what is under way does not depend on how
// many threads an SM holds.  Of 96 KB a CTA, two CTAs an SM, a third is on its way in, the rest on its way out: 1660 pages of 69,632 bytes in
// eight pools 290 us (6.37 TB/s, 0.97 of the copy rate); half and half 320, 32 KB pieces and one CTA 296.
constexpr uint32_t kPiece = 16384, kStages = 6, kAhead = 2;
constexpr uint32_t kCopySmem = kStages * kPiece + 256;
constexpr uint32_t kCopyWaitLimit = 1u << 22;
constexpr int kCopyTimeout = 60;  // status word: a piece did not arrive

struct CopyParams {
  uint8_t* pool[kPoolsAtOnce];
  uint64_t bytes[kPoolsAtOnce];  // of a page
  const int* pairs;
  const int* report;  // null: all `most` pairs,
  bool until_end;     // or those in front of the first negative one
  int* status;
  uint32_t pools, pages, most, parts;  // parts that a page is copied in, kPiece or less each
};

// How many pairs are in front of the first negative one, or `most`; by a warp, 32 places at a time: as many trips to memory as a report up to 32 pairs, one
// more for every factor of 32 (7696 pairs: 3, of a copy of 290 us).
__device__ __forceinline__ uint32_t pairs_until_end(const int* pairs, uint32_t most) {
  uint32_t lo = 0, hi = most;  // pairs in front of lo, none at hi
  while (lo < hi) {
    const uint32_t at = lo + static_cast<uint32_t>(static_cast<uint64_t>(hi - lo) * (threadIdx.x % 32) / 32);
    const uint32_t none = __ballot_sync(0xffffffffu, __ldcg(pairs + 2 * static_cast<size_t>(at)) < 0);
    const int first = none ? __ffs(static_cast<int>(none)) - 1 : 32;  // the lane whose place is the first without a pair
    if (first < 32) hi = __shfl_sync(0xffffffffu, at, first);
    if (first > 0) lo = __shfl_sync(0xffffffffu, at, first - 1) + 1;
  }
  return hi;
}

// kWords: some pages are not whole sixteen bytes (without it: 307 us instead of 309 for the 1660 pages and the compaction in front of them).
template <bool kWords>
__global__ void __launch_bounds__(32) pages_copy_kernel(const __grid_constant__ CopyParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* const targets = reinterpret_cast<uint64_t*>(smem + kStages * kPiece);
  uint32_t* const sizes = reinterpret_cast<uint32_t*>(targets + kStages);
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), bars = base + kStages * kPiece + 128, lane = threadIdx.x;
  if (lane < kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + lane * 8) : "memory");
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  const uint32_t count = p.until_end ? pairs_until_end(p.pairs, p.most) : p.report ? min(static_cast<uint32_t>(max(p.report[2], 0)), p.most) : p.most;
  const uint64_t all = static_cast<uint64_t>(count) * p.pools * p.parts;
  uint32_t n = 0;     // pieces asked for
  uint32_t done = 0;  // pieces handed on
  bool ok = true;
  // piece `done`, which has arrived: on its way out
  const auto hand_on = [&] {
    const uint32_t stage = done % kStages, bar = bars + stage * 8, parity = done / kStages & 1;
    uint32_t here = 0;
    for (uint32_t spin = 0; spin < kCopyWaitLimit && !here; ++spin)
      asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(here) : "r"(bar), "r"(parity) : "memory");
    if (!here) {
      ok = false;
      *reinterpret_cast<volatile int*>(p.status) = kCopyTimeout;
      return;
    }
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(targets[stage]), "r"(base + stage * kPiece), "r"(sizes[stage]) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    ++done;
  };
  for (uint64_t item0 = blockIdx.x; item0 < all; item0 += 32ull * gridDim.x) {
    // thirty-two pieces' addresses, a lane each
    const uint64_t item = item0 + static_cast<uint64_t>(lane) * gridDim.x;
    uint64_t from_at = 0, to_at = 0;
    uint32_t bytes = 0;
    bool words = false;
    if (item < all) {
      const uint32_t part = static_cast<uint32_t>(item % p.parts);
      const uint64_t of = item / p.parts;
      const uint32_t pool = static_cast<uint32_t>(of % p.pools), pair = static_cast<uint32_t>(of / p.pools);
      const uint32_t from = static_cast<uint32_t>(p.pairs[2 * pair]), to = static_cast<uint32_t>(p.pairs[2 * pair + 1]);
      if (from < p.pages && to < p.pages && from != to) {
        const uint64_t size = p.bytes[pool], each = ((kWords ? size + 15 : size) / 16 + p.parts - 1) / p.parts * 16, begin = min(part * each, size);
        bytes = static_cast<uint32_t>(min(each, size - begin));
        from_at = reinterpret_cast<uint64_t>(p.pool[pool]) + from * size + begin;
        to_at = reinterpret_cast<uint64_t>(p.pool[pool]) + to * size + begin;
        if constexpr (kWords) words = ((reinterpret_cast<uint64_t>(p.pool[pool]) | size) & 15) != 0;
      }
    }
    // such pages (two numbers a kv head, of an odd number of heads): the warp's, four bytes a lane
    for (uint32_t left = kWords ? __ballot_sync(0xffffffffu, bytes != 0 && words) : 0; left; left &= left - 1) {
      const int l = __ffs(left) - 1;
      const uint32_t* const src = reinterpret_cast<const uint32_t*>(__shfl_sync(0xffffffffu, from_at, l));
      uint32_t* const dst = reinterpret_cast<uint32_t*>(__shfl_sync(0xffffffffu, to_at, l));
      const uint32_t count4 = __shfl_sync(0xffffffffu, bytes, l) / 4;
      constexpr uint32_t kBatch = 8;
      for (uint32_t i0 = lane; i0 < count4; i0 += 32 * kBatch) {
        uint32_t v[kBatch];
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j)
          if (i0 + 32 * j < count4) v[j] = __ldcg(src + i0 + 32 * j);
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j)
          if (i0 + 32 * j < count4) __stcg(dst + i0 + 32 * j, v[j]);
      }
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, bytes != 0 && !words); left; left &= left - 1) {
      const int l = __ffs(left) - 1;
      const uint64_t src = __shfl_sync(0xffffffffu, from_at, l), dst = __shfl_sync(0xffffffffu, to_at, l);
      const uint32_t size = __shfl_sync(0xffffffffu, bytes, l);
      if (lane == 0 && ok) {
        if (n - done >= kAhead) hand_on();
        if (ok) {
          const uint32_t stage = n % kStages, bar = bars + stage * 8;
          asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kStages - kAhead) : "memory");  // what the stage held has left it
          targets[stage] = dst;
          sizes[stage] = size;
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(size) : "memory");
          asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(base + stage * kPiece), "l"(src), "r"(size), "r"(bar)
                       : "memory");
          ++n;
        }
      }
    }
  }
  if (lane == 0) {
    while (ok && done < n) hand_on();
    // behind a wait that gave up: the pieces on their way in are waited for once more each, so that none lands in another block's memory
    for (uint32_t i = done; !ok && i < n; ++i) {
      uint32_t here = 0;
      for (uint32_t spin = 0; spin < kCopyWaitLimit && !here; ++spin)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(here) : "r"(bars + i % kStages * 8), "r"(i / kStages & 1) : "memory");
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
}

// One cluster, of one CTA where that has all its work in a few steps: its barriers cost less (two prompts and their six beams: 8.5 us, with
// eight CTAs 12; 64 rows of 129 pages: 16.5 / 14.6).
uint32_t cluster_for(const PageBook& k) {
  const uint64_t chunks = static_cast<uint64_t>(k.sequences) * ((k.width + kChunk - 1) / kChunk);
  return k.pages <= 2 * kBookThreads * kPagesAThread && chunks <= 64 && k.sequences <= kBookThreads ? 1u : kMaxCluster;
}

template <typename Kernel>
cudaError_t launch_book(const LaunchEnv& env, Kernel kernel, const BookParams& p) {
  cudaLaunchConfig_t cfg = {};
  const uint32_t ctas = cluster_for(p.book);
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kBookThreads);
  cfg.stream = env.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = env.overlap ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

uint64_t up16(uint64_t bytes) { return (bytes + 15) / 16 * 16; }

}  // namespace

uint64_t pages_scratch_bytes(const PageBook& k, bool fork, bool compact) {
  return up16(4ull * k.pages) * (compact ? 3 : 1) + 16ull * k.sequences + (fork ? 4ull * k.sequences * k.width : 0);
}

cudaError_t launch_pages_grow(const LaunchEnv& env, const PageBook& book, const int* news) {
  BookParams p = {};
  p.book = book;
  p.news = news;
  p.list = static_cast<int*>(env.workspace);
  p.state = reinterpret_cast<int4*>(static_cast<uint8_t*>(env.workspace) + up16(4ull * book.pages));
  return launch_book(env, pages_grow_kernel, p);
}

cudaError_t launch_pages_fork(const LaunchEnv& env, const PageBook& book, const int* parents, const int* keep, int* pairs) {
  BookParams p = {};
  p.book = book;
  p.parents = parents;
  p.keep = keep;
  p.pairs = pairs;
  p.list = static_cast<int*>(env.workspace);
  p.state = reinterpret_cast<int4*>(static_cast<uint8_t*>(env.workspace) + up16(4ull * book.pages));
  p.stage = reinterpret_cast<int*>(p.state + book.sequences);
  return launch_book(env, pages_fork_kernel, p);
}

cudaError_t launch_pages_compact(const LaunchEnv& env, const PageBook& book, int* pairs) {
  BookParams p = {};
  p.book = book;
  p.pairs = pairs;
  p.list = static_cast<int*>(env.workspace);
  p.moves = p.list + up16(4ull * book.pages) / 4;
  p.place = p.moves + up16(4ull * book.pages) / 4;
  return launch_book(env, pages_compact_kernel, p);
}

cudaError_t launch_pages_copy(const LaunchEnv& env, uint32_t count, const uint64_t* pools, const uint64_t* page_bytes, uint32_t pages, const int* pairs,
                              uint32_t most, const int* report, bool until_end) {
  static OncePerDevice once;
  cudaError_t e = once.run([] {
    const cudaError_t e = cudaFuncSetAttribute(pages_copy_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopySmem);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(pages_copy_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopySmem);
  });
  if (e != cudaSuccess) return e;
  bool words = false;
  CopyParams p;
  uint64_t largest = 0;
  for (uint32_t i = 0; i < count; ++i) {
    p.pool[i] = reinterpret_cast<uint8_t*>(pools[i]);
    p.bytes[i] = page_bytes[i];
    largest = std::max(largest, page_bytes[i]);
    words |= ((pools[i] | page_bytes[i]) & 15) != 0;
  }
  p.pairs = pairs;
  p.report = report;
  p.until_end = until_end;
  p.status = env.status;
  p.pools = count;
  p.pages = pages;
  p.most = most;
  p.parts = static_cast<uint32_t>((largest + kPiece - 1) / kPiece);
  const uint64_t items = static_cast<uint64_t>(most) * count * p.parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<uint64_t>(items, static_cast<uint64_t>(env.sm_count) * 2)));
  cfg.blockDim = dim3(32);
  cfg.dynamicSmemBytes = kCopySmem;
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, words ? pages_copy_kernel<true> : pages_copy_kernel<false>, p);
}

}  // namespace kq
