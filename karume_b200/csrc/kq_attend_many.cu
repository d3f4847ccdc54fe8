// Attention over the paged 4-bit cache (layout in kq_cache.cuh) for many query rows a sequence: prompts, on the tcgen05
// tensor cores.
//
//   out = sum_j softmax_j(scale q . k_j) v_j,   k_j = u_j s_j + o_j, v_j likewise, codes u in 0..15
//
// A CTA takes 256 query rows (query and head of one kv head's group, packed: all heads of the group share what is unpacked)
// and walks over the keys they see in tiles of 128.  Warps:
//   0-3, 4-7   one row each thread of the first / second 128 rows: scores from tensor memory, weights back into it, and
//              the sums of the output in registers (what the tensor core adds is one tile's, so a long row does not drift)
//   8-11       unpack a tile: keys as [token][dim], values transposed as [dim][token], both K-major with 128-byte swizzle
//   12         issues the MMAs:   S_r = Q_r K^T (both in shared memory),   O_r = P_r V (P in tensor memory, over S)
//   13         copies the codes and scales of the next tile (bulk copies, page by page)
// The two row blocks take turns: while one's weights are being computed the tensor core works for the other.
//
//   16-bit queries  keys and values are unpacked to what they stand for, rounded to binary16 once (2^-11, as the weights).
//   f32 queries     codes enter exactly: keys as the subnormals u 2^-24 and u 2^-20 that their bits already are, values as
//                   codes around zero; scale and offset are applied to the scores and weights in f32.  Queries and weights are
//                   two binary16 parts each (fixed-point, the low ones multiplied first), 22 bits and more.
#include <algorithm>

#include "kq_cache.cuh"
#include "kq_umma.cuh"

namespace kq {
namespace {

constexpr int kManyThreads = 512;
constexpr int kKeys = 128;    // of a tile
constexpr int kBlock = 256;   // query rows of a CTA
constexpr int kManyTimeout = 50;

template <typename T, int D>
struct Many {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kParts = kSplit ? 2 : 1;
  static constexpr int kOperand = 128 * D * 2;             // bytes of 128 rows (or tokens) of D values
  static constexpr int kBufs = kSplit && D == 128 ? 1 : 2;  // unpacked tiles: as many as fit beside the queries
  static constexpr int kGroup = 4 * D + 16;                // raw values of eight tokens, 16 bytes apart: lanes of eight groups meet no bank twice
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kParts * kOperand;
  static constexpr int kV = kK + kBufs * kOperand;
  static constexpr int kRawK = kV + kBufs * kOperand;
  static constexpr int kRawV = kRawK + kKeys * (D / 2);
  static constexpr int kRawParams = kRawV + 16 * kGroup;   // K, then V (scale, offset)
  static constexpr int kTable = kRawParams + 2 * kKeys * 4;  // f32: [2][128] (ks, ko, vs, v mid); 16-bit: K pairs, V scales, V offsets
  static constexpr int kRows = kTable + 2 * kKeys * 16;    // [256] (factor, sum, last key, first key)
  static constexpr int kLost = kRows + kBlock * 16;        // [2] 128 bits: tokens whose value is NaN
  static constexpr int kBinade = kLost + 32;               // [2][4]: largest binade of the values' scales, by warp
  static constexpr int kBars = kBinade + 32;
  static constexpr int kMisc = kBars + 18 * 8;
  static constexpr int kSmem = kMisc + 64 + 1024;          // the operands start on a multiple of 1024
};

struct ManyParams {
  AttendArgs a;
  uint32_t group, page_shift, beyond;  // sequences of more than `beyond` query rows a kv head are this kernel's
  int* status;
};

enum Bar { kRawKFull, kRawKFree, kRawVFull, kRawVFree, kKFull, kKEmpty = 6, kVFull = 8, kVEmpty = 10, kSFull = 12, kPReady = 14, kOFull = 16, kBarCount = 18 };

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hadd2_bits(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Sixteen columns of the thread's lane: begun, and (behind the wait) there.
__device__ __forceinline__ void tmem_ld16_begin(uint32_t taddr, float (&f)[16]) {
  uint32_t* v = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
        "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16_done(float (&f)[16]) {
  uint32_t* v = reinterpret_cast<uint32_t*>(f);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// N columns, sixteen at a time: use(column, values), the next ones on their way meanwhile
template <int N, typename Use>
__device__ __forceinline__ void tmem_columns(uint32_t taddr, Use use) {
  float x[2][16];
  tmem_ld16_begin(taddr, x[0]);
#pragma unroll
  for (int c = 0; c < N / 16; ++c) {
    tmem_ld16_done(x[c & 1]);
    if (c + 1 < N / 16) tmem_ld16_begin(taddr + (c + 1) * 16, x[(c + 1) & 1]);
    use(c * 16, x[c & 1]);
  }
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// binary16 operands, f32 accumulators; descriptors by their low words
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
               ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(umma::kDescHigh), "r"(leader) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 y, {%2, %5};\n\t"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
               ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "r"(umma::kDescHigh), "r"(leader) : "memory");
}
__device__ __forceinline__ uint32_t desc_low(uint32_t smem) { return ((smem >> 4) & 0x3FFFu) | (1u << 16); }
__host__ __device__ constexpr uint32_t f16_idesc(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(half2_bits(v[0], v[1]), half2_bits(v[2], v[3]), half2_bits(v[4], v[5]), half2_bits(v[6], v[7]));
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* v) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    r[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kManyThreads, 1) attend_many_kernel(const __grid_constant__ ManyParams p) {
  using F = Many<T, D>;
  constexpr int kParts = F::kParts, kBufs = F::kBufs;
  constexpr bool kSplit = F::kSplit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + (1024 - (static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw)) & 1023u)) % 1024;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  float4* const rows = reinterpret_cast<float4*>(smem + F::kRows);
  uint32_t* const tmem_word = reinterpret_cast<uint32_t*>(smem + F::kMisc + 16);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + F::kMisc + 20);
  uint32_t* const found = reinterpret_cast<uint32_t*>(smem + F::kMisc + 24);  // sequence, number in it
  const auto bar = [&](int i) { return base + F::kBars + i * 8; };
  const auto wait = [&](int i, uint32_t parity) {
    const bool ok = umma::wait_bounded(bar(i), parity & 1u, abort_flag, p.status, kManyTimeout);
    __syncwarp();  // what follows is often an aligned instruction
    return ok;
  };

  if (tid == 0) {
    umma::mbar_init(bar(kRawKFull), 1);
    umma::mbar_init(bar(kRawVFull), 1);
    umma::mbar_init(bar(kRawKFree), 128);
    umma::mbar_init(bar(kRawVFree), 128);
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(bar(kKFull + i), 128);
      umma::mbar_init(bar(kVFull + i), 128);
      umma::mbar_init(bar(kKEmpty + i), 1);
      umma::mbar_init(bar(kVEmpty + i), 1);
      umma::mbar_init(bar(kSFull + i), 1);
      umma::mbar_init(bar(kOFull + i), 1);
      umma::mbar_init(bar(kPReady + i), 128);
    }
    *abort_flag = 0;
    found[0] = 0xFFFFFFFFu;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  __syncthreads();

  // ---- which rows: units are (sequence, block of rows from the last, kv head) ----------------------
  const uint32_t sequences = p.a.batch.sequences, each = (sequences + kManyThreads - 1) / kManyThreads, heads = p.a.cache.kv_heads;
  const auto blocks_of = [&](uint32_t b) {
    const Span s = span_of(p.a.batch, b);
    const uint64_t n = static_cast<uint64_t>(s.count) * p.group;
    return s.length > 0 && n > p.beyond ? static_cast<uint32_t>((n + kBlock - 1) / kBlock) : 0u;
  };
  uint32_t mine = 0;
  for (uint32_t b = tid * each; b < min((tid + 1) * each, sequences); ++b) mine += blocks_of(b) * heads;
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= static_cast<uint32_t>(o)) upto += v;
  }
  uint32_t* const scan = reinterpret_cast<uint32_t*>(smem + F::kTable);
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  for (uint32_t i = 0; i < warp; ++i) upto += scan[i];
  if (upto - mine <= blockIdx.x && blockIdx.x < upto) {
    uint32_t b = tid * each, left = blockIdx.x - (upto - mine);
    for (uint32_t n = blocks_of(b) * heads; left >= n; n = blocks_of(++b) * heads) left -= n;
    found[0] = b;
    found[1] = left;
  }
  __syncthreads();
  const uint32_t seq = found[0];
  if (seq == 0xFFFFFFFFu) return;
  const Span span = span_of(p.a.batch, seq);
  const uint32_t blocks = blocks_of(seq), head = found[1] % heads, block = blocks - 1 - found[1] / heads;  // the longest first
  const int row0 = static_cast<int>(block * kBlock), n_rows = span.count * static_cast<int>(p.group), before = span.length - span.count;
  const int window = static_cast<int>(min(p.a.window, 0x7fffffffu));
  const int q_first = row0 / static_cast<int>(p.group), q_last = min(row0 + kBlock - 1, n_rows - 1) / static_cast<int>(p.group);
  const int key_last = before + q_last;
  const int key_first = window && before + q_first + 1 > window ? before + q_first + 1 - window : 0;
  const int tile0 = key_first / kKeys, tiles = key_last < 0 ? 0 : key_last / kKeys + 1 - tile0;

  // ---- queries --------------------------------------------------------------------------------------
  {
    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
    const uint32_t c = lane % kLanes;
#pragma unroll 2
    for (uint32_t r = warp * kAtOnce + lane / kLanes; r < kBlock; r += 16 * kAtOnce) {
      const int row = row0 + static_cast<int>(r), query = row / static_cast<int>(p.group);
      const bool there = row < n_rows;
      float v[8] = {};
      if (there)
        load8_rotated(static_cast<const T*>(p.a.q) + static_cast<size_t>(span.first + query) * p.a.q_stride +
                          static_cast<size_t>(head * p.group + static_cast<uint32_t>(row - query * static_cast<int>(p.group))) * D,
                      c * 8, p.a.rope, before + query, v);
      float big = 0.0f, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        big = fmaxf(big, fabsf(v[i]));
        sum += v[i];
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2) {
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      const int e = static_cast<int>(__float_as_uint(big) >> 23);
      const int up = big > 0.0f && e < 255 ? min(max(140 - e, -100), 120) : 0;  // below 2^14
      const float lift = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
      float hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = v[i] * lift;
        if constexpr (kSplit) {  // odd dims meet codes sixteen times as large
          const float top = rintf(x * 0.125f) * 8.0f, down = (i & 1) ? 0.0625f : 1.0f;
          hi[i] = top * down;
          lo[i] = rintf((x - top) * 256.0f) * (0.00390625f * down);
        } else {
          hi[i] = x;
        }
      }
      const uint32_t at = base + F::kQ + (r / 128) * kParts * F::kOperand + (c / 8) * 16384 + umma::swz(r % 128, c % 8);
      umma::sts128(at, make_uint4(half2_bits(hi[0], hi[4]), half2_bits(hi[1], hi[5]), half2_bits(hi[2], hi[6]), half2_bits(hi[3], hi[7])));
      if constexpr (kSplit)
        umma::sts128(at + F::kOperand, make_uint4(half2_bits(lo[0], lo[4]), half2_bits(lo[1], lo[5]), half2_bits(lo[2], lo[6]), half2_bits(lo[3], lo[7])));
      if (c == 0) {
        const float factor = p.a.scale * 1.4426950408889634f;
        const int last = there ? before + query : 0x7fffffff;  // rows beyond the end see anything and are not stored
        const int from = there && window && last + 1 > window ? last + 1 - window : 0;
        // f32: score = factor 2^(24 - up) (acc ks + ko sum 2^(up - 24))
        rows[r] = kSplit ? make_float4(factor * exp2f(static_cast<float>(24 - up)), sum * exp2f(static_cast<float>(up - 24)), __int_as_float(last), __int_as_float(from))
                         : make_float4(factor * exp2f(static_cast<float>(-up)), 0.0f, __int_as_float(last), __int_as_float(from));
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(tmem_word))), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_word;

  if (warp < 8) {
    // ---- softmax and output: a row a thread --------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const uint32_t wg = warp / 4, lanes = (warp % 4 * 32) << 16;
    const uint32_t t_s = tmem + lanes + wg * 128, t_o = tmem + lanes + 256 + wg * 128;
    const int r = static_cast<int>(tid);
    const float4 rc = rows[r];
    const float factor = rc.x, q_sum = rc.y;
    const int last = __float_as_int(rc.z), from = __float_as_int(rc.w);
    const int last_all = __reduce_min_sync(0xffffffffu, last), from_all = __reduce_max_sync(0xffffffffu, from);
    float O[D];
#pragma unroll
    for (int i = 0; i < D; ++i) O[i] = 0.0f;
    float M = -INFINITY, l = 0.0f, centre = 0.0f;
    for (int j = 0; j < tiles; ++j) {
      const int first = (tile0 + j) * kKeys;
      const bool whole = first >= from_all && first + kKeys - 1 <= last_all;
      const int sees0 = from - first, sees1 = last - first;  // columns the row sees
      const float4* table = reinterpret_cast<const float4*>(smem + F::kTable) + (j & 1) * kKeys;
      wait(kSFull + wg, j);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float m = -INFINITY, binade = 0.0f;
      if constexpr (kSplit) {
        const float* bn = reinterpret_cast<const float*>(smem + F::kBinade) + (j & 1) * 4;
        binade = fmaxf(fmaxf(bn[0], bn[1]), fmaxf(bn[2], bn[3]));
      }
      float vs_big = 0.0f;
      tmem_columns<kKeys>(t_s, [&](int c, float (&x)[16]) {
        if constexpr (kSplit) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4 k = table[c + i];
            x[i] = fmaf(x[i], k.x, k.y * q_sum);
            if (!whole && c + i >= sees0 && c + i <= sees1) vs_big = fmaxf(vs_big, k.z);
          }
        }
        if (whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) m = fmaxf(m, x[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i >= sees0 && c + i <= sees1) m = fmaxf(m, x[i]);
        }
      });
      if constexpr (kSplit)
        if (!whole) binade = fmaxf(static_cast<float>(static_cast<int>(__float_as_uint(vs_big) >> 23) - 126), -14.0f);
      // M: the largest score (f32: and the binade of the values' scales); moves only when a weight would grow past 2^8
      const float top = m == -INFINITY ? m : m * factor + binade;
      const bool more = top > M + 8.0f;
      if (__any_sync(0xffffffffu, more)) {
        const float keep = !more ? 1.0f : ex2(M - top);
        if (more) M = top;
        l *= keep;
        centre *= keep;
#pragma unroll
        for (int i = 0; i < D; ++i) O[i] *= keep;
      }
      int up = 0;  // f32: P is lifted to just below 2^14 in each tile, and its sums brought back
      if constexpr (kSplit) up = top == -INFINITY ? 0 : min(max(14 - static_cast<int>(ceilf(top - M)), 0), 120);
      const float shift = (M == -INFINITY ? 0.0f : -M) + static_cast<float>(up), drop = __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
      float l_tile = 0.0f, centre_tile = 0.0f;
      tmem_columns<kKeys>(t_s, [&](int c, float (&x)[16]) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float w[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float z = x[i + k];
            float4 t = {};
            if constexpr (kSplit) {
              t = table[c + i + k];
              z = fmaf(z, t.x, t.y * q_sum);
            }
            w[k] = ex2(fmaf(z, factor, shift));
            if (!whole && (c + i + k < sees0 || c + i + k > sees1)) {
              w[k] = 0.0f;  // what is not seen may hold anything
            } else if constexpr (kSplit) {
              l_tile += w[k];
              centre_tile = fmaf(w[k], t.w, centre_tile);
              w[k] *= t.z;
            } else {
              l_tile += w[k];
            }
          }
          if constexpr (kSplit) {
            constexpr float kEight = 100663296.0f;  // 1.5 2^26: numbers beside it are multiples of eight
            const float h0 = __fsub_rn(__fadd_rn(w[0], kEight), kEight), h1 = __fsub_rn(__fadd_rn(w[1], kEight), kEight);
            hi[i / 2] = half2_bits(h0, h1);
            lo[i / 2] = half2_bits(w[0] - h0, w[1] - h1);
          } else {
            hi[i / 2] = half2_bits(w[0], w[1]);
          }
        }
        // sixteen keys' weights go where their scores were: eight columns, and eight for the low parts
        tmem_st8(t_s + c, hi);
        if constexpr (kSplit) tmem_st8(t_s + c + 8, lo);
      });
      l = fmaf(l_tile, drop, l);
      centre = fmaf(centre_tile, drop, centre);
      if constexpr (!kSplit) {
        const uint4 lost = *reinterpret_cast<const uint4*>(smem + F::kLost + (j & 1) * 16);
        if (lost.x | lost.y | lost.z | lost.w) {  // values that are NaN entered as zeros: whoever sees one is NaN
          const uint32_t bits[4] = {lost.x, lost.y, lost.z, lost.w};
          for (int i = max(sees0, 0); i <= min(sees1, kKeys - 1); ++i)
            if (bits[i / 32] >> (i % 32) & 1) l = quiet_nan();
          __syncwarp();
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      umma::mbar_arrive(bar(kPReady + wg));
      wait(kOFull + wg, j);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      tmem_columns<D>(t_o, [&](int c, float (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) O[c + i] = kSplit ? fmaf(x[i], drop, O[c + i]) : O[c + i] + x[i];
      });
    }
    const int row = row0 + r;
    if (row < n_rows) {
      const int query = row / static_cast<int>(p.group);
      T* out = static_cast<T*>(p.a.out) + static_cast<size_t>(span.first + query) * p.a.out_stride +
               static_cast<size_t>(head * p.group + static_cast<uint32_t>(row - query * static_cast<int>(p.group))) * D;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int i = 0; i < D; i += 8) {
        float o[8];
        // f32: the codes' powers of two, even dims (2 u - 15) 2^-24, odd ones (u - 7.5) 2^-20
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = kSplit ? fmaf(O[i + k], (k & 1) ? 1048576.0f : 8388608.0f, centre) * inv : O[i + k] * inv;
        store8(out + i, o);
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 12) {
      // ---- unpacking ---------------------------------------------------------------------------------
      const uint32_t t = tid - 256, w4 = warp - 8;
      constexpr uint32_t kExp = 0x64006400u, k1024 = 0xE400E400u, k16th = 0x2C002C00u, k64 = 0xD400D400u;  // 1024 | x, -1024, 1/16, -64
      constexpr uint32_t kCentre0 = 0x800F800Fu, kCentre1 = 0x80788078u;                                   // -15 2^-24, -7.5 2^-20
      uint32_t* const k_par = reinterpret_cast<uint32_t*>(smem + F::kTable);                 // 16-bit: (scale, offset) of each key
      __half* const v_scale = reinterpret_cast<__half*>(smem + F::kTable + 512);
      __half* const v_offset = v_scale + kKeys;
      const uint32_t* const raw_params = reinterpret_cast<const uint32_t*>(smem + F::kRawParams);
      bool ok = true;  // after a wait that gave up nothing is handed on: no barrier is arrived on beyond its phase
      for (int j = 0; j < tiles; ++j) {
        const int first = (tile0 + j) * kKeys;
        const uint32_t buf = j % kBufs;
        ok = wait(kRawKFull, j) && ok;
        if (j >= kBufs) wait(kKEmpty + buf, j / kBufs - 1);
        if (kBufs == 2 && j >= 2) wait(kVEmpty + buf, j / 2 - 1);  // what the softmax warps read of tile j - 2 has been read
        {
          const bool seen = first + static_cast<int>(t) <= key_last;
          uint32_t kp = seen ? raw_params[t] : 0u, vp = seen ? raw_params[kKeys + t] : 0u;
          float2 k = __half22float2(*reinterpret_cast<const __half2*>(&kp)), v = __half22float2(*reinterpret_cast<const __half2*>(&vp));
          if constexpr (kSplit) {
            reinterpret_cast<float4*>(smem + F::kTable)[(j & 1) * kKeys + t] = make_float4(k.x, k.y, v.x, fmaf(7.5f, v.x, v.y));
            const int big = __reduce_max_sync(0xffffffffu, static_cast<int>(__float_as_uint(v.x) >> 23) - 126);
            if (lane == 0) reinterpret_cast<float*>(smem + F::kBinade)[(j & 1) * 4 + w4] = static_cast<float>(max(big, -14));
          } else {
            // the largest value must stay finite in binary16: a scale that was rounded up gives one unit back
            if (fmaf(15.0f, k.x, k.y) >= 65520.0f) kp -= 1;
            if (fmaf(15.0f, v.x, v.y) >= 65520.0f) vp -= 1;
            const uint32_t lost = __ballot_sync(0xffffffffu, v.x != v.x || v.y != v.y);
            if (lane == 0) reinterpret_cast<uint32_t*>(smem + F::kLost)[(j & 1) * 4 + w4] = lost;
            if (v.x != v.x || v.y != v.y) vp = 0;
            k_par[t] = kp;
            v_scale[t] = __ushort_as_half(static_cast<unsigned short>(vp));
            v_offset[t] = __ushort_as_half(static_cast<unsigned short>(vp >> 16));
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        {
          constexpr int kPieces = D / 32;  // 16-byte pieces of a token
          const uint32_t q = t % kPieces;
          const uint32_t swap = D == 128 ? q / 2 * 2 : 0;  // pieces of the second 64 dims in another order: other banks
#pragma unroll 1
          for (uint32_t it = 0; it < kPieces; ++it) {
            const uint32_t row = (it * 128 + t) / kPieces;
            const uint4 raw = *reinterpret_cast<const uint4*>(smem + F::kRawK + row * (D / 2) + q * 16);
            const uint32_t x[4] = {swap ? raw.z : raw.x, swap ? raw.w : raw.y, swap ? raw.x : raw.z, swap ? raw.y : raw.w};
            uint32_t s2 = 0, o2 = 0;
            if constexpr (!kSplit) {
              const uint32_t kp = k_par[row];
              s2 = __byte_perm(kp, kp, 0x1010);
              o2 = __byte_perm(kp, kp, 0x3232);
            }
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) {
              const uint32_t word = q * 4 + (w ^ swap), x8 = x[w] >> 8;
              uint4 out;
              if constexpr (kSplit) {
                out = make_uint4(x[w] & 0x000F000Fu, x[w] & 0x00F000F0u, x8 & 0x000F000Fu, x8 & 0x00F000F0u);
              } else {
                out.x = hfma2_bits(hadd2_bits((x[w] & 0x000F000Fu) | kExp, k1024), s2, o2);
                out.y = hfma2_bits(hfma2_bits((x[w] & 0x00F000F0u) | kExp, k16th, k64), s2, o2);
                out.z = hfma2_bits(hadd2_bits((x8 & 0x000F000Fu) | kExp, k1024), s2, o2);
                out.w = hfma2_bits(hfma2_bits((x8 & 0x00F000F0u) | kExp, k16th, k64), s2, o2);
              }
              umma::sts128(base + F::kK + buf * F::kOperand + (word / 8) * 16384 + umma::swz(row, word % 8), out);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (ok) {
          umma::mbar_arrive(bar(kKFull + buf));
          umma::mbar_arrive(bar(kRawKFree));
        }
        ok = wait(kRawVFull, j) && ok;
        if (j >= kBufs) wait(kVEmpty + buf, j / kBufs - 1);
        {
          const uint32_t tg = lane % 8;
#pragma unroll 1
          for (uint32_t lin = w4; lin < D / 16; lin += 4) {
            const uint32_t word = lin % (D / 32) * 4 + lane / 8, atom = lin / (D / 32);
            const uint32_t* from_v = reinterpret_cast<const uint32_t*>(smem + F::kRawV + (atom * 8 + tg) * F::kGroup) + word;
            uint32_t c01[4], c23[4];  // dims 0..3 / 4..7 of two tokens
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t a = from_v[2 * k * (D / 8)], b = from_v[(2 * k + 1) * (D / 8)];
              c01[k] = __byte_perm(a, b, 0x5410);
              c23[k] = __byte_perm(a, b, 0x7632);
            }
            uint4 s4 = {}, o4 = {};
            if constexpr (!kSplit) {
              s4 = *reinterpret_cast<const uint4*>(v_scale + atom * 64 + tg * 8);
              o4 = *reinterpret_cast<const uint4*>(v_offset + atom * 64 + tg * 8);
            }
            const uint32_t s2[4] = {s4.x, s4.y, s4.z, s4.w}, o2[4] = {o4.x, o4.y, o4.z, o4.w};
            const uint32_t to = base + F::kV + buf * F::kOperand + atom * (D * 128);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              uint32_t y[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t x = d < 4 ? c01[k] : c23[k];
                if (d & 2) x >>= 8;
                if constexpr (kSplit) {
                  y[k] = (d & 1) ? hadd2_bits(x & 0x00F000F0u, kCentre1) : hfma2_bits(x & 0x000F000Fu, 0x40004000u, kCentre0);
                } else {
                  x = (d & 1) ? hfma2_bits((x & 0x00F000F0u) | kExp, k16th, k64) : hadd2_bits((x & 0x000F000Fu) | kExp, k1024);
                  y[k] = hfma2_bits(x, s2[k], o2[k]);
                }
              }
              umma::sts128(to + umma::swz(word * 8 + d, tg), make_uint4(y[0], y[1], y[2], y[3]));
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (ok) {
          umma::mbar_arrive(bar(kVFull + buf));
          umma::mbar_arrive(bar(kRawVFree));
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the 16-bit table is written anew for the next tile
      }
    } else if (warp == 12) {
      // ---- MMAs ----------------------------------------------------------------------------------------
      const uint32_t leader = umma::elect_lane();
      const auto scores = [&](int j, uint32_t r) {
        const uint32_t buf = j % kBufs, d = tmem + r * 128;
        const uint32_t q = desc_low(base + F::kQ + r * kParts * F::kOperand), k = desc_low(base + F::kK + buf * F::kOperand);
#pragma unroll
        for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            mma_ss(leader, d, q + (part * F::kOperand + s / 4 * 16384 + s % 4 * 32) / 16, k + (s / 4 * 16384 + s % 4 * 32) / 16, f16_idesc(kKeys),
                   part != kParts - 1 || s != 0);
        umma::commit_one(leader, bar(kSFull + r));
      };
      if (tiles > 0) {
        wait(kKFull, 0);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        scores(0, 0);
        scores(0, 1);
        umma::commit_one(leader, bar(kKEmpty));
      }
      for (int j = 0; j < tiles; ++j) {
        const uint32_t buf = j % kBufs;
        for (uint32_t r = 0; r < 2; ++r) {
          wait(kPReady + r, j);
          if (r == 0) wait(kVFull + buf, j / kBufs);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t v = desc_low(base + F::kV + buf * F::kOperand);
#pragma unroll
          for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
            for (int s = 0; s < kKeys / 16; ++s)
              mma_ts(leader, tmem + 256 + r * 128, tmem + r * 128 + s * 16 + part * 8, v + (s / 4 * (D * 128) + s % 4 * 32) / 16, f16_idesc(D),
                     part != kParts - 1 || s != 0);
          umma::commit_one(leader, bar(kOFull + r));
          if (r == 1) umma::commit_one(leader, bar(kVEmpty + buf));
          if (j + 1 < tiles) {
            if (r == 0) {
              wait(kKFull + (j + 1) % kBufs, (j + 1) / kBufs);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            scores(j + 1, r);
            if (r == 1) umma::commit_one(leader, bar(kKEmpty + (j + 1) % kBufs));
          }
        }
      }
    } else if (warp == 13) {
      // ---- copies --------------------------------------------------------------------------------------
      const uint32_t P = p.a.cache.page_tokens, block_bytes = static_cast<uint32_t>(cache_block_bytes(P, D));
      const int* const pages = p.a.batch.pages + static_cast<size_t>(seq) * p.a.batch.width;
      const auto page_of = [&](int key) -> uint32_t {
        const uint32_t index = static_cast<uint32_t>(key) >> p.page_shift;
        return key <= key_last && index < p.a.batch.width ? static_cast<uint32_t>(__ldg(pages + index)) : 0xFFFFFFFFu;
      };
      const auto copy = [&](uint32_t to, const uint8_t* from, uint32_t bytes, int i) {
        asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar(i)) : "memory");
      };
      uint32_t page_k = 0, page_v = 0;
      bool ok = true;
      const auto look = [&](int j) {  // lane i < 8: sixteen keys and their scales; lane i < 16: eight values
        page_k = page_v = 0xFFFFFFFFu;
        if (j < tiles) {
          if (lane < 8) page_k = page_of((tile0 + j) * kKeys + static_cast<int>(lane) * 16);
          if (lane < 16) page_v = page_of((tile0 + j) * kKeys + static_cast<int>(lane) * 8);
        }
      };
      look(0);
      for (int j = 0; j < tiles; ++j) {
        const int first = (tile0 + j) * kKeys, key_k = first + static_cast<int>(lane) * 16, key_v = first + static_cast<int>(lane) * 8;
        const bool have_k = page_k < p.a.cache.pages, have_v = page_v < p.a.cache.pages;
        const uint8_t* const block_k = p.a.cache.pool + (static_cast<uint64_t>(page_k) * heads + head) * block_bytes;
        const uint8_t* const block_v = p.a.cache.pool + (static_cast<uint64_t>(page_v) * heads + head) * block_bytes;
        look(j + 1);
        if (j > 0) ok = wait(kRawKFree, j - 1) && ok;
        ok = __all_sync(0xffffffffu, ok);
        const uint32_t n_k = __popc(__ballot_sync(0xffffffffu, have_k)), n_v = __popc(__ballot_sync(0xffffffffu, have_v));
        if (lane < 8 && !have_k && key_k <= key_last) {  // no such page: what it would hold is NaN
          uint32_t* params = reinterpret_cast<uint32_t*>(smem + F::kRawParams) + lane * 16;
          for (int i = 0; i < 16; ++i) params[i] = params[kKeys + i] = 0x7E007E00u;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (!ok) break;  // a wait gave up: nothing more is copied
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(kRawKFull)), "r"(n_k * 16 * (D / 2 + 8)) : "memory");
        __syncwarp();
        if (have_k) {
          const uint32_t slot = static_cast<uint32_t>(key_k) & (P - 1);
          copy(base + F::kRawK + lane * 16 * (D / 2), block_k + slot * (D / 2), 16 * (D / 2), kRawKFull);
          copy(base + F::kRawParams + lane * 64, block_k + P * D + slot * 4, 64, kRawKFull);
          copy(base + F::kRawParams + kKeys * 4 + lane * 64, block_k + P * D + (P + slot) * 4, 64, kRawKFull);
        }
        if (j > 0) ok = wait(kRawVFree, j - 1) && ok;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(kRawVFull)), "r"(n_v * 4 * D) : "memory");
        __syncwarp();
        if (have_v) copy(base + F::kRawV + lane * F::kGroup, block_v + (P + (static_cast<uint32_t>(key_v) & (P - 1))) * (D / 2), 4 * D, kRawVFull);
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (warp == 12) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <typename T, int D>
cudaError_t many_as(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond) {
  using F = Many<T, D>;
  static_assert(F::kSmem <= 227 * 1024 && F::kTable % 16 == 0 && F::kRows % 16 == 0 && F::kLost % 16 == 0 && F::kBars % 8 == 0 && F::kRawParams % 16 == 0,
                "shared memory and the alignment of its arrays");
  static OncePerDevice once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(attend_many_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem); });
  if (e != cudaSuccess) return e;
  ManyParams p;
  p.a = a;
  p.group = a.heads / a.cache.kv_heads;
  p.page_shift = 0;
  while ((1u << p.page_shift) < a.cache.page_tokens) ++p.page_shift;
  p.beyond = beyond;
  p.status = env.status;
  // at most so many blocks of rows: full ones, and one begun for each sequence
  const uint64_t rows = static_cast<uint64_t>(a.batch.tokens) * p.group;
  const uint64_t blocks = rows / kBlock + std::min<uint64_t>(a.batch.sequences, rows / (beyond + 1));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks * a.cache.kv_heads));
  cfg.blockDim = dim3(kManyThreads);
  cfg.dynamicSmemBytes = F::kSmem;
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attend_many_kernel<T, D>, p);
}

template <typename T>
cudaError_t many_of(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond) {
  return a.cache.head_dim == 64 ? many_as<T, 64>(env, a, beyond) : many_as<T, 128>(env, a, beyond);
}

}  // namespace

bool attend_many_supports(const AttendArgs& a) { return a.cache.head_dim <= 128; }

cudaError_t launch_attend_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond) {
  if (a.dtype == KQ_F32) return many_of<float>(env, a, beyond);
  if (a.dtype == KQ_F16) return many_of<__half>(env, a, beyond);
  return many_of<__nv_bfloat16>(env, a, beyond);
}

}  // namespace kq
