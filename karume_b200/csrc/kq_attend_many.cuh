// Attention over the paged 4-bit cache (layout in kq_cache.cuh) for many query rows a sequence: prompts, on the tcgen05
// tensor cores.
//
//   out = sum_j softmax_j(scale q . k_j) v_j,   k_j = u_j s_j + o_j, v_j likewise, codes u in 0..15
//
// A CTA takes 256 (f32: 128) query rows, (query, head of one kv head's group) packed: all heads of the group share what is
// unpacked.  It walks over the keys they see in tiles of 128.  Warps:
//   0-7    softmax: scores from tensor memory, weights back into it (over the scores)
//   8-13   unpack a tile: keys as [token][dim], values transposed as [dim][token], both K-major, 128-byte swizzle
//   14     issues the MMAs:   S = Q K^T (both in shared memory),   O = P V (P in tensor memory)
//   15     copies the codes and scales of the next tiles (bulk copies, page by page)
// 16-bit: two blocks of 128 rows, a thread a row; while one block's weights are computed the tensor core works for the other;
// O is added up in tensor memory, where the tensor core cuts it at its last bit at every sixteen keys: with values of one sign 6e-9 of
// a sum a key (8e-4 at 131072 keys walked by one CTA, 5e-5 where blocks of rows are so few that CTAs share the keys).
// f32: one block, two threads a row (half of the keys each, then half of the dims); the next tile's scores are made meanwhile;
// O is one tile's, added in registers, so that a long row does not drift.
// Few blocks of rows: the tiles of keys of each are shared by several CTAs, and the last one joins their sums in order.
//
// Measured: 4096 new tokens behind 904, 32 heads over 8, bfloat16: 291 us (682 TFLOP/s; with a lane's rows of queries one after the other instead of
// step by step 299; tensor pipe 33 %, issue slots 52 %).  At 305 us of it a tile
// of 256 rows is 2.6 us of a CTA (the MMAs 1.1): the turn from scores to weights and back, neither the unpacking (left out: 292 of 305 us)
// nor the exponentials (left out: 307) alone; a CTA's beginning and end were 21 us (rows found 1.8, queries 7.2, the first
// tile's way 4, output 5.9 (2.4 since it leaves in whole rows: 305 -> 293 us), the next CTA's start 1.8), three to four times an SM; the last CTAs end 27 us after the mean one.
// Three f32 prompts of up to 777 tokens behind 724, 12 heads over 2: 65 us, two products for one (queries and weights have two parts).
//
//   16-bit queries  keys and values are unpacked to what they stand for, rounded to binary16 once (2^-11, as the weights); rows beyond
//                   binary16's range to a sixteenth of it, which scores and weights make up for.
//   f32 queries     codes enter exactly, around zero: (2 u - 15) 2^-24 and (u - 7.5) 2^-20, one operation from the subnormals that
//                   their bits already are; scale and offset are applied to the scores and weights in f32.  Queries and weights are
//                   two binary16 parts each (fixed-point: sums of high parts are exact), 22 bits and more.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kq_cache.cuh"
#include "kq_umma.cuh"

namespace kq {
namespace {

constexpr int kKeys = 128;    // of a tile
constexpr int kManyTimeout = 50;

enum Bar { kRawKFull, kRawKFree = 2, kRawVFull = 4, kRawVFree = 6, kKFull = 8, kKEmpty = 10, kVFull = 12, kVEmpty = 14, kSFull = 16, kPReady = 18, kOFull = 20, kLoaded = 21, kAllDone = 22, kBarCount = 23 };

template <typename T, int D>
struct Many {
  static constexpr bool kSplit = sizeof(T) == 4;
  static constexpr int kParts = kSplit ? 2 : 1;
  // Query rows of a CTA.  16-bit: two blocks of 128, a softmax thread a row, the blocks taking turns; f32: one block, two threads a
  // row (half of the keys, then of the dims each: scores and sums stay in registers), the tiles of keys taking turns.
  static constexpr int kBlock = kSplit ? 128 : 256;
  static constexpr int kUnpackWarps = 6, kUnpack = kUnpackWarps * 32;
  static constexpr int kMmaWarp = 8 + kUnpackWarps, kCopyWarp = kMmaWarp + 1;
  static constexpr int kThreads = (kCopyWarp + 1) * 32;
  static constexpr int kAtOnce = 32;                       // 16-bit: scores a softmax thread has in hand
  static constexpr int kOperand = 128 * D * 2;             // bytes of 128 rows (or tokens) of D values
  // Unpacked tiles (16-bit: keys are needed only while scores are made) and tiles of codes on their way, as many as fit
  static constexpr int kKBufs = kSplit ? 2 : 1, kVBufs = 2, kRaws = kSplit && D == 128 ? 1 : 2;
  static constexpr int kGroup = 4 * D + 16;                // raw values of eight tokens, 16 bytes apart: lanes of eight groups meet no bank twice
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + 2 * kOperand;              // two blocks, or the two parts of one
  static constexpr int kV = kK + kKBufs * kOperand;
  static constexpr int kRaw = kV + kVBufs * kOperand;
  static constexpr int kRawV = kKeys * (D / 2);            // in a tile of codes: keys, values,
  static constexpr int kRawParams = kRawV + 16 * kGroup;   // keys' and values' (scale, offset)
  static constexpr int kRawBytes = kRawParams + 2 * kKeys * 4;
  // [2] x 16-bit: [2][128] (scale, offset) of keys and values; f32: [4][128] scale and centre of keys, then of values (2^13 scale)
  static constexpr int kTable = kRaw + kRaws * kRawBytes;
  static constexpr int kTableBytes = (kSplit ? 4 : 2) * kKeys * 4;
  static constexpr int kRows = kTable + 2 * kTableBytes;   // [kBlock] (factor, sum, last key, first key)
  // [2][3] 128 bits: values that are not finite, or stand for sixteen times what was unpacked; which of these are the latter; keys that are
  static constexpr int kRare = kRows + kBlock * 16;
  static constexpr int kBinade = kRare + 96;               // [2][4]: f32: the largest of 32 values' scales (2^13 scale)
  static constexpr int kHalves = kBinade + 32;             // f32: [2][2][128] (largest score, largest scale) of each half of a row's keys
  static constexpr int kBars = kHalves + (kSplit ? 2 * 2 * 128 * 8 : 0);
  static constexpr int kMisc = kBars + kBarCount * 8;
  static constexpr int kPartFloats = kBlock * (D + 2);
  static constexpr int kUnits = 512;                       // more than these are not shared by CTAs
  static constexpr int kSmem = kMisc + 96 + 1024;          // the operands start on a multiple of 1024
};

struct ManyParams {
  AttendArgs a;
  uint32_t group, page_shift, beyond;  // sequences of more than `beyond` query rows a kv head are this kernel's
  int* status;
  float* parts;            // null: a CTA walks over all keys of its rows.  Else [CTAs][kPartFloats]: sums, then (M, l) of each row
  unsigned int* counters;  // [units], zero between launches
  uint32_t ctas;           // that share the keys' tiles evenly
  bool prefix;             // kGroups: the keys that groups of sequences have in common, else the sequences' own
  SharedArgs sh;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// a whole number that is more than log2 of a scale (of binary16: no smaller than 2^-24)
__device__ __forceinline__ float binade_of(float scale) { return static_cast<float>(max(static_cast<int>(__float_as_uint(scale) >> 23) - 126, -24)); }
// two f32 operations as one
__device__ __forceinline__ uint64_t bits2(float2 v) { return *reinterpret_cast<const uint64_t*>(&v); }
__device__ __forceinline__ float2 float2_of(uint64_t v) { return *reinterpret_cast<const float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return float2_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return float2_of(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return float2_of(r);
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
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
// ... and any number of them
template <int N>
__device__ __forceinline__ void tmem_ld_begin(uint32_t taddr, float (&f)[N]) {
  if constexpr (N == 16) {
    tmem_ld16_begin(taddr, f);
  } else {
    static_assert(N == 32, "columns at a time");
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
  }
}
template <int N>
__device__ __forceinline__ void tmem_ld_done(float (&f)[N]) {
  if constexpr (N == 16) {
    tmem_ld16_done(f);
  } else {
    uint32_t* v = reinterpret_cast<uint32_t*>(f);
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) : : "memory");
    asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
  }
}
// N columns, sixteen at a time: use(column, values), the next ones on their way meanwhile.  kFlat: unrolled, so that the
// column is a constant (registers are indexed with it); otherwise a loop, for the instruction cache.
template <int N, bool kFlat, typename Use>
__device__ __forceinline__ void tmem_columns(uint32_t taddr, Use use) {
  float x[2][16];
  tmem_ld16_begin(taddr, x[0]);
#pragma unroll(kFlat ? N / 32 : 1)
  for (int c = 0; c < N; c += 32) {
    tmem_ld16_done(x[0]);
    tmem_ld16_begin(taddr + c + 16, x[1]);
    use(c, x[0]);
    tmem_ld16_done(x[1]);
    if (c + 32 < N) tmem_ld16_begin(taddr + c + 32, x[0]);
    use(c + 16, x[1]);
  }
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// The thread's lane of n columns times `keep`: weights (two binary16 a column) or sums.  Seldom run: a call, so that the loop
// around it keeps its registers.
template <bool kHalves>
__device__ __noinline__ void scale_columns(uint32_t taddr, int n, float keep) {
  const __half2 keep2 = __float2half2_rn(keep);
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");  // the weights of the keys in front may still be on their way there
  for (int at = 0; at < n; at += 16) {
    float w[16];
    tmem_ld16_begin(taddr + at, w);
    tmem_ld16_done(w);
    uint32_t y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&w[i]), keep2);
      y[i] = kHalves ? *reinterpret_cast<const uint32_t*>(&h) : __float_as_uint(w[i] * keep);
    }
    tmem_st8(taddr + at, y);
    tmem_st8(taddr + at + 8, y + 8);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// The thread's lane: scores (f32, a key a column) or weights (binary16, sixteen keys in eight columns of every sixteen) of the keys
// in `keys` sixteen times as large.  Seldom run, as above.
template <bool kHalves>
__device__ __noinline__ void sixteenfold(uint32_t taddr, const uint32_t* keys) {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  for (int at = 0; at < kKeys; at += 16) {
    const uint32_t of = keys[at / 32] >> (at % 32);
    float w[16];
    tmem_ld16_begin(taddr + at, w);
    tmem_ld16_done(w);
    uint32_t y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t two = of >> (2 * i % 16);
      const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&w[i]), __floats2half2_rn(two & 1 ? 16.0f : 1.0f, two & 2 ? 16.0f : 1.0f));
      y[i] = kHalves ? *reinterpret_cast<const uint32_t*>(&h) : __float_as_uint(of >> i & 1 ? w[i] * 16.0f : w[i]);
    }
    tmem_st8(taddr + at, y);
    if constexpr (!kHalves) tmem_st8(taddr + at + 8, y + 8);
  }
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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

__device__ __forceinline__ void load2(const float* p, float& a, float& b) {
  const float2 v = *reinterpret_cast<const float2*>(p);
  a = v.x;
  b = v.y;
}
template <typename T>
__device__ __forceinline__ void load2(const T* p, float& a, float& b) {
  const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
  a = to_f32(reinterpret_cast<const T*>(&v)[0]);
  b = to_f32(reinterpret_cast<const T*>(&v)[1]);
}
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

// kGroups: prefix: a "sequence" is a group of them, its rows all their new ones, its keys those in common, read through one member's
// pages; the sums go to `sh`.  Rest: the keys behind those, joined with the sums.
template <typename T, int D, bool kGroups>
__global__ void __launch_bounds__(Many<T, D>::kThreads, 1) attend_many_kernel(const __grid_constant__ ManyParams p) {
  using F = Many<T, D>;
  constexpr int kParts = F::kParts, kBlock = F::kBlock, kKBufs = F::kKBufs, kVBufs = F::kVBufs, kRaws = F::kRaws;
  constexpr bool kSplit = F::kSplit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + (1024 - (static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw)) & 1023u)) % 1024;
  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  float4* const rows = reinterpret_cast<float4*>(smem + F::kRows);
  uint32_t* const tmem_word = reinterpret_cast<uint32_t*>(smem + F::kMisc + 16);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + F::kMisc + 20);
  uint32_t* const found = reinterpret_cast<uint32_t*>(smem + F::kMisc + 24);  // sequence, number in it, part, parts, unit
  const auto bar = [&](int i) { return base + F::kBars + i * 8; };
  const auto wait = [&](int i, uint32_t parity) {
    const bool ok = umma::wait_bounded(bar(i), parity & 1u, abort_flag, p.status, kManyTimeout);
    __syncwarp();  // what follows is often an aligned instruction
    return ok;
  };
  // Each lane has fenced what it did.  f32: one arrival for the warp, since 32 on one word take their turns (three prompts: 75 -> 67 us);
  // 16-bit, whose warps have longer to the next barrier: each lane its own (4096 new tokens: 293 us, with one 297).
  constexpr uint32_t kArrivals = kSplit ? 1 : 32;  // of a warp
  const auto arrive = [&](int i) {
    if constexpr (kSplit) {
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(bar(i));
    } else {
      umma::mbar_arrive(bar(i));
    }
  };

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(bar(kKFull + i), F::kUnpackWarps * kArrivals);
      umma::mbar_init(bar(kKEmpty + i), 1);
      umma::mbar_init(bar(kRawKFull + i), 1);
      umma::mbar_init(bar(kRawVFull + i), 1);
      umma::mbar_init(bar(kRawKFree + i), F::kUnpackWarps * kArrivals);
      umma::mbar_init(bar(kRawVFree + i), F::kUnpackWarps * kArrivals);
      umma::mbar_init(bar(kVFull + i), F::kUnpackWarps * kArrivals);
      umma::mbar_init(bar(kVEmpty + i), 1);
      umma::mbar_init(bar(kSFull + i), 1);
      umma::mbar_init(bar(kOFull + i), kSplit && i == 1 ? 8 * kArrivals : 1);  // f32: one O; the second is kLoaded
      umma::mbar_init(bar(kPReady + i), (kSplit ? 8 : 4) * kArrivals);
    }
    umma::mbar_init(bar(kAllDone), 1);
    *abort_flag = 0;
    found[0] = 0xFFFFFFFFu;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait_prior_grid();
  __syncthreads();

  // ---- which rows: units are (sequence, block of rows from the last, kv head) ----------------------
  const bool prefix = kGroups && p.prefix, sharing = kGroups && worth_sharing(p.a, p.sh);
  if (prefix && !sharing) return;
  const uint32_t sequences = prefix ? p.sh.groups : p.a.batch.sequences, each = (sequences + F::kThreads - 1) / F::kThreads, heads = p.a.cache.kv_heads;
  int4* const groups = reinterpret_cast<int4*>(smem + F::kRaw);  // until the codes come
  int* const leads = reinterpret_cast<int*>(groups + groups::kAtOnce);
  static_assert(groups::kAtOnce * 20 <= F::kRawBytes, "the groups' place");
  if (prefix) {
    for (uint32_t g = warp; g < sequences; g += F::kThreads / 32) {
      int2 every, lead;
      const int4 of = group_of_rows(p.a.batch, p.sh, g, static_cast<int>(min(p.a.window, 0x7fffffffu)), every, lead);
      if (lane == 0) {
        groups[g] = of;
        leads[g] = lead.x;
        if (blockIdx.x == 0) p.sh.keys[g] = lead.y;
      }
    }
    __syncthreads();
  }
  const auto rows_of = [&](uint32_t b) {
    if (prefix) return Span{groups[b].x, groups[b].y, groups[b].z};
    return span_of(p.a.batch, b);
  };
  const auto blocks_of = [&](uint32_t b) {
    const Span s = rows_of(b);
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
  uint32_t* const scan = reinterpret_cast<uint32_t*>(smem + F::kRows);
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  uint32_t units = 0;
  for (uint32_t i = 0; i < F::kThreads / 32; ++i) {
    if (i < warp) upto += scan[i];
    units += scan[i];
  }
  const int window = static_cast<int>(min(p.a.window, 0x7fffffffu));
  // the tiles of a unit: first and number
  const auto tiles_of = [&](uint32_t b, uint32_t number) {
    const Span s = rows_of(b);
    if (prefix) return make_int2(groups[b].w / kKeys, (s.length - 1) / kKeys + 1 - groups[b].w / kKeys);
    const int block = static_cast<int>(blocks_of(b) - 1 - number / heads), n = s.count * static_cast<int>(p.group);
    const int first = block * kBlock / static_cast<int>(p.group), last = min(block * kBlock + kBlock - 1, n - 1) / static_cast<int>(p.group);
    const int key_last = s.length - s.count + last, from = s.length - s.count + first + 1 - window;
    int tile0 = window && from > 0 ? from / kKeys : 0;
    if constexpr (kGroups) {
      if (sharing) tile0 = max(tile0, common_keys(p.a.batch, p.sh, b, s) / kKeys);
      if (key_last / kKeys < tile0) return make_int2(tile0, 0);
    }
    return make_int2(tile0, key_last < 0 ? 0 : key_last / kKeys + 1 - tile0);
  };
  if (!p.parts) {
    if (upto - mine <= blockIdx.x && blockIdx.x < upto) {
      uint32_t b = tid * each, left = blockIdx.x - (upto - mine);
      for (uint32_t n = blocks_of(b) * heads; left >= n; n = blocks_of(++b) * heads) left -= n;
      found[0] = b;
      found[1] = left;
      found[3] = 1;
    }
  } else if (units > 0) {  // parts of units, as many as make the CTAs' shares even
    uint32_t* const of = reinterpret_cast<uint32_t*>(smem);  // sequence and number of each unit
    uint32_t at = upto - mine;
    for (uint32_t b = tid * each; b < min((tid + 1) * each, sequences); ++b)
      for (uint32_t n = blocks_of(b) * heads, i = 0; i < n; ++i, ++at)
        if (at < F::kUnits) {
          of[2 * at] = b;
          of[2 * at + 1] = i;
        }
    __syncthreads();
    const int mine_tiles = tid < units ? tiles_of(of[2 * tid], of[2 * tid + 1]).y : 0;
    const uint32_t warp_tiles = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(min(mine_tiles, 1 << 22)));
    __syncthreads();
    if (lane == 0) scan[warp] = warp_tiles;
    __syncthreads();
    uint32_t all = 0;
    for (uint32_t i = 0; i < F::kThreads / 32; ++i) all += scan[i];
    // about the smallest share of tiles with which the parts are one wave of CTAs; more units than CTAs stay whole
    int share = units > p.ctas ? 1 << 24 : max(static_cast<int>((all + p.ctas - 1) / p.ctas), 2);
    uint32_t n_parts = 0;
    for (;; share += share / 16 + 1) {
      n_parts = tid < units ? min(static_cast<uint32_t>(max((mine_tiles + share - 1) / share, 1)), p.ctas + 1) : 0u;
      const bool more = __syncthreads_or(n_parts > 1);
      const uint32_t warp_parts = __reduce_add_sync(0xffffffffu, n_parts);
      if (lane == 0) scan[warp] = warp_parts;
      __syncthreads();
      uint32_t sum = 0;
      for (int i = 0; i < F::kThreads / 32; ++i) sum += scan[i];
      __syncthreads();
      if (sum <= p.ctas || !more) break;
    }
    uint32_t to = n_parts;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= static_cast<uint32_t>(o)) to += v;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = to;
    __syncthreads();
    for (uint32_t i = 0; i < warp; ++i) to += scan[i];
    if (to - n_parts <= blockIdx.x && blockIdx.x < to) {
      found[0] = of[2 * tid];
      found[1] = of[2 * tid + 1];
      found[2] = blockIdx.x - (to - n_parts);
      found[3] = n_parts;
      found[4] = tid;
    }
  }
  __syncthreads();
  const uint32_t seq = found[0];
  if (seq == 0xFFFFFFFFu) return;
  const Span span = rows_of(seq);
  const uint32_t read_through = prefix ? static_cast<uint32_t>(leads[seq]) : seq;  // whose row of the page table
  const int common = kGroups && !prefix && sharing ? common_keys(p.a.batch, p.sh, seq, span) : 0;
  const uint32_t blocks = blocks_of(seq), head = found[1] % heads, block = blocks - 1 - found[1] / heads;  // the longest first
  const uint32_t all_parts = found[3], my_part = all_parts > 1 ? found[2] : 0;
  const int row0 = static_cast<int>(block * kBlock), n_rows = span.count * static_cast<int>(p.group), before = span.length - span.count;
  const int key_last = prefix ? span.length - 1 : before + min(row0 + kBlock - 1, n_rows - 1) / static_cast<int>(p.group);
  const int2 walk = tiles_of(seq, found[1]);
  const int part_from = static_cast<int>(static_cast<int64_t>(walk.y) * my_part / all_parts), part_to = static_cast<int>(static_cast<int64_t>(walk.y) * (my_part + 1) / all_parts);
  const int tile0 = walk.x + part_from, tiles = part_to - part_from;
  __syncthreads();  // `scan` and the units' list lie where the queries go

  // ---- queries --------------------------------------------------------------------------------------
  // kGroups: the copying warp is on its way to the first tiles meanwhile; the others meet without it.
  constexpr uint32_t kAskers = kGroups ? F::kCopyWarp : F::kThreads / 32;
  const bool asks = !kGroups || warp != F::kCopyWarp;
  const auto meet = [&] {
    if constexpr (!kGroups) __syncthreads();
    else if (asks) asm volatile("bar.sync 4, %0;" ::"n"(F::kCopyWarp * 32) : "memory");
  };
  const int q_of_row0 = row0 / static_cast<int>(p.group), head_of_row0 = row0 - q_of_row0 * static_cast<int>(p.group);
  const float inv_group = 1.0f / static_cast<float>(p.group);
  // query and head of row row0 + r: numbers below 2^17, so that the rounded-down product with the reciprocal is the quotient
  const auto query_and_head = [&](int r) {
    const int q = static_cast<int>((static_cast<float>(r + head_of_row0) + 0.5f) * inv_group);
    return make_int2(q_of_row0 + q, r + head_of_row0 - q * static_cast<int>(p.group));
  };
  // Groups: where each row of the block is, looked up by a thread each (by the lanes that load a row it took 6 of 14 us)
  if (prefix) {
    for (uint32_t r = tid; r < kBlock; r += F::kThreads) {
      const int2 qh = query_and_head(min(static_cast<int>(r), n_rows - 1 - row0));
      const int2 place = place_of_row(p.a.batch, static_cast<uint32_t>(span.first + qh.x));
      rows[r] = make_float4(__int_as_float(place.x), __int_as_float(place.y), 0.0f, 0.0f);
    }
    static_assert(!kGroups || kBlock <= F::kCopyWarp * 32, "rows of the warps that meet");
    meet();
  }
  const auto position_of = [&](uint32_t r, int query) {
    if (prefix) return __float_as_int(rows[r].x);
    return before + query;
  };
  const auto pointer_of = [&](int2 qh) {
    return static_cast<const T*>(p.a.q) + static_cast<size_t>(span.first + qh.x) * p.a.q_stride + (head * p.group + static_cast<uint32_t>(qh.y)) * D;
  };
  // a row is lifted to just below 2^14
  const auto lift_of = [](float big) {
    const int e = static_cast<int>(__float_as_uint(big) >> 23);
    return big > 0.0f && e < 255 ? min(max(140 - e, -100), 100) : 0;
  };
  const auto power = [](int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); };  // |e| up to 126
  // f32: fixed-point parts; odd dims meet codes eight times as large
  const auto parts_of = [](float x, bool odd, float& hi, float& lo) {
    constexpr float kEight = 100663296.0f;  // 1.5 2^26: numbers beside it are multiples of eight
    const float top = __fsub_rn(__fadd_rn(x, kEight), kEight), down = odd ? 0.125f : 1.0f;
    hi = top * down;
    lo = __half2float(__float2half_rn((x - top) * down));
  };
  const auto row_constants = [&](uint32_t r, int up, float sum) {
    const float factor = p.a.scale * 1.4426950408889634f;
    const bool there = row0 + static_cast<int>(r) < n_rows;
    int last = there ? before + query_and_head(static_cast<int>(r)).x : 0x7fffffff;  // rows beyond the end see anything and are not stored
    int from = there && window && last + 1 > window ? last + 1 - window : 0;
    if constexpr (kGroups) {
      if (prefix && there) {
        const int position = __float_as_int(rows[r].x);
        last = min(__float_as_int(rows[r].y), span.length) - 1;
        from = window && position + 1 > window ? position + 1 - window : 0;
      } else if (there) {
        from = max(from, common);
      }
    }
    // f32: score = factor 2^(23 - up) (acc scale + centre sum 2^-23), the sum of the lifted parts as they are multiplied: a rounding
    // then weighs as much as the key, not as the code times its scale, which in a row with one large value is large everywhere
    rows[r] = kSplit ? make_float4(factor * power(23 - up), sum * power(-23), __int_as_float(last), __int_as_float(from))
                     : make_float4(factor * power(-up), 0.0f, __int_as_float(last), __int_as_float(from));
  };
  if (rope_is_plain(p.a.rope) && p.a.rope.rotary == D) {
    // Half layout, whole heads: a lane has two pairs of a row, so that the angles are read coalesced (runs of eight dims a lane read them
    // at a stride of 64 bytes, 9000 clocks a CTA); words of dims (d, d + 4) are put together with the lane two further on.
    constexpr uint32_t kLanes = D / 4, kRowsAtOnce = 32 / kLanes, kStep = kAskers * kRowsAtOnce, kEach = (kBlock + kStep - 1) / kStep;
    constexpr uint32_t kTurns = (kEach + 8) / 9, kBatch = (kEach + kTurns - 1) / kTurns;  // rows a lane has at a time
    static_assert(kBatch <= kLanes, "a lane for the constants of each row");
    const uint32_t c = lane % kLanes;
    const uint32_t word = (c & 1) * 2 + (c >> 1 & 1);  // of its eight dims' chunk: dims (0, 4), (1, 5), (2, 6), (3, 7) from lanes 0, 2, 1, 3
#pragma unroll 1
    for (uint32_t r0 = warp * kRowsAtOnce + lane / kLanes, turn = 0; asks && turn < kTurns; r0 += kStep * kBatch, ++turn) {
      float x[kBatch][4], big[kBatch], sum[kBatch];
      float4 cs[kBatch];
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) {
        const uint32_t r = min(r0 + k * kStep, static_cast<uint32_t>(kBlock) - 1);
        const int2 qh = query_and_head(min(static_cast<int>(r), n_rows - 1 - row0));
        const T* from_q = pointer_of(qh);
        const int position = position_of(r, qh.x);
        const bool inside = position >= 0 && static_cast<uint32_t>(position) < p.a.rope.positions;
        load2(from_q + 2 * c, x[k][0], x[k][1]);
        load2(from_q + D / 2 + 2 * c, x[k][2], x[k][3]);
        cs[k] = reinterpret_cast<const float4*>(p.a.rope.table + static_cast<size_t>(inside ? position : 0) * (D / 2))[c];
        if (!inside) cs[k].x = cs[k].z = quiet_nan();
      }
      // (step by step for all rows, so that one row's shuffles do not wait for another's)
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) {
        const bool there = row0 + static_cast<int>(r0 + k * kStep) < n_rows;
        const float2 a = rotate_pair(x[k][0], x[k][2], make_float2(cs[k].x, cs[k].y)), b = rotate_pair(x[k][1], x[k][3], make_float2(cs[k].z, cs[k].w));
        // dims 2 c, 2 c + 1, and those half a head on
        x[k][0] = there ? a.x : 0.0f;
        x[k][1] = there ? b.x : 0.0f;
        x[k][2] = there ? a.y : 0.0f;
        x[k][3] = there ? b.y : 0.0f;
        big[k] = fmaxf(fmaxf(fabsf(x[k][0]), fabsf(x[k][1])), fmaxf(fabsf(x[k][2]), fabsf(x[k][3])));
        sum[k] = 0.0f;
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2)
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) big[k] = fmaxf(big[k], __shfl_xor_sync(0xffffffffu, big[k], o));
      int my_up = 0;
      float my_sum = 0.0f;
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k) {
        const uint32_t r = r0 + k * kStep;
        const int up = lift_of(big[k]);
        const float lift = power(up);
        if (c == k) my_up = up;
        float hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kSplit) {
            parts_of(x[k][i] * lift, i & 1, hi[i], lo[i]);
            sum[k] = fmaf(hi[i] + lo[i], (i & 1) ? 8.0f : 1.0f, sum[k]);
          } else {
            hi[i] = x[k][i] * lift;
          }
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float* h = part ? lo : hi;
            const uint32_t mine2 = half2_bits(h[2 * half], h[2 * half + 1]), other2 = __shfl_xor_sync(0xffffffffu, mine2, 2);
            const uint32_t out = c & 2 ? __byte_perm(other2, mine2, 0x7632) : __byte_perm(mine2, other2, 0x5410);
            const uint32_t chunk = half * (D / 16) + c / 4;
            const uint32_t at = base + F::kQ + ((r / 128) * kParts + part) * F::kOperand + (chunk / 8) * 16384 + umma::swz(r % 128, chunk % 8) + word * 4;
            if (kBlock % (kStep * kBatch) == 0 || r < kBlock) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(out) : "memory");
          }
      }
      if constexpr (kSplit) {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o /= 2)
#pragma unroll
          for (uint32_t k = 0; k < kBatch; ++k) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
          if (c == k) my_sum = sum[k];
      }
      if (c < kBatch && r0 + c * kStep < kBlock) row_constants(r0 + c * kStep, my_up, my_sum);
    }
  } else {
    constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes;
    const uint32_t c = lane % kLanes;
#pragma unroll 1
    for (uint32_t r = warp * kRowsAtOnce + lane / kLanes; asks && r - lane / kLanes < kBlock; r += kAskers * kRowsAtOnce) {
      const bool there = row0 + static_cast<int>(r) < n_rows;
      const int2 qh = query_and_head(min(static_cast<int>(r), n_rows - 1 - row0));
      float v[8], big = 0.0f, sum = 0.0f;
      load8_rotated(pointer_of(qh), c * 8, p.a.rope, position_of(r, qh.x), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = there ? v[i] : 0.0f;
        big = fmaxf(big, fabsf(v[i]));
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      const int up = lift_of(big);
      const float lift = power(up);
      float hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kSplit) {
          parts_of(v[i] * lift, i & 1, hi[i], lo[i]);
          sum = fmaf(hi[i] + lo[i], (i & 1) ? 8.0f : 1.0f, sum);
        } else {
          hi[i] = v[i] * lift;
        }
      }
      if constexpr (kSplit) {
#pragma unroll
        for (int o = kLanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      }
      const uint32_t at = base + F::kQ + (r / 128) * kParts * F::kOperand + (c / 8) * 16384 + umma::swz(r % 128, c % 8);
      umma::sts128(at, make_uint4(half2_bits(hi[0], hi[4]), half2_bits(hi[1], hi[5]), half2_bits(hi[2], hi[6]), half2_bits(hi[3], hi[7])));
      if constexpr (kSplit)
        umma::sts128(at + F::kOperand, make_uint4(half2_bits(lo[0], lo[4]), half2_bits(lo[1], lo[5]), half2_bits(lo[2], lo[6]), half2_bits(lo[3], lo[7])));
      if (c == 0) row_constants(r, up, sum);
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (warp == F::kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(tmem_word))), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  meet();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = asks ? *tmem_word : 0;

  if (warp < 8) {
    // ---- softmax and output: a row a thread --------------------------------------------------------
    if constexpr (kSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const uint32_t wg = warp / 4, lanes = (warp % 4 * 32) << 16;
    const int r = static_cast<int>(kSplit ? tid % 128 : tid);
    const float4 rc = rows[r];
    const float factor = rc.x, q_sum = rc.y;
    const int last = __float_as_int(rc.z), from = __float_as_int(rc.w);
    const int last_all = __reduce_min_sync(0xffffffffu, last), from_all = __reduce_max_sync(0xffffffffu, from);
    // Weights are 2^(score - M + lift).  M is a whole number (what it moves by is an exact power of two) that follows the row's
    // largest score, f32: and the binade of the values' scales beside it; it moves when a weight (times its value's scale)
    // would pass 2^14.  f32 lets M lag by one bit, to keep the fixed-point parts' 22; 16-bit by eight.
    float M = -INFINITY, l = 0.0f, centre = 0.0f;
    float O[kSplit ? D / 2 : 1];
    if constexpr (kSplit) {
      // ---- f32: this thread's keys and dims are half wg of the tile's and of the head's -----------------------------
#pragma unroll
      for (int i = 0; i < D / 2; ++i) O[i] = 0.0f;
      float2* const halves = reinterpret_cast<float2*>(smem + F::kHalves);
      float keep_sums = 1.0f;  // what the tile before is still to be scaled by
      const auto drain = [&](int j, float keep) {
        wait(kOFull, j);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_columns<D / 2, true>(tmem + lanes + 384 + wg * (D / 2), [&](int c, float (&x)[16]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) O[c + i] = fmaf(x[i], keep, O[c + i]);
        });
      };
      for (int j = 0; j < tiles; ++j) {
        const int first = (tile0 + j) * kKeys + static_cast<int>(wg) * 64;
        const bool whole = first >= from_all && first + 63 <= last_all;
        const int sees0 = from - first, sees1 = last - first;  // of the thread's 64 columns those that the row sees
        const float* table = reinterpret_cast<const float*>(smem + F::kTable + (j & 1) * F::kTableBytes) + wg * 64;
        const uint32_t t_s = tmem + lanes + (j & 1) * 128 + wg * 64;
        wait(kSFull + (j & 1), j / 2);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float z[64];
#pragma unroll
        for (int c = 0; c < 64; c += 32) tmem_ld_begin(t_s + c, reinterpret_cast<float (&)[32]>(z[c]));
#pragma unroll
        for (int c = 0; c < 64; c += 32) tmem_ld_done(reinterpret_cast<float (&)[32]>(z[c]));
#pragma unroll
        for (int c = 0; c < 64; c += 32) {  // the low parts' share
          float low[32];
          tmem_ld_begin(tmem + lanes + 256 + wg * 64 + c, low);
          tmem_ld_done(low);
#pragma unroll
          for (int i = 0; i < 32; ++i) z[c + i] += low[i];
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        arrive(kLoaded);
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 k_scale = *reinterpret_cast<const float2*>(table + i), k_mid = *reinterpret_cast<const float2*>(table + kKeys + i);
          const float2 s = fma2(make_float2(z[i], z[i + 1]), k_scale, mul2(k_mid, make_float2(q_sum, q_sum)));
          z[i] = s.x;
          z[i + 1] = s.y;
        }
        float scale_seen = 0.0f;
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            if (i < sees0 || i > sees1) z[i] = -INFINITY;  // what is not seen may hold anything
            else scale_seen = fmaxf(scale_seen, table[2 * kKeys + i]);
          }
        } else {
          const float* bn = reinterpret_cast<const float*>(smem + F::kBinade) + (j & 1) * 4 + wg * 2;  // warps 2 wg, 2 wg + 1 made these keys' scales
          scale_seen = fmaxf(bn[0], bn[1]);
        }
        float big[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) big[i] = fmaxf(fmaxf(z[i], z[i + 16]), fmaxf(z[i + 32], z[i + 48]));
#pragma unroll
        for (int o = 8; o > 0; o /= 2)
#pragma unroll
          for (int i = 0; i < o; ++i) big[i] = fmaxf(big[i], big[i + o]);
        // the row's other half
        halves[((j & 1) * 2 + wg) * 128 + r] = make_float2(big[0], scale_seen);
        asm volatile("bar.sync 3, 256;" ::: "memory");
        const float2 other = halves[((j & 1) * 2 + (wg ^ 1)) * 128 + r];
        const float binade = binade_of(fmaxf(scale_seen, other.y) * (1.0f / 8192.0f));
        const float top = fmaxf(big[0], other.x) * factor + binade;
        const bool more = top > M + 1.0f;
        keep_sums = 1.0f;
        if (__any_sync(0xffffffffu, more)) {
          const float now = more ? ceilf(top) : M;
          keep_sums = M == -INFINITY ? 0.0f : exp2f(M - now);
          M = now;
          l *= keep_sums;
          centre *= keep_sums;
#pragma unroll
          for (int i = 0; i < D / 2; ++i) O[i] *= keep_sums;
        }
        const float shift = M == -INFINITY ? 0.0f : -M;  // the values' scales carry 2^13
        float2 part = {}, mid = {};
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 e = fma2(make_float2(z[c + i], z[c + i + 1]), make_float2(factor, factor), make_float2(shift, shift));
            const float2 w = make_float2(ex2(e.x), ex2(e.y));
            float2 v_scale = *reinterpret_cast<const float2*>(table + 2 * kKeys + c + i), v_mid = *reinterpret_cast<const float2*>(table + 3 * kKeys + c + i);
            if (!whole) {
              if (c + i < sees0 || c + i > sees1) v_scale.x = v_mid.x = 0.0f;
              if (c + i + 1 < sees0 || c + i + 1 > sees1) v_scale.y = v_mid.y = 0.0f;
            }
            part = add2(part, w);
            mid = fma2(w, v_mid, mid);
            const float2 y = mul2(w, v_scale);
            // the high part: whole numbers (their sums are exact) of eleven bits, so that small weights keep 22 bits too
            constexpr float kOne = 12582912.0f;  // 1.5 2^23: numbers beside it are whole
            float2 h = add2(add2(y, make_float2(kOne, kOne)), make_float2(-kOne, -kOne));
            h.x = __uint_as_float(__float_as_uint(h.x) & 0xFFFFE000u);
            h.y = __uint_as_float(__float_as_uint(h.y) & 0xFFFFE000u);
            const float2 low = fma2(h, make_float2(-1.0f, -1.0f), y);
            hi[i / 2] = half2_bits(h.x, h.y);
            lo[i / 2] = half2_bits(low.x, low.y);
          }
          // sixteen keys' weights go where their scores were: eight columns, and eight for the low parts
          tmem_st8(t_s + c, hi);
          tmem_st8(t_s + c + 8, lo);
        }
        l += part.x + part.y;
        centre += mid.x + mid.y;
        if (j > 0) drain(j - 1, keep_sums);  // before the next sums are made in the same columns
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        arrive(kPReady + (j & 1));
      }
      if (tiles > 0) drain(tiles - 1, 1.0f);
      // both halves' weights
      asm volatile("bar.sync 3, 256;" ::: "memory");
      halves[wg * 128 + r] = make_float2(l, centre);
      asm volatile("bar.sync 3, 256;" ::: "memory");
      const float2 first_half = halves[r], second_half = halves[128 + r];
      l = first_half.x + second_half.x;
      centre = first_half.y + second_half.y;
    } else {
      // ---- 16-bit: row r, all keys; the sums stay in tensor memory ------------------------------------------------
      // So that M's move is seen before anything is written, a few scores are looked at at a time; what was written of the tile before
      // is then scaled too.
      constexpr int kN = F::kAtOnce;
      // The largest weight is 2^(kLift + kLag), and sixteen times that stays below 2^16.
      constexpr float kLift = 3.0f, kLag = 8.0f;
      const uint32_t t_s = tmem + lanes + wg * 128, t_o = tmem + lanes + 256 + wg * 128;
      for (int j = 0; j < tiles; ++j) {
        const int first = (tile0 + j) * kKeys;
        const bool whole = first >= from_all && first + kKeys - 1 <= last_all;
        const int sees0 = from - first, sees1 = last - first;  // columns the row sees
        wait(kSFull + wg, j);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float limit = M + kLag, shift = M == -INFINITY ? kLift : kLift - M;
        const auto tile = [&](auto all_seen) {
          constexpr bool kAll = decltype(all_seen)::value;
          float x[2][kN];
          const auto some = [&](int c, float* z, auto begin_next) {
            float big[kN / 2];
#pragma unroll
            for (int i = 0; i < kN; ++i)
              if (!kAll && (c + i < sees0 || c + i > sees1)) z[i] = -INFINITY;  // what is not seen may hold anything
#pragma unroll
            for (int i = 0; i < kN / 2; ++i) big[i] = fmaxf(z[i], z[i + kN / 2]);
#pragma unroll
            for (int o = kN / 4; o > 0; o /= 2)
#pragma unroll
              for (int i = 0; i < o; ++i) big[i] = fmaxf(big[i], big[i + o]);
            const float top = big[0] * factor;
            if (__any_sync(0xffffffffu, top > limit)) {
              const float now = top > limit ? ceilf(top) : M;
              const float keep = M == -INFINITY ? 0.0f : exp2f(M - now);
              M = now;
              limit = M + kLag;
              shift = M == -INFINITY ? kLift : kLift - M;
              l *= keep;
              scale_columns<true>(t_s, c, keep);
              if (j > 0) {  // the sums of the tiles before
                wait(kOFull + wg, j - 1);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                scale_columns<false>(t_o, D, keep);
              }
            }
            begin_next();
            uint32_t w2[kN / 2];
            float part[4] = {};
#pragma unroll
            for (int i = 0; i < kN; i += 2) {
              const float w0 = ex2(fmaf(z[i], factor, shift)), w1 = ex2(fmaf(z[i + 1], factor, shift));
              part[i / 2 % 2 * 2] += w0;
              part[i / 2 % 2 * 2 + 1] += w1;
              w2[i / 2] = half2_bits(w0, w1);
            }
            l += (part[0] + part[1]) + (part[2] + part[3]);
            // sixteen keys' weights go where their scores were, into eight columns
#pragma unroll
            for (int i = 0; i < kN / 16; ++i) tmem_st8(t_s + c + i * 16, w2 + i * 8);
          };
          tmem_ld_begin(t_s, x[0]);
#pragma unroll 1
          for (int c = 0; c < kKeys; c += 2 * kN) {
            tmem_ld_done(x[0]);
            some(c, x[0], [&] { tmem_ld_begin(t_s + c + kN, x[1]); });
            tmem_ld_done(x[1]);
            some(c + kN, x[1], [&] {
              if (c + 2 * kN < kKeys) tmem_ld_begin(t_s + c + 2 * kN, x[0]);
            });
          }
        };
        const uint4 big = *reinterpret_cast<const uint4*>(smem + F::kRare + (j & 1) * 48 + 32);  // (this look and that at `rare`: 4096 new tokens 304 us, without them 300)
        if (big.x | big.y | big.z | big.w) sixteenfold<false>(t_s, reinterpret_cast<const uint32_t*>(smem + F::kRare + (j & 1) * 48 + 32));
        if (whole) tile(std::true_type());
        else tile(std::false_type());
        const uint4 rare = *reinterpret_cast<const uint4*>(smem + F::kRare + (j & 1) * 48);
        if (rare.x | rare.y | rare.z | rare.w) {
          const uint32_t* const bits = reinterpret_cast<const uint32_t*>(smem + F::kRare) + (j & 1) * 12;
          sixteenfold<true>(t_s, bits + 4);
          // values that are not finite entered as zeros: whoever sees one is NaN
          for (int i = max(sees0, 0); i <= min(sees1, kKeys - 1); ++i)
            if ((bits[i / 32] & ~bits[4 + i / 32]) >> (i % 32) & 1) l = quiet_nan();
          __syncwarp();
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        arrive(kPReady + wg);
      }
    }
    const int row = row0 + r;
    const auto out_of = [&](int row_of) {
      const int query = row_of / static_cast<int>(p.group);
      return static_cast<T*>(p.a.out) + static_cast<size_t>(span.first + query) * p.a.out_stride +
             static_cast<size_t>(head * p.group + static_cast<uint32_t>(row_of - query * static_cast<int>(p.group))) * D;
    };
    // read again: what was not needed in the loop takes no registers there
    const uint32_t n_parts = reinterpret_cast<volatile uint32_t*>(found)[3];
    const bool shared = n_parts > 1 || (kGroups && prefix && p.parts);  // sums over common keys stay in parts
    const float inv = shared || (kGroups && (prefix || common > 0)) ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    float* const part = shared ? p.parts + static_cast<size_t>(blockIdx.x) * F::kPartFloats : nullptr;
    // Of the sums in the scratch of row `row_of`, their place; and what a row's own weights count beside them: (own, theirs), divided by all.
    const auto sums_of = [&](int row_of) {
      const int query = row_of / static_cast<int>(p.group);
      return static_cast<size_t>(span.first + query) * p.a.heads + head * p.group + static_cast<uint32_t>(row_of - query * static_cast<int>(p.group));
    };
    constexpr float kLifted = kSplit ? 0.0f : 3.0f;  // 16-bit weights and sums are so many powers of two larger than M says
    // eight values of a row that is complete, with its M and sum of weights
    const auto finish = [&](int row_of, int i, float m, float total, const float* o) {
      if constexpr (kGroups) {
        const size_t of = sums_of(row_of);
        if (prefix) {
          const uint4 place = whole_place(p.sh, p.a, of);
          __stcg(reinterpret_cast<float4*>(p.sh.scratch) + place.x + i / 4, make_float4(o[0], o[1], o[2], o[3]));
          __stcg(reinterpret_cast<float4*>(p.sh.scratch) + place.x + i / 4 + 1, make_float4(o[4], o[5], o[6], o[7]));
          if (i == 0) {
            __stcg(reinterpret_cast<float2*>(p.sh.scratch) + place.y, make_float2(m - kLifted, total));
            __stcg(p.sh.places + of, place);
          }
          return;
        }
        if (common > 0) {
          const uint4 place = __ldcg(p.sh.places + of);
          float z[8];
#pragma unroll
          for (int half = 0; half < 8; half += 4) {
            float top = m - kLifted, all = total, v[4] = {o[half], o[half + 1], o[half + 2], o[half + 3]};
            join_common(p.sh, place, (i + half) / 4, top, all, v);
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
            for (int e = 0; e < 4; ++e) z[half + e] = v[e] * inv;
          }
          store8(out_of(row_of) + i, z);
          return;
        }
      }
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = o[e] * inv;
      store8(out_of(row_of) + i, z);
    };
    const bool apart = kGroups && (prefix || common > 0);  // rows are finished with sums in the scratch
    const auto store = [&](int i, const float* o) {
      if (shared) {
        store8(part + static_cast<size_t>(r) * D + i, o);
        return;
      }
      if constexpr (kGroups)
        if (apart && row < n_rows) {
          finish(row, i, M, l, o);
          return;
        }
      if (row < n_rows) store8(out_of(row) + i, o);
    };
    if constexpr (kSplit) {
#pragma unroll
      for (int i = 0; i < D / 2; i += 8) {
        float o[8];
        // powers of two: the weights' 2^13, the codes' even dims (2 u - 15) 2^-24, odd ones (u - 7.5) 2^-20
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = fmaf(O[i + k], (k & 1) ? 128.0f : 1024.0f, centre) * inv;
        store(static_cast<int>(wg) * (D / 2) + i, o);
      }
    } else if (tiles == 0) {
      const float zero[8] = {};
      for (int i = 0; i < D; i += 8) store(i, zero);
    } else {
      wait(kOFull + wg, tiles - 1);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // Rows go out whole, through the block's queries' memory, which every score has been made of by now: a thread's own row is 16
      // bytes of 32 rows an instruction.
      uint8_t* const mine = smem + F::kQ + wg * F::kOperand + warp % 4 * (32 * D * 2);
      if (kGroups && prefix && shared) {  // sums in f32: half of a row at a time
        constexpr uint32_t kChunks = D / 8, kAtOnce = 32 / kChunks;
        for (int half = 0; half < 2; ++half) {
          tmem_columns<D / 2, false>(tmem + lanes + 256 + wg * 128 + half * (D / 2), [&](int c, float (&x)[16]) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
              *reinterpret_cast<float4*>(mine + lane * (D * 2) + ((c / 4 + h) ^ (lane & 7)) * 16) = make_float4(x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]);
            __syncwarp();
          });
#pragma unroll 4
          for (uint32_t i = lane / kChunks; i < 32; i += kAtOnce) {
            const uint32_t chunk = lane % kChunks;
            *reinterpret_cast<float4*>(part + static_cast<size_t>(wg * 128 + warp % 4 * 32 + i) * D + half * (D / 2) + chunk * 4) =
                *reinterpret_cast<const float4*>(mine + i * (D * 2) + (chunk ^ (i & 7)) * 16);
          }
          __syncwarp();
        }
      } else
      tmem_columns<D, false>(tmem + lanes + 256 + wg * 128, [&](int c, float (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= inv;
        if (shared || apart) {
          store(c, x);
          store(c + 8, x + 8);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            store8(reinterpret_cast<T*>(mine + lane * (D * 2) + ((c / 8 + h) ^ (lane & 7)) * 16), x + 8 * h);
        }
        __syncwarp();
      });
      if (!shared && !apart) {
        constexpr uint32_t kChunks = D / 8, kAtOnce = 32 / kChunks;  // of a row; rows an instruction
#pragma unroll 4
        for (uint32_t i = lane / kChunks; i < 32; i += kAtOnce) {
          const uint32_t of = wg * 128 + warp % 4 * 32 + i, chunk = lane % kChunks;
          if (row0 + static_cast<int>(of) >= n_rows) break;
          const int2 qh = query_and_head(static_cast<int>(of));
          *reinterpret_cast<uint4*>(static_cast<T*>(p.a.out) + static_cast<size_t>(span.first + qh.x) * p.a.out_stride +
                                    static_cast<size_t>(head * p.group + static_cast<uint32_t>(qh.y)) * D + chunk * 8) =
              *reinterpret_cast<const uint4*>(mine + i * (D * 2) + (chunk ^ (i & 7)) * 16);
        }
        __syncwarp();
      }
    }
    if (shared) {  // the last CTA of the unit joins the parts, in order
      if (!kSplit || wg == 0) {
        if constexpr (kGroups) {
          if (prefix) {
            reinterpret_cast<float2*>(part + kBlock * D)[r] = make_float2(M - kLifted, l);
            const size_t at = static_cast<size_t>(p.parts - p.sh.scratch) + static_cast<size_t>(blockIdx.x) * F::kPartFloats;
            if (my_part == 0 && row < n_rows)
              __stcg(p.sh.places + sums_of(row), make_uint4(static_cast<uint32_t>(at / 4 + r * (D / 4)), static_cast<uint32_t>((at + kBlock * D) / 2 + r), F::kPartFloats, n_parts));
          }
        }
        if (!prefix) reinterpret_cast<float2*>(part + kBlock * D)[r] = make_float2(M, l);
      }
    }
    if (shared && !prefix) {
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (tid == 0) {
        unsigned int arrived;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(arrived) : "l"(p.counters + found[4]) : "memory");
        if (arrived == n_parts - 1) p.counters[found[4]] = 0;
        found[5] = arrived;
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (found[5] == n_parts - 1) {
        const float* const parts = p.parts + static_cast<size_t>(blockIdx.x - found[2]) * F::kPartFloats;
        for (int at = static_cast<int>(tid); at < kBlock * D / 8; at += 256) {
          const int of = at / (D / 8), i = at % (D / 8) * 8;
          if (row0 + of >= n_rows) break;
          float m = -INFINITY, total = 0.0f, o[8] = {};
          for (uint32_t k = 0; k < n_parts; ++k) m = fmaxf(m, __ldcg(parts + static_cast<size_t>(k) * F::kPartFloats + kBlock * D + 2 * of));
#pragma unroll 4
          for (uint32_t k = 0; k < n_parts; ++k) {
            const float* from_part = parts + static_cast<size_t>(k) * F::kPartFloats;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(from_part + kBlock * D) + of);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(from_part + static_cast<size_t>(of) * D + i)), y = __ldcg(reinterpret_cast<const float4*>(from_part + static_cast<size_t>(of) * D + i) + 1);
            const float keep = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
            const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            total = fmaf(keep, ml.y, total);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(keep, v[e], o[e]);
          }
          if constexpr (kGroups) {
            finish(row0 + of, i, m, total, o);
          } else {
            const float scale = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] *= scale;
            store8(out_of(row0 + of) + i, o);
          }
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  } else {
    if constexpr (kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp < F::kMmaWarp) {
      // ---- unpacking ---------------------------------------------------------------------------------
      const uint32_t t = tid - 256, w4 = warp - 8;
      constexpr uint32_t kExp = 0x64006400u, k1024 = 0xE400E400u, k16th = 0x2C002C00u, k64 = 0xD400D400u;  // 1024 | x, -1024, 1/16, -64
      constexpr uint32_t kCentre0 = 0x800F800Fu, kCentre1 = 0x80788078u;                                   // -15 2^-24, -7.5 2^-20
      bool ok = true;  // after a wait that gave up nothing is handed on: no barrier is arrived on beyond its phase
      for (int j = 0; j < tiles; ++j) {
        const int first = (tile0 + j) * kKeys;
        const uint32_t buf = j % kVBufs, kbuf = j % kKBufs, raw = j % kRaws;
        const uint8_t* const codes = smem + F::kRaw + raw * F::kRawBytes;
        uint32_t* const k_par = reinterpret_cast<uint32_t*>(smem + F::kTable + (j & 1) * F::kTableBytes);  // (scale, offset) of each key;
        __half* const v_scale = reinterpret_cast<__half*>(k_par + kKeys);                                  // values' scales, then offsets
        __half* const v_offset = v_scale + kKeys;
        ok = wait(kRawKFull + raw, j / kRaws) && ok;
        if (j >= 2) wait(kVEmpty + buf, j / 2 - 1);  // what the softmax warps read of tile j - 2 has been read
        if (t < kKeys) {
          const bool seen = first + static_cast<int>(t) <= key_last;
          const uint32_t* const raw_params = reinterpret_cast<const uint32_t*>(codes + F::kRawParams);
          uint32_t kp = seen ? raw_params[t] : 0u, vp = seen ? raw_params[kKeys + t] : 0u;
          const float2 k = __half22float2(*reinterpret_cast<const __half2*>(&kp)), v = __half22float2(*reinterpret_cast<const __half2*>(&vp));
          if constexpr (kSplit) {
            float* const table = reinterpret_cast<float*>(k_par) + t;
            table[0] = k.x;
            table[kKeys] = fmaf(7.5f, k.x, k.y);
            table[2 * kKeys] = v.x * 8192.0f;
            table[3 * kKeys] = fmaf(7.5f, v.x, v.y);
            const uint32_t big = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(v.x, 0.0f)));  // not NaN
            if (lane == 0) reinterpret_cast<float*>(smem + F::kBinade)[(j & 1) * 4 + w4] = __uint_as_float(big) * 8192.0f;
          } else {
            // A row stands for up to 16 * 65504.  Where that rounds to an infinity in binary16 (its scale is one at least then),
            // a sixteenth is unpacked, and the softmax warps put it right in the key's score or the value's weight.
            constexpr float kLargest = 65504.0f, kBeyond = 65520.0f;
            const bool not_finite = !(fabsf(v.x) <= kLargest && fabsf(v.y) <= kLargest);
            const bool k_big = fabsf(fmaf(15.0f, k.x, k.y)) >= kBeyond, v_big = !not_finite && fabsf(fmaf(15.0f, v.x, v.y)) >= kBeyond;
            const uint32_t lost = __ballot_sync(0xffffffffu, not_finite), big_keys = __ballot_sync(0xffffffffu, k_big), big_values = __ballot_sync(0xffffffffu, v_big);
            if (lane == 0) {
              uint32_t* const rare = reinterpret_cast<uint32_t*>(smem + F::kRare) + (j & 1) * 12 + w4;
              rare[0] = lost | big_values;
              rare[4] = big_values;
              rare[8] = big_keys;
            }
            if (k_big) kp = hmul2_bits(kp, k16th);
            if (v_big) vp = hmul2_bits(vp, k16th);
            if (not_finite) vp = 0;
            k_par[t] = kp;
            v_scale[t] = __ushort_as_half(static_cast<unsigned short>(vp));
            v_offset[t] = __ushort_as_half(static_cast<unsigned short>(vp >> 16));
          }
        }
        if (j >= kKBufs) wait(kKEmpty + kbuf, j / kKBufs - 1);
        asm volatile("bar.sync 1, %0;" ::"n"(F::kUnpack) : "memory");
        {
          constexpr int kPieces = D / 32;  // 16-byte pieces of a token
          const uint32_t q = t % kPieces;
          const uint32_t swap = D == 128 ? q / 2 * 2 : 0;  // pieces of the second 64 dims in another order: other banks
#pragma unroll 1
          for (uint32_t at = t; at < kKeys * kPieces; at += F::kUnpack) {
            const uint32_t row = at / kPieces;
            const uint4 raw = *reinterpret_cast<const uint4*>(codes + row * (D / 2) + q * 16);
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
                out = make_uint4(hfma2_bits(x[w] & 0x000F000Fu, 0x40004000u, kCentre0), hadd2_bits(x[w] & 0x00F000F0u, kCentre1),
                                 hfma2_bits(x8 & 0x000F000Fu, 0x40004000u, kCentre0), hadd2_bits(x8 & 0x00F000F0u, kCentre1));
              } else {
                out.x = hfma2_bits(hadd2_bits((x[w] & 0x000F000Fu) | kExp, k1024), s2, o2);
                out.y = hfma2_bits(hfma2_bits((x[w] & 0x00F000F0u) | kExp, k16th, k64), s2, o2);
                out.z = hfma2_bits(hadd2_bits((x8 & 0x000F000Fu) | kExp, k1024), s2, o2);
                out.w = hfma2_bits(hfma2_bits((x8 & 0x00F000F0u) | kExp, k16th, k64), s2, o2);
              }
              umma::sts128(base + F::kK + kbuf * F::kOperand + (word / 8) * 16384 + umma::swz(row, word % 8), out);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if constexpr (kSplit) ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          arrive(kKFull + kbuf);
          arrive(kRawKFree + raw);
        }
        ok = wait(kRawVFull + raw, j / kRaws) && ok;
        {
          const uint32_t tg = lane % 8;
#pragma unroll 1
          for (uint32_t lin = warp - 8; lin < D / 16; lin += F::kUnpackWarps) {
            const uint32_t word = lin % (D / 32) * 4 + lane / 8, atom = lin / (D / 32);
            const uint32_t* from_v = reinterpret_cast<const uint32_t*>(codes + F::kRawV + (atom * 8 + tg) * F::kGroup) + word;
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
        if constexpr (kSplit) ok = __all_sync(0xffffffffu, ok);
        if (ok) {
          arrive(kVFull + buf);
          arrive(kRawVFree + raw);
        }
      }
    } else if (warp == F::kMmaWarp) {
      // ---- MMAs ----------------------------------------------------------------------------------------
      const uint32_t leader = umma::elect_lane();
      // scores into tensor memory's columns at t * 128 (of row block t, or f32: of every other tile), keys from buffer `kbuf`; f32: the
      // queries' low parts into columns of their own: added to the high ones they would be cut off step by step
      const auto scores = [&](uint32_t t, uint32_t kbuf) {
        const uint32_t q = desc_low(base + F::kQ + (kSplit ? 0 : t) * F::kOperand), k = desc_low(base + F::kK + kbuf * F::kOperand);
#pragma unroll
        for (int part = kParts - 1; part >= 0; --part)
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            mma_ss(leader, tmem + (part ? 256 : t * 128), q + (part * F::kOperand + s / 4 * 16384 + s % 4 * 32) / 16, k + (s / 4 * 16384 + s % 4 * 32) / 16, f16_idesc(kKeys),
                   s != 0);
        umma::commit_one(leader, bar(kSFull + t));
      };
      const auto outputs = [&](uint32_t t, uint32_t buf, uint32_t add) {
        const uint32_t v = desc_low(base + F::kV + buf * F::kOperand);
        // f32: the high parts first, whose sums are exact: products' bits line up with the operands' exponents, and a subnormal's is the
        // smallest normal one, so a high part's step would cut 2^-19 off a sum that held low ones
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int s = 0; s < kKeys / 16; ++s)
            mma_ts(leader, tmem + (kSplit ? 384 : 256 + t * 128), tmem + t * 128 + s * 16 + part * 8, v + (s / 4 * (D * 128) + s % 4 * 32) / 16, f16_idesc(D),
                   part != 0 || s != 0 ? 1 : add);
        umma::commit_one(leader, bar(kOFull + (kSplit ? 0 : t)));
      };
      const auto keys_ready = [&](int j) {
        wait(kKFull + j % kKBufs, j / kKBufs);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      };
      if constexpr (kSplit) {
        // the next tile's scores are made while the softmax works on this one's
        if (tiles > 0) {
          keys_ready(0);
          scores(0, 0);
          umma::commit_one(leader, bar(kKEmpty));
        }
        for (int j = 0; j < tiles; ++j) {
          const uint32_t t = j & 1;
          if (j + 1 < tiles) {
            keys_ready(j + 1);
            wait(kLoaded, j);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            scores(t ^ 1, (j + 1) % kKBufs);
            umma::commit_one(leader, bar(kKEmpty + (j + 1) % kKBufs));
          }
          wait(kPReady + t, j / 2);
          wait(kVFull + t, j / 2);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          outputs(t, t, 0);
          umma::commit_one(leader, bar(kVEmpty + t));
        }
      } else {
        if (tiles > 0) {
          keys_ready(0);
          scores(0, 0);
          scores(1, 0);
          umma::commit_one(leader, bar(kKEmpty));
        }
        for (int j = 0; j < tiles; ++j) {
          const uint32_t buf = j % kVBufs;
          for (uint32_t t = 0; t < 2; ++t) {
            wait(kPReady + t, j);
            if (t == 0) wait(kVFull + buf, j / kVBufs);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            outputs(t, buf, j > 0);
            if (t == 1) umma::commit_one(leader, bar(kVEmpty + buf));
            if (j + 1 < tiles) {
              if (t == 0) keys_ready(j + 1);
              scores(t, (j + 1) % kKBufs);
              if (t == 1) umma::commit_one(leader, bar(kKEmpty + (j + 1) % kKBufs));
            }
          }
        }
      }
      if (__any_sync(0xffffffffu, *abort_flag)) {  // a wait gave up: none may outlive the tensor memory
        umma::commit_one(leader, bar(kAllDone));
        wait(kAllDone, 0);
      }
    } else if (warp == F::kCopyWarp) {
      // ---- copies --------------------------------------------------------------------------------------
      const uint32_t P = p.a.cache.page_tokens, block_bytes = static_cast<uint32_t>(cache_block_bytes(P, D));
      const int* const pages = p.a.batch.pages + static_cast<size_t>(read_through) * p.a.batch.width;
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
        const uint32_t raw = j % kRaws, codes = base + F::kRaw + raw * F::kRawBytes;
        if (j >= kRaws) ok = wait(kRawKFree + raw, j / kRaws - 1) && ok;
        ok = __all_sync(0xffffffffu, ok);
        const uint32_t n_k = __popc(__ballot_sync(0xffffffffu, have_k)), n_v = __popc(__ballot_sync(0xffffffffu, have_v));
        if (ok && lane < 8 && !have_k && key_k <= key_last) {  // no such page: what it would hold is NaN
          uint32_t* params = reinterpret_cast<uint32_t*>(smem + F::kRaw + raw * F::kRawBytes + F::kRawParams) + lane * 16;
          for (int i = 0; i < 16; ++i) params[i] = params[kKeys + i] = 0x7E007E00u;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        __syncwarp();
        if (!ok) break;  // a wait gave up: nothing more is copied
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(kRawKFull + raw)), "r"(n_k * 16 * (D / 2 + 8)) : "memory");
        __syncwarp();
        if (have_k) {
          const uint32_t slot = static_cast<uint32_t>(key_k) & (P - 1);
          copy(codes + lane * 16 * (D / 2), block_k + slot * (D / 2), 16 * (D / 2), kRawKFull + raw);
          copy(codes + F::kRawParams + lane * 64, block_k + P * D + slot * 4, 64, kRawKFull + raw);
          copy(codes + F::kRawParams + kKeys * 4 + lane * 64, block_k + P * D + (P + slot) * 4, 64, kRawKFull + raw);
        }
        if (j >= kRaws) ok = wait(kRawVFree + raw, j / kRaws - 1) && ok;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar(kRawVFull + raw)), "r"(n_v * 4 * D) : "memory");
        __syncwarp();
        if (have_v) copy(codes + F::kRawV + lane * F::kGroup, block_v + (P + (static_cast<uint32_t>(key_v) & (P - 1))) * (D / 2), 4 * D, kRawVFull + raw);
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncthreads();
  if (warp == F::kMmaWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <typename T, int D, bool kGroups>
cudaError_t many_as(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh, bool prefix) {
  using F = Many<T, D>;
  static_assert(F::kSmem <= 227 * 1024 && F::kTable % 16 == 0 && F::kRows % 16 == 0 && F::kRare % 16 == 0 && F::kBars % 8 == 0 && F::kRawParams % 16 == 0 && F::kRawBytes % 16 == 0,
                "shared memory and the alignment of its arrays");
  static OncePerDevice once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(attend_many_kernel<T, D, kGroups>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem); });
  if (e != cudaSuccess) return e;
  ManyParams p;
  p.a = a;
  p.group = a.heads / a.cache.kv_heads;
  p.page_shift = 0;
  while ((1u << p.page_shift) < a.cache.page_tokens) ++p.page_shift;
  p.beyond = beyond;
  p.status = env.status;
  p.prefix = prefix;
  p.sh = sh;
  const uint64_t blocks = groups::most_blocks(static_cast<uint64_t>(a.batch.tokens) * p.group, F::kBlock, prefix ? sh.groups : a.batch.sequences, beyond);
  cudaLaunchConfig_t cfg = {};
  const uint64_t units = blocks * a.cache.kv_heads;
  // Few units: their keys are shared, so that every SM has its part (a part more for each unit's odd end).
  p.parts = nullptr;
  p.counters = env.counters;
  p.ctas = static_cast<uint32_t>(env.sm_count);
  uint64_t grid = units;
  if (units < 2ull * p.ctas && units <= F::kUnits && units <= env.counter_count && env.workspace &&
      (units + p.ctas) * F::kPartFloats * sizeof(float) <= env.workspace_bytes) {
    p.parts = static_cast<float*>(env.workspace);
    grid = units + p.ctas;
  }
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(F::kThreads);
  cfg.dynamicSmemBytes = F::kSmem;
  cfg.stream = env.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = env.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attend_many_kernel<T, D, kGroups>, p);
}

template <bool kGroups>
cudaError_t launch_many(const LaunchEnv& env, const AttendArgs& a, uint32_t beyond, const SharedArgs& sh, bool prefix) {
  const auto in = [&](auto type) {
    using T = decltype(type);
    return a.cache.head_dim == 64 ? many_as<T, 64, kGroups>(env, a, beyond, sh, prefix) : many_as<T, 128, kGroups>(env, a, beyond, sh, prefix);
  };
  if (a.dtype == KQ_F32) return in(float());
  if (a.dtype == KQ_F16) return in(__half());
  return in(__nv_bfloat16());
}

}  // namespace
}  // namespace kq
