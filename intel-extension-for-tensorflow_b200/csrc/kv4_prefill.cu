// Attention of many query rows over the 4-bit paged cache: prompts and their chunks.
//
// Bound: the tensor cores' 4 head_dim operations per (row, token) pair, and beside them the exponentials: 16 per clock and SM
// against the 32 pairs per clock that the two products of head_dim 128 allow.
//
// A unit of work is 256 query rows of one key/value head (new tokens times the query heads that share it; 128 rows for
// head_dim 256) against the tokens they see, in tiles of 128 (64 where keys and values are split).  One block of 640 (512) threads per SM takes an equal, contiguous part
// of the list of all units' tiles; units that several blocks share are joined by a second kernel:
//   warps 0, 1   issue tcgen05.mma (f16 operands, fp32 accumulators in tensor memory) for a half of 128 rows each: S = q K^T
//                and O += P V, 64 tokens at a time.  A half has two S, so that the next one is there before its softmax asks
//                for it.  (One warp for both halves spent more time on its waits and instructions than the tensor cores on
//                the products: 1760 clocks per half and 64 tokens against 640.)
//                Tensor memory: two S of each half (64 columns; P overwrites it as halves), O of each half
//   warps 4-11   softmax, a thread per row: weights 2^(s - m + 7) straight from S with the maximum m of earlier tokens; only
//                when a row's weights of 64 tokens add up to more than 2^15 is the maximum looked for, the accumulator rescaled
//                and the 64 tokens done again, once.  Weights go back to tensor memory as the second product's A operand.
//   warps 12-15, 16-19  keys and values, a thread per token: page lookup, codes and params into registers one tile ahead, values
//                lo + step * code as halves into shared memory in the layout the tensor cores read (128-byte swizzle; keys
//                K-major, values MN-major: both are rows of channels).
// Operands are halves, q scaled by a power of two per row (see kv4_steps.cu).  For bf16 inputs keys and values are rounded to
// halves once, 2^-12 of themselves, which is nothing next to the results' own rounding (2^-9).  For half inputs, where three such
// roundings (keys, values, weights) would nearly double the results' error (rms 0.00038 against 0.00021 of their own
// rounding alone), keys and values are split into two halves each and a tile holds 64 tokens' first halves and behind them
// the second ones: twice the products, 0.00026.  The order of channels is the codes' in a word, for q, keys and the output alike.
// Measured with warm caches, 2048 new tokens after 8192 with 32 / 8 heads of 128: bf16 344 us, 0.90 PFLOP/s (softmax warps: 1650
// clocks per 128 rows and 64 tokens, the products 1280 for both halves); half 769 us (0.80 PFLOP/s of products).  1024 tokens with
// head_dim 256: 431 and 1548 us (one stage: the conversion is not hidden).  Six prompts up to 1900, window 1024: bf16 385, half 496
// us.  With cold ones 377 us for the first, bf16.
// Rows of the cache that no query may see are zeros here; a value group stored as NaN, or whose values pass the largest half, is
// zeros too and makes the rows that see it NaN at the end.  Every wait is bounded.
#include <algorithm>

#include "kv4_attention.h"

namespace itexb {
namespace {

constexpr int kTileRows = 128;               // of a tile: its tokens or, where keys and values are split, 64 tokens' rounded
                                             // values and behind them what the rounding left
constexpr int kPart = 64;                    // tokens per product
template <bool SPLIT> constexpr int kTokens = SPLIT ? kPart : kTileRows;   // per tile
constexpr int kRows = 128;                   // per half: lanes of tensor memory
constexpr float kUp = 7.f;                   // weights are 2^(score - maximum + 7),
constexpr float kLimit = 32768.f;            // and their sum over 64 tokens at most 2^15, so that none overflows a half
constexpr float kNone = 3.0e38f;             // -maximum + 7 of no scores; -kNone: the largest of no products
constexpr float kFarthest = 2.9e38f;         // of some scores at most
// Scores this large (of any row of a warp) have their maximum taken off before they are scaled: 7 - maximum as one fp32 number
// would be off by 2^-25 of the maximum, in all weights alike, but where the maximum moves and where parts are joined.
constexpr float kFar = 1024.f;
constexpr long long kWaitCycles = 4000000000ll;   // about 2 s

template <int DIM> struct Shape {
  static constexpr int kHalves = DIM == 256 ? 1 : 2;       // of 128 rows
  static constexpr int kStages = DIM == 256 ? 1 : 2;       // tiles of keys, and of values
  // groups of four warps: issue, softmax of each half, keys, values
  static constexpr int kThreads = (3 + kHalves) * 128;
  // registers per thread of these groups; their sum is at most what the launch gives (a multiple of 8 up to 65536 / kThreads)
  static constexpr int kIssueRegs = DIM == 256 ? 80 : 56, kSoftmaxRegs = DIM == 256 ? 176 : 152, kConvertRegs = DIM == 256 ? 128 : 56;
  static constexpr int kQBytes = kHalves * kRows * DIM * 2, kTileBytes = kTileRows * DIM * 2;
  static constexpr int kSmem = kQBytes + 2 * kStages * kTileBytes;
  static constexpr int kOColumn = kHalves * 128;           // of the first half's O; S `u` of half m starts at column 128 m + 64 u
};

__device__ __forceinline__ uint32_t SmemAt(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void BarInit(uint64_t* b, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(SmemAt(b)), "r"(count) : "memory"); }
__device__ __forceinline__ void BarArrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(SmemAt(b)) : "memory"); }
__device__ __forceinline__ bool BarTry(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(SmemAt(b)), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded: false when the wait ran out or, with `quit`, another role gave up.
__device__ __forceinline__ bool BarWait(uint64_t* b, uint32_t parity, volatile int* quit, int32_t* status) {
  if (BarTry(b, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t n = 1;; ++n) {
    if (BarTry(b, parity)) return true;
    if ((n & 255u) == 0) {
      if (quit != nullptr && *quit) return false;
      if (clock64() - t0 > kWaitCycles) {
        if (quit != nullptr) *quit = 1;
        if (status != nullptr) atomicCAS(status, 0, ITEXB_STATUS_WAIT_EXPIRED);
        return false;
      }
    }
  }
}
__device__ __forceinline__ void FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void Commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(SmemAt(b)) : "memory");
}
// Operand descriptors: rows of 128 bytes in groups of eight, 1024 bytes apart, 128-byte swizzle.  The low word holds the
// address and `lead`, the bytes between blocks of 64 channels where channels are the operand's outer dimension (values); the high
// word is a constant.  `off`: bytes from `low`'s address on.
__device__ __forceinline__ uint32_t DescLow(uint32_t at, uint32_t lead) { return ((at & 0x3ffffu) >> 4) | ((lead >> 4) << 16); }
constexpr uint32_t kDescHigh = uint32_t(1024 >> 4) | (1u << 14) | (2u << 29);
template <bool ADD> __device__ __forceinline__ void MmaSmem(uint32_t d, uint32_t a_low, uint32_t b_low, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a_low), "r"(b_low), "r"(idesc), "n"(kDescHigh), "n"(int(ADD))
      : "memory");
}
template <bool ADD> __device__ __forceinline__ void MmaTmem(uint32_t d, uint32_t a, uint32_t b_low, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b_low), "r"(idesc), "n"(kDescHigh), "n"(int(ADD))
      : "memory");
}
// One lane of a converged warp; the code around it stays uniform, so that operands live in uniform registers.
__device__ __forceinline__ bool ElectOne() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Load and wait in one statement: as two, every register was copied between them.
__device__ __forceinline__ void TmemLoad32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
        "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
        "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void TmemLoad64(uint32_t at, uint32_t (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), 
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), 
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), 
        "=r"(v[30]), "=r"(v[31]), "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]), 
        "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]), "=r"(v[49]), 
        "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), 
        "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void TmemStore32(uint32_t at, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), 
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), 
      "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void TmemStore16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ void TmemLoad16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                 "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void TmemStoreDone() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int N> __device__ __forceinline__ void RegistersDown() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void RegistersUp() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// The power of two that goes into the weights of a row whose largest product so far is `ref`.
__device__ __forceinline__ float ShiftOf(float ref, float scale) {
  return ref <= -kNone ? kNone : fminf(fmaxf(fmaf(-ref, scale, kUp), -kFarthest), kFarthest);
}

// A row's accumulator times f.
template <int DIM> __device__ __forceinline__ void Rescale(uint32_t o_at, float f) {
#pragma unroll 1
  for (int c = 0; c < DIM / 16; ++c) {
    uint32_t v[16];
    TmemLoad16(o_at + c * 16, v);
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
    TmemStore16(o_at + c * 16, v);
  }
  TmemStoreDone();
}

// Byte offset of 16-byte piece `piece` of row `row` in a tile of rows of DIM halves: blocks of 64 channels, 128-byte swizzle.
__device__ __forceinline__ uint32_t PieceAt(int row, int piece) {
  return uint32_t(piece >> 3) * (128 * 128) + uint32_t(row) * 128 + uint32_t(((piece & 7) ^ (row & 7)) * 16);
}
__device__ __forceinline__ uint32_t AndOr(uint32_t x, uint32_t mask, uint32_t constant) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(constant));
  return r;
}
__device__ __forceinline__ uint32_t HalfAdd2(uint32_t a, uint32_t b) { uint32_t r; asm("add.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t HalfSub2(uint32_t a, uint32_t b) { uint32_t r; asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t HalfMul2(uint32_t a, uint32_t b) { uint32_t r; asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ uint32_t HalfFma2(uint32_t a, uint32_t b, uint32_t c) { uint32_t r; asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c)); return r; }
// What a pair of operands holds of lo + step * code: the value rounded once, or in two parts, the sum of the rounded product
// and lo as rounded, and what these two roundings left (exact but for its own rounding, 2^-11 of a rounding).
enum Part { kValue, kSum, kLeft };
// For the codes at two nibbles of a word: the code's bits in the mantissa of 1024 (bits 0-3) or 64 (bits 4-7), the constant
// subtracted (exact).
template <int PART> __device__ __forceinline__ uint32_t Value2(uint32_t bits, uint32_t minus, uint32_t step2, uint32_t then2, uint32_t lo2) {
  const uint32_t c = HalfAdd2(bits, minus);
  if (PART == kValue) return HalfFma2(c, step2, lo2);
  const uint32_t p = HalfMul2(c, step2);
  if (PART == kSum) return HalfFma2(p, then2, lo2);
  const uint32_t sum = HalfAdd2(p, lo2);
  // the product's rounding and the sum's, whichever of its terms is the larger
  const uint32_t of_p = HalfFma2(c, step2, p ^ 0x80008000u), lo_part = HalfSub2(sum, p), p_part = HalfSub2(sum, lo_part);
  return HalfAdd2(HalfAdd2(HalfSub2(p, p_part), HalfSub2(lo2, lo_part)), of_p);
}
template <int PART> __device__ __forceinline__ uint4 Values8(uint32_t w, uint32_t step2, uint32_t then2, uint32_t lo2) {
  const uint32_t u = w >> 8;
  return make_uint4(Value2<PART>(AndOr(w, 0x000F000Fu, 0x64006400u), 0xE400E400u, step2, then2, lo2),
                    Value2<PART>(AndOr(w, 0x00F000F0u, 0x54005400u), 0xD400D400u, step2, then2, lo2),
                    Value2<PART>(AndOr(u, 0x000F000Fu, 0x64006400u), 0xE400E400u, step2, then2, lo2),
                    Value2<PART>(AndOr(u, 0x00F000F0u, 0x54005400u), 0xD400D400u, step2, then2, lo2));
}
// |step| of 2048 or |lo| of 32768 and more: below, neither a rounded product (30720 at most) nor its sum with lo passes 65504.
__device__ __forceinline__ bool Wide(uint32_t p) { return (p & 0x7fff0000u) >= 0x68000000u || (p & 0x7fffu) >= 0x7800u; }

// Eight outputs, from the codes' order (0 4 1 5 2 6 3 7) back to the channels'.
__device__ __forceinline__ void StoreOut8(const AttnArgs& a, int bf16, int64_t at, const float (&f)[8]) {
  union { uint4 x; uint32_t u[4]; uint16_t e[8]; } out;
#pragma unroll
  for (int e = 0; e < 4; ++e) {   // channels 2e, 2e + 1
    const float lo = f[e < 2 ? 4 * e : 4 * e - 7], hi = f[e < 2 ? 4 * e + 2 : 4 * e - 5];
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(out.u[e]) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(out.u[e]) : "f"(hi), "f"(lo));
  }
  uint16_t* to = static_cast<uint16_t*>(a.out) + at;
  if ((reinterpret_cast<uintptr_t>(to) & 15) == 0) *reinterpret_cast<uint4*>(to) = out.x;
  else
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = out.e[e];
}

// A token's row of codes and params.
template <int DIM, int GROUP> struct Row {
  static constexpr int NG = DIM / GROUP;
  uint4 codes[DIM / 32];
  uint32_t params[NG];
  __device__ __forceinline__ void Load(const uint8_t* c, const __half2* p) {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) codes[i] = __ldg(reinterpret_cast<const uint4*>(c) + i);
    if constexpr (NG == 1) params[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    else if constexpr (NG == 2) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      params[0] = x.x; params[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < NG; i += 4) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p + i));
        params[i] = x.x; params[i + 1] = x.y; params[i + 2] = x.z; params[i + 3] = x.w;
      }
    }
  }
  __device__ __forceinline__ void Clear() {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) codes[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < NG; ++i) params[i] = 0;
  }
  // -> the row's halves in shared memory
  template <int PART> __device__ __forceinline__ void Store(uint8_t* tile, int row) const {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) {
      const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int piece = i * 4 + k;
        uint32_t p = params[piece * 8 / GROUP], then2 = 0x3c003c00u;   // 1
        uint32_t step2 = __byte_perm(p, p, 0x3232), lo2 = __byte_perm(p, p, 0x1010);
        if (PART != kValue && Wide(p)) {   // of a wide group the first part is the value, the second nothing
          then2 = step2;
          step2 = PART == kSum ? 0x3c003c00u : 0u;
          lo2 = PART == kSum ? lo2 : 0u;
        }
        *reinterpret_cast<uint4*>(tile + PieceAt(row, piece)) = Values8<PART>(w[k], step2, then2, lo2);
      }
    }
  }
};
// A pair (lo, step) stored as NaN, or of values that are no finite halves: lo + 15 step or step is not one.
__device__ __forceinline__ bool BadPair(uint32_t p) {
  const uint32_t x = HalfFma2(__byte_perm(p, 0u, 0x4432), 0x4B804B80u, __byte_perm(p, p, 0x3210));   // (step, 0) * 15 + (lo, step)
  return (x & 0x7c00u) == 0x7c00u || (x & 0x7c000000u) == 0x7c000000u;
}

struct Head {              // the unit that a block goes on with at its start, for the joining kernel
  int b, kvh, row0;        // b < 0: it starts with a unit of its own
  int first, last;         // blocks that share the unit
};
struct PrefillArgs {
  AttnArgs a;
  int bf16, row_tiles;     // row tiles of a sequence at most
  float* part_o;           // [blocks][2][head_dim / 4][rows][4]: of a unit begun by an earlier block, of one left to the next
  float2* part_l;          // [blocks][2][rows] (shift, sum of weights)
  Head* heads;             // [blocks]
};
constexpr int kMaxBlocks = 148;
constexpr int kLeastTiles = 2;    // of a block's part, where there is little work: 64 tokens after 960 take 26 us with 1 or 2, 29 with 4

// A unit of work: M * 128 query rows of a sequence and key/value head.  The list of units runs over sequences, their row tiles
// and the heads, in this order.
struct Unit { int row0, row1, begin, some_begin, end, tiles; };
template <int ROWS, bool SPLIT> __device__ __forceinline__ Unit UnitOf(const AttnArgs& a, const Seq& q, int rt) {
  Unit u;
  const int rows = q.nnew * a.share;
  u.row0 = rt * ROWS;
  u.row1 = min(rows, u.row0 + ROWS);
  u.begin = u.some_begin = u.end = u.tiles = 0;
  if (u.row0 >= rows) return u;
  u.some_begin = RowBegin(a, q, int(QuickDiv(uint32_t(u.row0), a.div_share)));
  u.end = RowEnd(a, q, int(QuickDiv(uint32_t(u.row1 - 1), a.div_share)));
  u.begin = u.some_begin & ~15;
  u.tiles = max(1, (u.end - u.begin + kTokens<SPLIT> - 1) / kTokens<SPLIT>);   // rows that see nothing are one empty tile
  return u;
}

// What a block works on next; every role walks the same segments.
struct Segment { Seq q; Unit u; int b, kvh, tile0, tile1, halves; };
struct Walker { int64_t left; int b, rt, kvh, tile; bool fresh; };   // what lies behind it

struct Shared {   // behind the operand tiles
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], o_done[2][2], drained[2];
  uint32_t tmem;
  volatile int quit;
  int bad_tile;            // the block's last tile so far with a value group that is a BadPair, -1: none
  uint32_t there[4][4];    // of the last four tiles: tokens that exist, 32 per word
  int64_t sums[20], left;
  int b, rt, kvh, tile;    // where this block's part begins
  Walker walk[20];
  Segment seg[20];
};

template <int DIM, int GROUP, bool SPLIT>
__global__ void __launch_bounds__(Shape<DIM>::kThreads, 1) PrefillKernel(const __grid_constant__ PrefillArgs s) {
  using H = Shape<DIM>;
  constexpr int M = H::kHalves, ST = H::kStages, NG = DIM / GROUP, ROWS = M * kRows, kThreads = H::kThreads;
  constexpr int kParts = kTokens<SPLIT> / kPart;   // of a tile
  const AttnArgs& a = s.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const s_q = smem;
  uint8_t* const s_k = smem + H::kQBytes;
  uint8_t* const s_v = s_k + ST * H::kTileBytes;
  Shared& sh = *reinterpret_cast<Shared*>(s_v + ST * H::kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((SmemAt(smem) & 1023u) != 0) {   // the swizzle needs it; refuse rather than compute garbage
    if (threadIdx.x == 0 && a.status_word != nullptr) atomicCAS(a.status_word, 0, ITEXB_STATUS_WAIT_EXPIRED);
    return;
  }
  // Launched programmatically: what the previous kernel of the stream wrote is visible from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this block's part of the list: threads add up contiguous shares of the (sequence, row tile) pairs
  {
    const int64_t pairs = int64_t(a.num_seqs) * s.row_tiles, per = (pairs + kThreads - 1) / kThreads;
    const int64_t p0 = min(pairs, int64_t(threadIdx.x) * per), p1 = min(pairs, p0 + per);
    auto walk = [&](auto visit) {   // visit(b, rt, q, unit) -> go on
      int b = int(p0 / s.row_tiles), rt = int(p0 - int64_t(b) * s.row_tiles);
      Seq q{};
      for (int64_t p = p0; p < p1; ++p) {
        if (p == p0 || rt == 0) q = SeqOf(a, b, blockIdx.x == 0 && rt == 0);
        if (!visit(b, rt, q, UnitOf<ROWS, SPLIT>(a, q, rt))) return;
        if (++rt == s.row_tiles) { rt = 0; ++b; }
      }
    };
    int64_t sum = 0;
    walk([&](int, int, const Seq&, const Unit& u) { sum += int64_t(u.tiles) * a.c.kv_heads; return true; });
    int64_t before = sum;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, before, x);
      if (lane >= x) before += y;
    }
    if (lane == 31) sh.sums[warp] = before;
    if (threadIdx.x == 0) s.heads[blockIdx.x].b = -1;
    __syncthreads();
    int64_t total = 0;
#pragma unroll 1
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += sh.sums[w];
      total += sh.sums[w];
    }
    before -= sum;
    const int64_t blocks = max(int64_t(1), min(int64_t(gridDim.x), total / kLeastTiles));
    const int64_t pos = total * blockIdx.x / blocks;
    const int64_t stop = int64_t(blockIdx.x) < blocks ? total * (blockIdx.x + 1) / blocks : pos;
    if (threadIdx.x == 0) sh.left = stop - pos;
    if (stop > pos && pos >= before && pos < before + sum) {
      int64_t at = before;
      walk([&](int b, int rt, const Seq&, const Unit& u) {
        const int64_t n = int64_t(u.tiles) * a.c.kv_heads;
        if (pos >= at + n) { at += n; return true; }
        sh.b = b;
        sh.rt = rt;
        sh.kvh = int((pos - at) / u.tiles);
        sh.tile = int((pos - at) - int64_t(sh.kvh) * u.tiles);
        if (sh.tile > 0) {
          const int64_t x = at + int64_t(sh.kvh) * u.tiles;     // the unit's first tile in the list
          Head h;
          h.b = b; h.kvh = sh.kvh; h.row0 = u.row0;
          h.first = int(((x + 1) * blocks - 1) / total);
          h.last = int(((x + u.tiles) * blocks - 1) / total);
          s.heads[blockIdx.x] = h;
        }
        return false;
      });
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      BarInit(&sh.q_full[i], kRows);
      BarInit(&sh.k_full[i], 128);
      BarInit(&sh.k_empty[i], M);
      BarInit(&sh.v_full[i], 128);
      BarInit(&sh.v_empty[i], M);
      BarInit(&sh.drained[i], 1);
      for (int u = 0; u < 2; ++u) {
        BarInit(&sh.s_full[i][u], 2);      // the products' completion, and the issuer itself (for what it has seen others write)
        BarInit(&sh.p_full[i][u], kRows);
        BarInit(&sh.o_done[i][u], 2);
      }
    }
    sh.quit = 0;
    sh.bad_tile = -1;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t part = sh.left;       // tiles of this block
  if (part == 0) return;
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SmemAt(&sh.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  FenceBefore();
  __syncthreads();
  FenceAfter();
  const uint32_t tmem = sh.tmem;
  volatile int* const quit = &sh.quit;

  // The segments of this block's part, one after the other: each warp walks them by itself, its place in shared memory (in
  // registers it would cost every role twenty).
  Walker& wk = sh.walk[warp];
  Segment& g = sh.seg[warp];
  if (lane == 0) {
    wk.b = sh.b; wk.rt = sh.rt; wk.kvh = sh.kvh; wk.tile = sh.tile;
    wk.left = part;
    wk.fresh = true;
  }
  auto advance = [&]() {   // one thread
    if (wk.left <= 0) { g.tile0 = g.tile1 = 0; return; }
    if (wk.fresh) {
      g.q = SeqOf(a, wk.b, false);
      g.u = UnitOf<ROWS, SPLIT>(a, g.q, wk.rt);
      while (g.u.tiles == 0) {   // a sequence has fewer row tiles than the longest
        if (++wk.rt == s.row_tiles) { wk.rt = 0; g.q = SeqOf(a, ++wk.b, false); }
        g.u = UnitOf<ROWS, SPLIT>(a, g.q, wk.rt);
      }
      wk.fresh = false;
    }
    g.b = wk.b;
    g.kvh = wk.kvh;
    g.tile0 = wk.tile;
    g.tile1 = int(min(int64_t(g.u.tiles), wk.tile + wk.left));
    g.halves = g.u.row1 - g.u.row0 > kRows ? 2 : 1;
    wk.left -= g.tile1 - g.tile0;
    wk.tile = 0;
    if (++wk.kvh == a.c.kv_heads) {
      wk.kvh = 0;
      wk.fresh = true;
      if (++wk.rt == s.row_tiles) { wk.rt = 0; ++wk.b; }
    }
  };
  auto next_segment = [&]() {   // the whole warp
    __syncwarp();
    if (lane == 0) advance();
    __syncwarp();
    return g.tile1 > g.tile0;
  };

  // Registers go from the warps that issue and convert to the softmax warps; each role's branch states its own, so that its
  // code is compiled for it.
  if (warp < 4) {
    RegistersDown<H::kIssueRegs>();
    // ---------------- products: a warp for each half ----------------
    // The whole warp walks the loop, one lane issues.
    if (warp < M) {
      constexpr uint32_t kIdescS = (1u << 4) | (uint32_t(kPart >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (uint32_t(DIM >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      const int m = __shfl_sync(0xffffffffu, warp, 0);
      const uint32_t s_d = __shfl_sync(0xffffffffu, tmem, 0) + m * 128, o_d = s_d + H::kOColumn + m * (DIM - 128);
      const uint32_t q_low = DescLow(SmemAt(s_q), 16) + m * (kRows * DIM * 2 / 16), k_low = DescLow(SmemAt(s_k), 16), v_low = DescLow(SmemAt(s_v), 128 * 128);
      uint32_t t = 0;            // tiles of the block
      uint32_t parts = 0;        // 64 tokens each: those of this half whose weights have been multiplied; S by their parity
      uint32_t segs = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = __all_sync(0xffffffffu, ok && BarWait(bar, parity & 1, quit, a.status_word)); };
      // S number u, of part `at` of tile `tile`
      auto scores = [&](uint32_t tile, int at, int u) {
        FenceAfter();
        if (ElectOne()) {
          const uint32_t ka = k_low + (tile % ST) * (H::kTileBytes / 16) + at * (kPart * 128 / 16), d = s_d + u * kPart;
          MmaSmem<false>(d, q_low, ka, kIdescS);
#pragma unroll
          for (int k = 1; k < DIM / 16; ++k) {
            constexpr int kBlock = 128 * 128 / 16;
            MmaSmem<true>(d, q_low + (k / 4) * kBlock + (k % 4) * 2, ka + (k / 4) * kBlock + (k % 4) * 2, kIdescS);
          }
          if (SPLIT) {
#pragma unroll
            for (int k = 0; k < DIM / 16; ++k) {
              constexpr int kBlock = 128 * 128 / 16;
              MmaSmem<true>(d, q_low + (k / 4) * kBlock + (k % 4) * 2, ka + kPart * 128 / 16 + (k / 4) * kBlock + (k % 4) * 2, kIdescS);
            }
          }
          Commit(&sh.s_full[m][u]);
          BarArrive(&sh.s_full[m][u]);
          if (at == kParts - 1) Commit(&sh.k_empty[tile % ST]);
        }
        __syncwarp();
      };
      while (ok && next_segment()) {
        const int n = __shfl_sync(0xffffffffu, kParts * (g.tile1 - g.tile0), 0), halves = __shfl_sync(0xffffffffu, g.halves, 0);
        if (m >= halves) {
          // no rows here: the tiles are let through one by one, since a barrier's parity tells only neighbouring phases apart
          for (int j = 0; j < n / kParts && ok; ++j, ++t) {
            if (!wait(&sh.k_full[t % ST], t / ST)) break;
            if (ElectOne()) BarArrive(&sh.k_empty[t % ST]);
            if (!wait(&sh.v_full[t % ST], t / ST)) break;
            if (ElectOne()) BarArrive(&sh.v_empty[t % ST]);
            __syncwarp();
          }
          continue;
        }
        // the half's last weights of the segment before have been multiplied, its next rows of q are there
        if (parts > 0) wait(&sh.o_done[m][(parts - 1) & 1], (parts - 1) >> 1);
        wait(&sh.q_full[m], segs++);
        if (!wait(&sh.k_full[t % ST], t / ST)) break;
        scores(t, 0, parts & 1);
        for (int j = 0; j < n; ++j, ++parts) {
          const int u = parts & 1, at = j % kParts;   // at: part of tile t
          const bool last = at == kParts - 1;
          if (j + 1 < n) {
            // S of the part after this one goes where the weights of the one before it were
            if (last) wait(&sh.k_full[(t + 1) % ST], (t + 1) / ST);
            if (j > 0) wait(&sh.o_done[m][u ^ 1], (parts - 1) >> 1);
            if (!ok) break;
            scores(t + last, last ? 0 : at + 1, u ^ 1);
          }
          if (at == 0) wait(&sh.v_full[t % ST], t / ST);
          if (!wait(&sh.p_full[m][u], parts >> 1)) break;
          FenceAfter();
          if (ElectOne()) {
            const uint32_t va = v_low + (t % ST) * (H::kTileBytes / 16) + at * (kPart * 128 / 16), p = s_d + u * kPart;
            if (j > 0) MmaTmem<true>(o_d, p, va, kIdescO);
            else MmaTmem<false>(o_d, p, va, kIdescO);
#pragma unroll
            for (int k = 1; k < kPart / 16; ++k) MmaTmem<true>(o_d, p + k * 8, va + k * 128, kIdescO);
            if (SPLIT) {
#pragma unroll
              for (int k = 0; k < kPart / 16; ++k) MmaTmem<true>(o_d, p + k * 8, va + (kPart / 16 + k) * 128, kIdescO);
            }
            Commit(&sh.o_done[m][u]);
            BarArrive(&sh.o_done[m][u]);
            if (last) Commit(&sh.v_empty[t % ST]);
          }
          __syncwarp();
          t += last;
        }
      }
      // nothing in flight when tensor memory is given back
      if (ElectOne()) Commit(&sh.drained[m]);
      __syncwarp();
      BarWait(&sh.drained[m], 0, nullptr, a.status_word);
    }
  } else if (warp < 4 + 4 * M) {
    // ---------------- softmax ----------------
    RegistersUp<H::kSoftmaxRegs>();
    const int m = (warp - 4) >> 2, in_half = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_m = tmem + lanes + m * 128, o_at = tmem + lanes + H::kOColumn + m * DIM;
    uint32_t parts = 0, t4 = 0;   // 64 tokens each: of this half; all tiles of the block so far
    bool ok = true;
    while (ok && next_segment()) {
      const int n = g.tile1 - g.tile0;
      if (m >= g.halves) { t4 += n; continue; }
      const int rr = g.u.row0 + m * kRows + in_half;
      const bool on = rr < g.u.row1;
      const int i = int(QuickDiv(uint32_t(on ? rr : g.u.row0), a.div_share)), h = g.kvh * a.share + (on ? rr : g.u.row0) - i * a.share;
      const int lo = on ? RowBegin(a, g.q, i) : 0, hi = on ? RowEnd(a, g.q, i) : 0;
      // tokens that all rows of this warp see
      const int w_row = g.u.row0 + m * kRows + (warp & 3) * 32;
      const int w_first = int(QuickDiv(uint32_t(min(g.u.row1 - 1, w_row)), a.div_share)), w_last = int(QuickDiv(uint32_t(min(g.u.row1, w_row + 32) - 1), a.div_share));
      const int all_begin = RowBegin(a, g.q, max(w_first, w_last)), all_end = RowEnd(a, g.q, min(w_first, w_last));
      float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
      {
        // ---- the row of q: half, scaled, in the codes' order
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (g.q.row0 + i) * a.qt + int64_t(h) * a.qh;
        union Piece { uint4 v; uint32_t u[4]; uint16_t e[8]; };
        // up to 128 channels at a time in registers, all their loads in flight
        constexpr int kPieces = DIM / 8, kHeld = kPieces < 16 ? kPieces : 16;
        Piece x[kHeld];
        auto fetch = [&](int p0) {
#pragma unroll
          for (int p = 0; p < kHeld; ++p) {
            if (!on) x[p].v = make_uint4(0, 0, 0, 0);
            else if (a.q_aligned) x[p].v = __ldg(reinterpret_cast<const uint4*>(src) + p0 + p);
            else
#pragma unroll
              for (int e = 0; e < 8; ++e) x[p].e[e] = src[(p0 + p) * 8 + e];
          }
        };
        float down = a.scale_log2 < 0.f ? -1.f : (a.scale_log2 == 0.f ? 0.f : 1.f);
        if (s.bf16) {
          uint32_t bits = 0;
#pragma unroll 1
          for (int p0 = kPieces - kHeld; p0 >= 0; p0 -= kHeld) {   // the first ones last: they stay
            fetch(p0);
#pragma unroll
            for (int p = 0; p < kHeld; ++p)
#pragma unroll
              for (int e = 0; e < 4; ++e) bits = MaxBits2(x[p].u[e], bits);
          }
          const float most = __uint_as_float(max(bits << 16, bits & 0xffff0000u));
          const int e = min(max(int(__float_as_uint(most) >> 23), 1), 253);
          if (most > 0.f && most < INFINITY) {
            down *= __uint_as_float(uint32_t(254 - e) << 23);
            scale = fminf(fmaxf(scale * __uint_as_float(uint32_t(e) << 23), 1e-37f), kNone);
          }
        } else {
          fetch(0);
        }
        uint8_t* const to = s_q + m * (kRows * DIM * 2);
#pragma unroll 1
        for (int p0 = 0; p0 < kPieces; p0 += kHeld) {
          if (p0 > 0) fetch(p0);
#pragma unroll
          for (int p = 0; p < kHeld; ++p) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[p].u[e] = QueryHalf2(x[p].u[e], s.bf16, down);
            const uint32_t* u = x[p].u;
            *reinterpret_cast<uint4*>(to + PieceAt(in_half, p0 + p)) =
                make_uint4(__byte_perm(u[0], u[2], 0x5410), __byte_perm(u[0], u[2], 0x7632), __byte_perm(u[1], u[3], 0x5410), __byte_perm(u[1], u[3], 0x7632));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        BarArrive(&sh.q_full[m]);
      }
      // Weights are 2^((v - ref) * scale + 7) of a row's products v; ref is the largest of them, as of when it was last looked for.
      float ref = -kNone, shift = kNone, total = 0.f;
      bool far = false;                       // the warp's rows: ref is taken off first, else as 2^(v * scale + ShiftOf(ref))
      for (int j = 0; j < kParts * n && ok; ++j, ++parts) {
        const int u = parts & 1, at = j % kParts;
        ok = BarWait(&sh.s_full[m][u], (parts >> 1) & 1, quit, a.status_word);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        FenceAfter();
        const int j0 = g.u.begin + g.tile0 * kTokens<SPLIT> + j * kPart;
        const uint32_t* there = sh.there[t4 & 3] + 2 * at;
        const uint32_t s_at = s_m + u * kPart;
        const F2 scale2 = Make2(scale, scale);
        // of the half tile's tokens, those that exist and that this row sees; all of them in most half tiles
        uint64_t seen = uint64_t(there[0]) | (uint64_t(there[1]) << 32);
        const bool masked = j0 < all_begin || j0 + kPart > all_end || seen != ~uint64_t(0);
        if (masked) {
          const int from = min(max(lo - j0, 0), 64), to = min(max(hi - j0, 0), 64);
          seen &= (to == 64 ? ~uint64_t(0) : (uint64_t(1) << to) - 1) & ~(from == 64 ? ~uint64_t(0) : (uint64_t(1) << from) - 1);
        }
        uint32_t p[32];
#pragma unroll 1
        for (bool again = false;; again = true) {   // twice at most: with ref the maximum, no weight is above 2^7 but by rounding
          // P overwrites S only once its weights are known to be good
          uint32_t v[64];
          TmemLoad64(s_at, v);
          if (masked || far) {
            const float off = far ? ref : 0.f;
#pragma unroll
            for (int e = 0; e < 64; ++e)
              v[e] = (uint32_t(seen >> (e & 32)) & (1u << (e & 31))) == 0u ? 0xff800000u : __float_as_uint(__uint_as_float(v[e]) - off);
          }
          const F2 shift2 = Make2(shift, shift);
          F2 part[4] = {Make2(0.f, 0.f), Make2(0.f, 0.f), Make2(0.f, 0.f), Make2(0.f, 0.f)};
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const F2 d = Fma2(Make2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale2, shift2);
            const float x = Exp2(X(d)), y = Exp2(Y(d));
            part[(e >> 1) & 3] = Add2(part[(e >> 1) & 3], Make2(x, y));
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p[e / 2]) : "f"(y), "f"(x));
          }
          const F2 all = Add2(Add2(part[0], part[1]), Add2(part[2], part[3]));
          const float sum = X(all) + Y(all);
          if (again || !__any_sync(0xffffffffu, sum > kLimit)) {
            total += sum;
            break;
          }
          // a new maximum for the rows that passed it; the accumulator is scaled, these tokens are done again
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t w[16];
            TmemLoad16(s_at + c * 16, w);
            const uint32_t bits = uint32_t(seen >> (16 * c));
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if ((bits >> e) & 1u) top = fmaxf(top, __uint_as_float(w[e]));
          }
          const float to = fmaxf(ref, top), f = Exp2((ref - to) * scale);
          ref = to;
          far = __any_sync(0xffffffffu, to > -kNone && fabsf(to * scale) > kFar);
          shift = far ? kUp : ShiftOf(ref, scale);
          total *= f;
          if (j > 0) {   // once the half tile before has been added to it
            ok = ok && BarWait(&sh.o_done[m][u ^ 1], ((parts - 1) >> 1) & 1, quit, a.status_word);
            __syncwarp();
            FenceAfter();
            Rescale<DIM>(o_at, f);
          }
        }
        TmemStore32(s_at, p);
        TmemStoreDone();
        FenceBefore();
        BarArrive(&sh.p_full[m][u]);
        t4 += at == kParts - 1;
      }
      ok = __all_sync(0xffffffffu, ok) && __all_sync(0xffffffffu, BarWait(&sh.o_done[m][(parts - 1) & 1], ((parts - 1) >> 1) & 1, quit, a.status_word));
      if (!ok) break;
      FenceAfter();
      uint32_t nan_groups = 0;
      // Rare: find the value groups that are NaN among this part's tokens, a lane looking at one of 32, and keep those that this row
      // sees.  (The tile may be of a segment behind this one, whose conversion is ahead: then there are none to find.)
      if (__any_sync(0xffffffffu, *const_cast<volatile int*>(&sh.bad_tile) >= int(t4) - n)) {
        const int from = max(g.u.some_begin, g.u.begin + g.tile0 * kTokens<SPLIT>), to = min(g.u.end, g.u.begin + g.tile1 * kTokens<SPLIT>);
#pragma unroll 1
        for (int t0 = from; t0 < to; t0 += 32) {
          const int t = t0 + lane;
          uint32_t bad = 0;
          if (t < to) {
            const int col = int(QuickDiv(uint32_t(t), a.c.div_page)), page = __ldg(a.table + int64_t(g.b) * a.table_stride + col);
            if (page >= 0 && page < a.c.num_pages) {
              const __half2* at = a.c.v_params + int64_t(page) * a.c.pp + int64_t(g.kvh) * a.c.ph + int64_t(t - col * a.c.page_size) * a.c.pt;
              for (int x = 0; x < NG; ++x) bad |= uint32_t(BadPair(__ldg(reinterpret_cast<const uint32_t*>(at + x)))) << x;
            }
          }
          for (uint32_t left = __ballot_sync(0xffffffffu, bad != 0u); left != 0u; left &= left - 1u) {
            const int k = __ffs(int(left)) - 1;
            const uint32_t of_k = __shfl_sync(0xffffffffu, bad, k);
            if (t0 + k >= lo && t0 + k < hi) nan_groups |= of_k;
          }
        }
      }
      __syncwarp();
      const bool whole = g.tile1 - g.tile0 == g.u.tiles;
      const int64_t slot = int64_t(blockIdx.x) * 2 + (g.tile0 == 0);
      const int in_unit = m * kRows + in_half;
      if (!whole) s.part_l[slot * ROWS + in_unit] = make_float2(ShiftOf(ref, scale), total);
      float4* const part_to = reinterpret_cast<float4*>(s.part_o) + slot * (DIM / 4) * ROWS + in_unit;
      const float inv = total == 0.f ? 0.f : 1.f / total;
      const int64_t at = (g.q.row0 + i) * a.ot + int64_t(h) * a.oh;
#pragma unroll 1
      for (int c = 0; c < DIM / 32; ++c) {
        uint32_t v[32];
        __syncwarp();
        TmemLoad32(o_at + c * 32, v);
        if ((nan_groups >> (c * 32 / GROUP)) & 1u) {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0x7fffffffu;
        }
        if (!whole) {
#pragma unroll
          for (int w = 0; w < 8; ++w)
            part_to[(c * 8 + w) * ROWS] = make_float4(__uint_as_float(v[4 * w]), __uint_as_float(v[4 * w + 1]), __uint_as_float(v[4 * w + 2]), __uint_as_float(v[4 * w + 3]));
        } else if (on) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = total == 0.f ? 0.f : __uint_as_float(v[w * 8 + e]) * inv;
            StoreOut8(a, s.bf16, at + c * 32 + w * 8, f);
          }
        }
      }
      FenceBefore();
    }
  } else {
    // ---------------- codes to operands: one group of warps for the keys, one for the values ----------------
    if (H::kConvertRegs < 128) RegistersDown<H::kConvertRegs>();
    const bool values = warp >= 8 + 4 * M;
    const int t = threadIdx.x & 127, w = warp & 3;
    const uint8_t* const codes = values ? a.c.v_codes : a.c.k_codes;
    const __half2* const params = values ? a.c.v_params : a.c.k_params;
    uint8_t* const tiles = values ? s_v : s_k;
    uint64_t* const full = values ? sh.v_full : sh.k_full;
    uint64_t* const empty = values ? sh.v_empty : sh.k_empty;
    Row<DIM, GROUP> row;
    bool ok = true;
    // a tile: where this thread's token lies, -1 where there is none
    struct Place { int page, off, kvh; };
    bool more = next_segment();
    int ahead = g.tile0;
    auto place = [&]() {   // of the tile that `ahead` stands at, and one on
      Place x{-1, 0, 0};
      if (!more) return x;
      const int tok = g.u.begin + ahead * kTokens<SPLIT> + (SPLIT ? t % kPart : t);
      x.kvh = g.kvh;
      if (tok >= g.u.some_begin && tok < g.u.end) {
        const int col = int(QuickDiv(uint32_t(tok), a.c.div_page));
        x.off = tok - col * a.c.page_size;
        x.page = __ldg(a.table + int64_t(g.b) * a.table_stride + col);
        if (x.page < 0 || x.page >= a.c.num_pages) {
          ReportIndex(a.status_word);
          x.page = -1;
        }
      }
      if (++ahead == g.tile1) {
        more = next_segment();
        ahead = g.tile0;
      }
      return x;
    };
    auto load = [&](const Place& x) {
      if (x.page < 0) { row.Clear(); return; }
      row.Load(codes + int64_t(x.page) * a.c.cp + int64_t(x.kvh) * a.c.ch + int64_t(x.off) * a.c.ct,
               params + int64_t(x.page) * a.c.pp + int64_t(x.kvh) * a.c.ph + int64_t(x.off) * a.c.pt);
    };
    Place now = place(), next = place();
    load(now);
    uint32_t n = 0;      // tiles so far
    for (int64_t j = 0; j < part; ++j, ++n) {
      const Place after = place();
      if (n >= uint32_t(ST)) ok = BarWait(&empty[n % ST], (n / ST - 1) & 1, quit, a.status_word);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (values) {
        bool bad = false;
#pragma unroll
        for (int x = 0; x < NG; ++x)
          if (BadPair(row.params[x])) { row.params[x] = 0; bad = true; }
        if (bad) atomicMax(&sh.bad_tile, int(n));
      } else {
        const uint32_t there = __ballot_sync(0xffffffffu, now.page >= 0);
        if (lane == 0) sh.there[n & 3][w] = there;
      }
      if (SPLIT && t >= kPart) row.template Store<kLeft>(tiles + (n % ST) * H::kTileBytes, t);
      else row.template Store<SPLIT ? kSum : kValue>(tiles + (n % ST) * H::kTileBytes, t);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      BarArrive(&full[n % ST]);
      load(next);
      now = next;
      next = after;
    }
  }
  FenceBefore();
  __syncthreads();
  if (warp == 1) {
    FenceAfter();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// Joins the parts of a unit that several blocks worked on.  blockIdx.x: the block that went on with it first; a thread adds 8
// channels of one row.
template <int DIM>
__global__ void __launch_bounds__(256) PrefillJoinKernel(const __grid_constant__ PrefillArgs s) {
  constexpr int ROWS = Shape<DIM>::kHalves * kRows;
  const AttnArgs& a = s.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Head h = s.heads[blockIdx.x];
  if (h.b < 0 || h.first + 1 != int(blockIdx.x)) return;
  const Seq q = SeqOf(a, h.b, false);
  const int x = blockIdx.y * 256 + threadIdx.x, row = x % ROWS, piece = x / ROWS;   // threads along rows: the parts lie so
  const int rr = h.row0 + row;
  if (rr >= q.nnew * a.share) return;
  float least = kNone;
  for (int c = h.first; c <= h.last; ++c) least = fminf(least, s.part_l[(int64_t(c) * 2 + (c == h.first)) * ROWS + row].x);
  float sum = 0.f, f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0.f;
#pragma unroll 4
  for (int c = h.first; c <= h.last; ++c) {
    const int64_t slot = int64_t(c) * 2 + (c == h.first);
    const float2 l = s.part_l[slot * ROWS + row];
    const float w = l.x >= kNone ? (isnan(l.y) ? l.y : 0.f) : Exp2(least - l.x);
    const float4* from = reinterpret_cast<const float4*>(s.part_o) + (slot * (DIM / 4) + piece * 2) * ROWS + row;
    const float4 u = from[0], v = from[ROWS];
    const float o[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    sum = fmaf(l.y, w, sum);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf(o[e], w, f[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = sum == 0.f ? 0.f : f[e] / sum;
  const int i = int(QuickDiv(uint32_t(rr), a.div_share));
  StoreOut8(a, s.bf16, (q.row0 + i) * a.ot + int64_t(h.kvh * a.share + rr - i * a.share) * a.oh + piece * 8, f);
}

size_t PartBytes(const AttnArgs& a) {
  const size_t rows = (a.c.head_dim == 256 ? 1 : 2) * kRows;
  return size_t(kMaxBlocks) * 2 * rows * (size_t(a.c.head_dim) * sizeof(float) + sizeof(float2));
}

template <int DIM, int GROUP, bool SPLIT> int LaunchGroup(PrefillArgs& s, cudaStream_t st) {
  using H = Shape<DIM>;
  constexpr int kSmem = H::kSmem + int(sizeof(Shared)), ROWS = H::kHalves * kRows;
  auto kernel = PrefillKernel<DIM, GROUP, SPLIT>;
  ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int64_t rows = int64_t(s.a.max_new) * s.a.share;
  s.row_tiles = int((rows + ROWS - 1) / ROWS);
  int64_t span = std::min<int64_t>(s.a.max_kept, int64_t(s.a.table_cols) * s.a.c.page_size);
  if (s.a.window > 0) span = std::min<int64_t>(span, int64_t(s.a.window) + s.a.max_new);
  const int64_t most = (span / kTokens<SPLIT> + 2) * s.a.num_seqs * s.row_tiles * s.a.c.kv_heads;   // tiles
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(std::min<int64_t>(std::min(kMaxBlocks, SmCount()), std::max<int64_t>(1, most / kLeastTiles))));
  cfg.blockDim = dim3(H::kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const unsigned blocks = cfg.gridDim.x;
  ITEXB_CUDA(cudaLaunchKernelEx(&cfg, kernel, s));
  ITEXB_RETURN_IF_ERROR(CheckLaunch("PrefillKernel"));
  if (blocks == 1) return ITEXB_OK;
  cfg.gridDim = dim3(blocks, ROWS * (DIM / 8) / 256);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  ITEXB_CUDA(cudaLaunchKernelEx(&cfg, PrefillJoinKernel<DIM>, s));
  return CheckLaunch("PrefillJoinKernel");
}
template <int DIM, bool SPLIT> int LaunchDim(PrefillArgs& s, cudaStream_t st) {
  if (s.a.c.group == 32) return LaunchGroup<DIM, 32, SPLIT>(s, st);
  if (s.a.c.group == 64) return LaunchGroup<DIM, 64, SPLIT>(s, st);
  if constexpr (DIM >= 128) return LaunchGroup<DIM, 128, SPLIT>(s, st);
  return SetError(ITEXB_INTERNAL, "kv4_attention: group above head_dim");
}
template <bool SPLIT> int Launch(PrefillArgs& s, cudaStream_t st) {
  if (s.a.c.head_dim == 64) return LaunchDim<64, SPLIT>(s, st);
  if (s.a.c.head_dim == 128) return LaunchDim<128, SPLIT>(s, st);
  return LaunchDim<256, SPLIT>(s, st);
}

}  // namespace

size_t PrefillWorkspace(const AttnArgs& a) { return PartBytes(a) + kMaxBlocks * sizeof(Head); }

int LaunchPrefill(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st) {
  PrefillArgs s{};
  s.a = a;
  s.bf16 = dtype == ITEXB_DT_BFLOAT16;
  s.part_o = static_cast<float*>(workspace);
  s.part_l = reinterpret_cast<float2*>(s.part_o + size_t(kMaxBlocks) * 2 * (a.c.head_dim == 256 ? 1 : 2) * kRows * a.c.head_dim);
  s.heads = reinterpret_cast<Head*>(static_cast<uint8_t*>(workspace) + PartBytes(a));
  return s.bf16 ? Launch<false>(s, st) : Launch<true>(s, st);
}

}  // namespace itexb
