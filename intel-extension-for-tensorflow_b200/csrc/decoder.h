// Shared device helpers of the decoder operators (rotary positions, per-head norms, the 4-bit cache and attention).
#ifndef ITEXB_CSRC_DECODER_H_
#define ITEXB_CSRC_DECODER_H_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "common.h"
#include "gemm_sm100.h"  // FastDiv

namespace itexb {

__device__ __forceinline__ uint32_t QuickDiv(uint32_t x, const FastDiv& d) {  // x < 2^31
  return d.mul == 0u ? x : __umulhi(x, d.mul) >> d.shift;
}

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }

// Pairs of fp32 values handled by one instruction; each is rounded as alone.
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 Make2(float x, float y) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ F2 Same2(float x) { return Make2(x, x); }
__device__ __forceinline__ float X(F2 a) { return __uint_as_float(uint32_t(a.v)); }
__device__ __forceinline__ float Y(F2 a) { return __uint_as_float(uint32_t(a.v >> 32)); }
__device__ __forceinline__ F2 Fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ F2 Mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 Add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 Sub2(F2 a, F2 b) { return Fma2(b, Make2(-1.f, -1.f), a); }

// Two rounded values as one 32-bit word, the first in its low half.
template <typename T> __device__ __forceinline__ uint32_t Pack16(float lo, float hi) {
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// VEC elements moved as one access of VEC * sizeof(T) bytes (1, 2, 4, 8 or 16); the caller guarantees the alignment.
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ void LoadVec(const T* p, float (&f)[VEC]) {
  static_assert(sizeof(T) * VEC <= 16, "no wider access than the alignment that is asked of tensors");
  const Vec<T, VEC> x = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = ToFloat(x.v[i]);
}
template <typename T, int VEC> __device__ __forceinline__ void StoreVec(T* p, const float (&f)[VEC]) {
  static_assert(sizeof(T) * VEC <= 16, "no wider access than the alignment that is asked of tensors");
  union { Vec<T, VEC> x; uint32_t w[(sizeof(T) * VEC + 3) / 4]; } u;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) u.w[i / 2] = Pack16<T>(f[i], f[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.x.v[i] = FromFloat<T>(f[i]);
  }
  *reinterpret_cast<Vec<T, VEC>*>(p) = u.x;
}

__device__ __forceinline__ int64_t LoadIndex(const void* p, int is64, int64_t i) {
  return is64 ? __ldg(static_cast<const long long*>(p) + i) : int64_t(__ldg(static_cast<const int*>(p) + i));
}

// Copies to shared memory that run beside the thread's work (pieces of 16 or 8 bytes; smaller ones are copied at once).
template <typename P> __device__ __forceinline__ void CopyAhead(P* to, const P* from) {
  if constexpr (sizeof(P) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
  else if constexpr (sizeof(P) == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
  else *to = *from;
}
__device__ __forceinline__ void CommitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void WaitCopies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Rows of consecutive tokens in steps of a block's thread groups.
struct Walk {
  uint32_t token, head, dt, dh, heads;
  __device__ __forceinline__ Walk(uint32_t t0, uint32_t row, uint32_t step, uint32_t heads_, const FastDiv& div) : heads(heads_) {
    const uint32_t t = QuickDiv(row, div);
    token = t0 + t;
    head = row - t * heads;
    dt = QuickDiv(step, div);
    dh = step - dt * heads;
  }
  __device__ __forceinline__ void Next() {
    token += dt;
    head += dh;
    if (head >= heads) { head -= heads; ++token; }
  }
};

// Fraction of a turn of position * radians-per-position, in [-1/2, 1/2].  At position 10^6 a 32-bit product would be off
// by 0.06 rad; the 64-bit one is off by 10^-10.
__device__ __forceinline__ double TurnFraction(int64_t pos, double inv_freq) {
  const double turns = double(pos) * (inv_freq * 0.15915494309189533577);  // 1 / (2 pi)
  return turns - rint(turns);
}

__device__ __forceinline__ void ReportIndex(int32_t* status_word) {
  if (status_word != nullptr) atomicCAS(status_word, 0, ITEXB_STATUS_BAD_INDEX);
}

}  // namespace itexb

#endif  // ITEXB_CSRC_DECODER_H_
