// Rows into the 4-bit paged cache (itexb_kv4_append: rotation of the keys, quantization) and back (itexb_kv4_gather).
//
//   lo = half(min of the group), step = half(max(0, (max - lo) / 15)), code = clamp(rne((x - lo) * (1 / step)), 0, 15)
//
// The step is the next lower half where lo + 15 step would not round to a finite half, which is enough for every group of
// finite halves; where it still does not, or a group holds a NaN or an infinity, the pair is NaN.
//
// Both are bound by HBM (append, head_dim 128, groups of 64, bf16: 256 B in, 72 B out per row).  A thread owns 8
// consecutive elements, which are one 32-bit word of codes; the 4 - 16 threads of a group exchange minimum and maximum
// by shuffles, and the rotation of halves its partners.  Every step is a separately rounded fp32 operation on cosines and
// sines rounded from 64 bits, so the codes are those of the same formulas written with plain fp32 tensor operations.
// Measured at 16384 tokens, 8 heads of 128, groups of 64, bf16: append 48 us (1.8 TB/s; its 620 instructions per warp and 2
// rows of keys and values bound it at 82 % of the issue slots, not the bytes), gather 20 us (4.3 TB/s).
#include <algorithm>
#include <climits>

#include "kv4.h"

namespace itexb {
namespace {

constexpr int kThreads = 256;
constexpr float kPastHalf = 65520.f;   // rounds to an infinite half

struct RowArgs {
  Kv4View c;
  uint32_t rows;          // tokens * kv_heads
  FastDiv div_heads;
  void* k; int64_t kt, kh;
  void* v; int64_t vt, vh;
  const void* slots;
  const void* positions;
  const double* inv_freq;
  FastDiv div_pairs;
  int slots64, pos64, pairs, interleaved, vec;
  int eights;             // the rotated halves are whole pieces of eight
  float mscale;
  int32_t* status_word;
};

__device__ __forceinline__ float MinNan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float MaxNan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float MinNan(float a, float b, float c) { float r; asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float MaxNan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// The row of a slot; false where there is none (-1) or it lies outside the cache (reported).
__device__ __forceinline__ bool RowOf(const RowArgs& a, int64_t slot, bool report, uint32_t* page, uint32_t* off) {
  if (slot < 0 || slot >= int64_t(a.c.num_pages) * a.c.page_size) {
    if (slot != -1 && report) ReportIndex(a.status_word);
    return false;
  }
  *page = QuickDiv(uint32_t(slot), a.c.div_page);
  *off = uint32_t(slot) - *page * uint32_t(a.c.page_size);
  return true;
}

// Codes and (lo, step) of the group this thread's eight elements belong to; `lanes` threads share the group.
__device__ __forceinline__ uint32_t Quantize8(const float (&x)[8], int lanes, __half2* params) {
  float mn = MinNan(MinNan(x[0], x[1], x[2]), x[3], x[4]), mx = MaxNan(MaxNan(x[0], x[1], x[2]), x[3], x[4]);
  mn = MinNan(MinNan(mn, x[5], x[6]), x[7]);
  mx = MaxNan(MaxNan(mx, x[5], x[6]), x[7]);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    mn = MinNan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = MaxNan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const __half lo = __float2half_rn(mn);
  const float lof = __half2float(lo);
  __half step = __float2half_rn(fmaxf((mx - lof) / 15.f, 0.f));
  float stepf = __half2float(step);
  if (!(fabsf(fmaf(15.f, stepf, lof)) < kPastHalf)) {   // rare; NaN and infinities come here too
    step = __ushort_as_half(uint16_t(__half_as_ushort(step) - 1));
    stepf = __half2float(step);
    if (!isfinite(lof) || !(fmaf(15.f, stepf, lof) < kPastHalf)) {
      *params = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
      return 0u;
    }
  }
  *params = __halves2half2(lo, step);
  // All scaled by 1/16, which is exact: saturation to [0, 1] then leaves one bound to apply.  Adding 1.5 * 2^23 rounds to
  // the nearest even integer, and four codes are summed as digits of one integer below 2^16.
  const float inv = stepf > 0.f ? 1.f / stepf * 0.0625f : 0.f;
  const F2 lo2 = Make2(-lof, -lof), one = Make2(1.f, 1.f), sixteen = Make2(16.f, 16.f), magic = Make2(12582912.f, 12582912.f);
  F2 code[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 d = Fma2(Make2(x[2 * i], x[2 * i + 1]), one, lo2);
    code[i] = Sub2(Fma2(Make2(fminf(__saturatef(X(d) * inv), 0.9375f), fminf(__saturatef(Y(d) * inv), 0.9375f)), sixteen, magic), magic);
  }
  const F2 w8 = Make2(256.f, 256.f);
  const F2 a = Fma2(code[1], w8, code[0]), b = Fma2(code[3], w8, code[2]);
  return __byte_perm(__float_as_uint(fmaf(Y(a), 16.f, X(a)) + 12582912.f), __float_as_uint(fmaf(Y(b), 16.f, X(b)) + 12582912.f), 0x5410);
}

// A block takes one row of each tensor per thread group.  Measured with the loads of P such passes issued at once: 47, 52 and
// 59 us at P = 1, 2 and 4 (fewer warps per SM); with blocks that walk over many rows, copied ahead to shared memory: 48 us,
// and 1 us more for the 96 tokens of a decoding step.
template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads) Kv4AppendKernel(const __grid_constant__ RowArgs a) {
  extern __shared__ float4 s_mem[];
  float* s_table = reinterpret_cast<float*>(s_mem);   // [token][cosines, sines][pairs]
  constexpr int kTpr = DIM / 8, kRows = kThreads / kTpr;
  const uint32_t row0 = blockIdx.x * uint32_t(kRows), row = row0 + threadIdx.x / kTpr;
  const uint32_t row1 = min(a.rows, row0 + uint32_t(kRows));
  const uint32_t first = QuickDiv(row0, a.div_heads);
  const bool on = row < row1;
  const uint32_t token = QuickDiv(on ? row : row0, a.div_heads);
  const int head = int((on ? row : row0) - token * uint32_t(a.c.kv_heads));
  const int in_row = threadIdx.x % kTpr, e = in_row * 8;
  union { T v[8]; uint4 w[sizeof(T) / 2]; } rk, rv;   // eight elements as loaded
  int64_t slot = -1;
  if (on) {
    slot = LoadIndex(a.slots, a.slots64, token);
    const T* kr = static_cast<const T*>(a.k) + int64_t(token) * a.kt + int64_t(head) * a.kh + e;
    const T* vr = static_cast<const T*>(a.v) + int64_t(token) * a.vt + int64_t(head) * a.vh + e;
    if (a.vec) {
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) {
        rk.w[i] = reinterpret_cast<const uint4*>(kr)[i];
        rv.w[i] = reinterpret_cast<const uint4*>(vr)[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) { rk.v[i] = kr[i]; rv.v[i] = vr[i]; }
    }
  }
  if (a.positions != nullptr) {
    const int n = int(QuickDiv(row1 - 1, a.div_heads) - first + 1) * a.pairs;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int t = QuickDiv(i, a.div_pairs), p = i - t * a.pairs;
      double s, c;
      sincospi(2.0 * TurnFraction(LoadIndex(a.positions, a.pos64, int64_t(first) + t), a.inv_freq[p]), &s, &c);
      // first and second fours of each eight in planes of their own: neighbouring threads' 16-byte reads are neighbours
      float* to = s_table + t * 2 * a.pairs + (a.eights ? ((p >> 2) & 1) * (a.pairs / 2) + (p >> 3) * 4 + (p & 3) : p);
      to[0] = float(c * double(a.mscale));
      to[a.pairs] = float(s * double(a.mscale));
    }
    __syncthreads();
  }
  uint32_t page = 0, off = 0;
  const bool keep = on && RowOf(a, slot, in_row == 0 && head == 0, &page, &off);
  float k[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { k[i] = on ? ToFloat(rk.v[i]) : 0.f; v[i] = on ? ToFloat(rv.v[i]) : 0.f; }
  if (a.positions != nullptr) {
    const float* cs = s_table + (token - first) * 2 * a.pairs;
    const float* sn = cs + a.pairs;
    if (a.interleaved) {
      if (e < 2 * a.pairs) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (e / 2 + i < a.pairs) {
            const float x = k[2 * i], y = k[2 * i + 1], c = cs[e / 2 + i], s = sn[e / 2 + i];
            k[2 * i] = x * c - y * s;
            k[2 * i + 1] = y * c + x * s;
          }
        }
      }
    } else if (a.eights) {  // the eight partners are the eight of another thread of the row
      const int far = a.pairs / 8;
      const bool turned = in_row < 2 * far, upper = in_row >= far;
      const int from = int(threadIdx.x % 32) + (turned ? (upper ? -far : far) : 0);
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, k[i], from);
      if (turned) {
        const int at = (upper ? e - a.pairs : e) / 2;
        const F2 sign = upper ? Make2(1.f, 1.f) : Make2(-1.f, -1.f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float c[4], s[4];
          LoadVec<float, 4>(cs + h * (a.pairs / 2) + at, c);
          LoadVec<float, 4>(sn + h * (a.pairs / 2) + at, s);
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const F2 x = Mul2(Make2(k[4 * h + i], k[4 * h + i + 1]), Make2(c[i], c[i + 1]));
            const F2 y = Mul2(Make2(o[4 * h + i], o[4 * h + i + 1]), Make2(s[i], s[i + 1]));
            const F2 z = Fma2(y, sign, x);
            k[4 * h + i] = X(z);
            k[4 * h + i + 1] = Y(z);
          }
        }
      }
    } else if (on) {
      const T* kr = static_cast<const T*>(a.k) + int64_t(token) * a.kt + int64_t(head) * a.kh;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (e + i < 2 * a.pairs) {
          const bool upper = e + i >= a.pairs;
          const int at = upper ? e + i - a.pairs : e + i;
          const float o = ToFloat(kr[upper ? at : at + a.pairs]);
          k[i] = upper ? k[i] * cs[at] + o * sn[at] : k[i] * cs[at] - o * sn[at];
        }
      }
    }
  }
  const int lanes = a.c.group / 8;
  __half2 kp, vp;
  const uint32_t kw = Quantize8(k, lanes, &kp), vw = Quantize8(v, lanes, &vp);
  if (keep) {
    const int64_t ci = int64_t(page) * a.c.cp + int64_t(head) * a.c.ch + int64_t(off) * a.c.ct + in_row * 4;
    *reinterpret_cast<uint32_t*>(a.c.k_codes + ci) = kw;
    *reinterpret_cast<uint32_t*>(a.c.v_codes + ci) = vw;
    if (in_row % lanes == 0) {
      const int64_t pi = int64_t(page) * a.c.pp + int64_t(head) * a.c.ph + int64_t(off) * a.c.pt + in_row / lanes;
      a.c.k_params[pi] = kp;
      a.c.v_params[pi] = vp;
    }
  }
}

template <typename T> __device__ __forceinline__ void Store8(T* row, int e, bool vec, const float (&f)[8]) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) row[e + i] = FromFloat<T>(f[i]);
  } else if constexpr (sizeof(T) == 2) {
    StoreVec<T, 8>(row + e, f);
  } else {
    const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
    StoreVec<T, 4>(row + e, lo);
    StoreVec<T, 4>(row + e + 4, hi);
  }
}

template <typename T, int DIM, int P>
__global__ void __launch_bounds__(kThreads) Kv4GatherKernel(const __grid_constant__ RowArgs a) {
  constexpr int kTpr = DIM / 8, kGroups = kThreads / kTpr, kRows = kGroups * P;
  const int in_row = threadIdx.x % kTpr, e = in_row * 8;
  const uint32_t row0 = blockIdx.x * uint32_t(kRows) + threadIdx.x / kTpr;
  uint32_t kw[P], vw[P];
  __half2 kp[P], vp[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * kGroups;
    kw[p] = vw[p] = 0u;
    kp[p] = vp[p] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
    if (row < a.rows) {
      const uint32_t token = QuickDiv(row, a.div_heads);
      const int64_t head = row - token * uint32_t(a.c.kv_heads);
      uint32_t page = 0, off = 0;
      if (RowOf(a, LoadIndex(a.slots, a.slots64, token), in_row == 0 && head == 0, &page, &off)) {
        const int64_t ci = int64_t(page) * a.c.cp + head * a.c.ch + int64_t(off) * a.c.ct + in_row * 4;
        const int64_t pi = int64_t(page) * a.c.pp + head * a.c.ph + int64_t(off) * a.c.pt + e / a.c.group;
        kw[p] = *reinterpret_cast<const uint32_t*>(a.c.k_codes + ci);
        vw[p] = *reinterpret_cast<const uint32_t*>(a.c.v_codes + ci);
        kp[p] = a.c.k_params[pi];
        vp[p] = a.c.v_params[pi];
      }
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * kGroups;
    if (row >= a.rows) break;
    const uint32_t token = QuickDiv(row, a.div_heads);
    const int64_t head = row - token * uint32_t(a.c.kv_heads);
    const float2 fk = __half22float2(kp[p]), fv = __half22float2(vp[p]);
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      k[i] = float((kw[p] >> (4 * i)) & 15u) * fk.y + fk.x;
      v[i] = float((vw[p] >> (4 * i)) & 15u) * fv.y + fv.x;
    }
    Store8<T>(static_cast<T*>(a.k) + int64_t(token) * a.kt + head * a.kh, e, a.vec, k);
    Store8<T>(static_cast<T*>(a.v) + int64_t(token) * a.vt + head * a.vh, e, a.vec, v);
  }
}

int CheckRows(const char* what, int64_t tokens, int dtype, int slots_dtype, const Kv4View& c) {
  ITEXB_REQUIRE(dtype == ITEXB_DT_FLOAT || dtype == ITEXB_DT_BFLOAT16 || dtype == ITEXB_DT_HALF, ITEXB_INVALID_ARGUMENT,
                "%s: unsupported type %s", what, DtypeName(dtype));
  ITEXB_REQUIRE(slots_dtype == ITEXB_DT_INT32 || slots_dtype == ITEXB_DT_INT64, ITEXB_INVALID_ARGUMENT, "%s: slots must be int32 or int64, got %s",
                what, DtypeName(slots_dtype));
  ITEXB_REQUIRE(tokens >= 0 && tokens <= INT_MAX / c.kv_heads, ITEXB_INVALID_ARGUMENT, "%s: bad number of tokens", what);
  return ITEXB_OK;
}
bool RowsAligned(const void* p, int64_t t, int64_t h, int esz) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (t * esz) % 16 == 0 && (h * esz) % 16 == 0;
}

template <typename T, int DIM> int LaunchAppend(const RowArgs& a, cudaStream_t st) {
  constexpr int kRows = kThreads / (DIM / 8);
  size_t smem = 0;
  if (a.positions != nullptr) smem = size_t(std::min(kRows, kRows / a.c.kv_heads + 2)) * a.pairs * sizeof(float2);
  Kv4AppendKernel<T, DIM><<<(a.rows + kRows - 1) / kRows, kThreads, smem, st>>>(a);
  return CheckLaunch("Kv4AppendKernel");
}
template <typename T, int DIM, int P> int LaunchGather(const RowArgs& a, cudaStream_t st) {
  constexpr int kRows = kThreads / (DIM / 8) * P;
  Kv4GatherKernel<T, DIM, P><<<(a.rows + kRows - 1) / kRows, kThreads, 0, st>>>(a);
  return CheckLaunch("Kv4GatherKernel");
}
template <typename T, int DIM, bool APPEND> int LaunchDim(const RowArgs& a, cudaStream_t st) {
  if constexpr (APPEND) return LaunchAppend<T, DIM>(a, st);
  // Four passes where that still gives every SM four blocks: 16384 tokens of 8 heads of 128 take 20 us, with one pass 27.
  if (a.rows >= uint32_t(kThreads / (DIM / 8)) * 4 * 148 * 4) return LaunchGather<T, DIM, 4>(a, st);
  return LaunchGather<T, DIM, 1>(a, st);
}
template <typename T, bool APPEND> int LaunchType(const RowArgs& a, cudaStream_t st) {
  if (a.c.head_dim == 64) return LaunchDim<T, 64, APPEND>(a, st);
  if (a.c.head_dim == 128) return LaunchDim<T, 128, APPEND>(a, st);
  return LaunchDim<T, 256, APPEND>(a, st);
}
template <bool APPEND> int Launch(const RowArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ITEXB_DT_FLOAT) return LaunchType<float, APPEND>(a, st);
  if (dtype == ITEXB_DT_BFLOAT16) return LaunchType<__nv_bfloat16, APPEND>(a, st);
  return LaunchType<__half, APPEND>(a, st);
}

}  // namespace
}  // namespace itexb

using namespace itexb;

extern "C" int itexb_kv4_append(const itexb_kv4_append_params_t* p, itexb_stream_t stream) {
  const char* what = "kv4_append";
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "%s: NULL params", what);
  RowArgs a{};
  ITEXB_RETURN_IF_ERROR(CheckKv4(p->cache, what, &a.c));
  ITEXB_RETURN_IF_ERROR(CheckRows(what, p->tokens, p->dtype, p->slots_dtype, a.c));
  if (p->positions != nullptr) {
    ITEXB_REQUIRE(p->positions_dtype == ITEXB_DT_INT32 || p->positions_dtype == ITEXB_DT_INT64, ITEXB_INVALID_ARGUMENT,
                  "%s: positions must be int32 or int64, got %s", what, DtypeName(p->positions_dtype));
    ITEXB_REQUIRE(p->rotary_dim >= 0 && p->rotary_dim <= p->cache.head_dim && p->rotary_dim % 2 == 0, ITEXB_INVALID_ARGUMENT,
                  "%s: rotary_dim must be even and at most head_dim, got %d", what, p->rotary_dim);
    ITEXB_REQUIRE(p->inv_freq || p->rotary_dim == 0, ITEXB_INVALID_ARGUMENT, "%s: NULL frequencies", what);
  }
  if (p->tokens == 0) return ITEXB_OK;
  ITEXB_REQUIRE(p->k && p->v && p->slots, ITEXB_INVALID_ARGUMENT, "%s: NULL tensor", what);
  a.rows = uint32_t(p->tokens * p->cache.kv_heads);
  a.div_heads = MakeFastDiv(uint32_t(p->cache.kv_heads));
  a.k = const_cast<void*>(p->k); a.kt = p->k_token_stride; a.kh = p->k_head_stride;
  a.v = const_cast<void*>(p->v); a.vt = p->v_token_stride; a.vh = p->v_head_stride;
  a.slots = p->slots;
  a.slots64 = p->slots_dtype == ITEXB_DT_INT64;
  a.positions = p->positions != nullptr && p->rotary_dim > 0 ? p->positions : nullptr;
  a.pos64 = p->positions_dtype == ITEXB_DT_INT64;
  a.inv_freq = p->inv_freq;
  a.pairs = p->rotary_dim / 2;
  a.div_pairs = MakeFastDiv(uint32_t(std::max(1, a.pairs)));
  a.interleaved = p->interleaved != 0;
  a.eights = !a.interleaved && a.pairs % 8 == 0;
  a.mscale = p->mscale;
  a.status_word = p->status_word;
  const int esz = DtypeSize(p->dtype);
  a.vec = RowsAligned(a.k, a.kt, a.kh, esz) && RowsAligned(a.v, a.vt, a.vh, esz);
  return Launch<true>(a, p->dtype, AsCuda(stream));
}

extern "C" int itexb_kv4_gather(const itexb_kv4_gather_params_t* p, itexb_stream_t stream) {
  const char* what = "kv4_gather";
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "%s: NULL params", what);
  RowArgs a{};
  ITEXB_RETURN_IF_ERROR(CheckKv4(p->cache, what, &a.c));
  ITEXB_RETURN_IF_ERROR(CheckRows(what, p->tokens, p->dtype, p->slots_dtype, a.c));
  if (p->tokens == 0) return ITEXB_OK;
  ITEXB_REQUIRE(p->k && p->v && p->slots, ITEXB_INVALID_ARGUMENT, "%s: NULL tensor", what);
  a.rows = uint32_t(p->tokens * p->cache.kv_heads);
  a.div_heads = MakeFastDiv(uint32_t(p->cache.kv_heads));
  a.k = p->k; a.kt = p->k_token_stride; a.kh = p->k_head_stride;
  a.v = p->v; a.vt = p->v_token_stride; a.vh = p->v_head_stride;
  a.slots = p->slots;
  a.slots64 = p->slots_dtype == ITEXB_DT_INT64;
  a.status_word = p->status_word;
  const int esz = DtypeSize(p->dtype);
  a.vec = RowsAligned(a.k, a.kt, a.kh, esz) && RowsAligned(a.v, a.vt, a.vh, esz);
  return Launch<false>(a, p->dtype, AsCuda(stream));
}
