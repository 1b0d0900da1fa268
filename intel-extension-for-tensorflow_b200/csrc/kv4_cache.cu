// Rows into the 4-bit paged cache (itexb_kv4_append: rotation of the keys, quantization) and back (itexb_kv4_gather).
//
//   lo = half(min of the group), step = half(max(0, (max - lo) / 15)), code = clamp(rne((x - lo) * (1 / step)), 0, 15)
//
// Both are bound by HBM (append, head_dim 128, groups of 64, bf16: 256 B in, 72 B out per row).  A thread owns 8
// consecutive elements, which are one 32-bit word of codes; the 4 - 16 threads of a group exchange minimum and maximum
// by shuffles, and the rotation of halves its partners.  Every step is a separately rounded fp32 operation on cosines and sines rounded from 64 bits, so the codes are
// those of the same formulas written with plain fp32 tensor operations.
#include <algorithm>
#include <climits>

#include "kv4.h"

namespace itexb {
namespace {

constexpr int kThreads = 256;

struct RowArgs {
  Kv4View c;
  uint32_t rows;          // tokens * kv_heads
  FastDiv div_heads;
  void* k; int64_t kt, kh;
  void* v; int64_t vt, vh;
  const void* slots;
  const void* positions;
  const double* inv_freq;
  int slots64, pos64, pairs, interleaved, vec;
  float mscale;
  int32_t* status_word;
};

__device__ __forceinline__ float MinNan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float MaxNan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

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
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { mn = MinNan(mn, x[i]); mx = MaxNan(mx, x[i]); }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    mn = MinNan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = MaxNan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const __half lo = __float2half_rn(mn);
  const float lof = __half2float(lo);
  const __half step = __float2half_rn(fmaxf((mx - lof) / 15.f, 0.f));
  const float stepf = __half2float(step);
  if (!isfinite(lof) || !isfinite(stepf)) {
    *params = __halves2half2(__ushort_as_half(0x7fff), __ushort_as_half(0x7fff));
    return 0u;
  }
  *params = __halves2half2(lo, step);
  const float inv = stepf > 0.f ? 1.f / stepf : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= uint32_t(min(max(__float2int_rn((x[i] - lof) * inv), 0), 15)) << (4 * i);
  return w;
}

// A block's rows are taken in P passes whose loads are all issued before the table is formed, as in rope.cu.
template <typename T, int DIM, int P>
__global__ void __launch_bounds__(kThreads) Kv4AppendKernel(const __grid_constant__ RowArgs a) {
  extern __shared__ float2 s_table[];
  constexpr int kTpr = DIM / 8, kGroups = kThreads / kTpr, kRows = kGroups * P;
  const uint32_t row0 = blockIdx.x * uint32_t(kRows);
  const uint32_t row1 = min(a.rows, row0 + uint32_t(kRows));
  const uint32_t first = QuickDiv(row0, a.div_heads);
  const int in_row = threadIdx.x % kTpr, e = in_row * 8;
  union Raw { T v[8]; uint4 w[sizeof(T) / 2]; };   // eight elements as loaded
  Raw rk[P], rv[P];
  int64_t slot[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * kGroups + threadIdx.x / kTpr;
    slot[p] = -1;
    if (row < row1) {
      const uint32_t token = QuickDiv(row, a.div_heads);
      const int64_t head = row - token * uint32_t(a.c.kv_heads);
      slot[p] = LoadIndex(a.slots, a.slots64, token);
      const T* kr = static_cast<const T*>(a.k) + int64_t(token) * a.kt + head * a.kh + e;
      const T* vr = static_cast<const T*>(a.v) + int64_t(token) * a.vt + head * a.vh + e;
      if (a.vec) {
#pragma unroll
        for (int i = 0; i < int(sizeof(T) / 2); ++i) {
          rk[p].w[i] = reinterpret_cast<const uint4*>(kr)[i];
          rv[p].w[i] = reinterpret_cast<const uint4*>(vr)[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) { rk[p].v[i] = kr[i]; rv[p].v[i] = vr[i]; }
      }
    }
  }
  if (a.positions != nullptr) {
    const int n = int(QuickDiv(row1 - 1, a.div_heads) - first + 1) * a.pairs;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int t = i / a.pairs, p = i - t * a.pairs;
      double s, c;
      sincospi(2.0 * TurnFraction(LoadIndex(a.positions, a.pos64, int64_t(first) + t), a.inv_freq[p]), &s, &c);
      s_table[i] = make_float2(float(c * double(a.mscale)), float(s * double(a.mscale)));
    }
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * kGroups + threadIdx.x / kTpr;
    if (P > 1 && row0 + p * kGroups >= row1) break;
    const bool on = row < row1;
    const uint32_t token = QuickDiv(on ? row : row0, a.div_heads);
    const int head = int((on ? row : row0) - token * uint32_t(a.c.kv_heads));
    uint32_t page = 0, off = 0;
    const bool keep = on && RowOf(a, slot[p], in_row == 0 && head == 0, &page, &off);
    float k[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { k[i] = on ? ToFloat(rk[p].v[i]) : 0.f; v[i] = on ? ToFloat(rv[p].v[i]) : 0.f; }
    if (a.positions != nullptr) {
      const float2* cs = s_table + (token - first) * a.pairs;
      if (a.interleaved) {
        if (e < 2 * a.pairs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (e / 2 + i < a.pairs) {
              const float2 q = cs[e / 2 + i];
              const float x = k[2 * i], y = k[2 * i + 1];
              k[2 * i] = x * q.x - y * q.y;
              k[2 * i + 1] = y * q.x + x * q.y;
            }
          }
        }
      } else if (a.pairs % 8 == 0) {  // the eight partners are the eight of another thread of the row
        const int far = a.pairs / 8;
        const bool turned = in_row < 2 * far, upper = in_row >= far;
        const int from = int(threadIdx.x % 32) + (turned ? (upper ? -far : far) : 0);
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, k[i], from);
        if (turned) {
          const float2* q = cs + (upper ? e - a.pairs : e);
#pragma unroll
          for (int i = 0; i < 8; ++i) k[i] = upper ? k[i] * q[i].x + o[i] * q[i].y : k[i] * q[i].x - o[i] * q[i].y;
        }
      } else if (on) {
        const T* kr = static_cast<const T*>(a.k) + int64_t(token) * a.kt + int64_t(head) * a.kh;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (e + i < 2 * a.pairs) {
            const bool upper = e + i >= a.pairs;
            const int at = upper ? e + i - a.pairs : e + i;
            const float o = ToFloat(kr[upper ? at : at + a.pairs]);
            k[i] = upper ? k[i] * cs[at].x + o * cs[at].y : k[i] * cs[at].x - o * cs[at].y;
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

template <typename T, int DIM, int P, bool APPEND> int LaunchPasses(const RowArgs& a, cudaStream_t st) {
  constexpr int kRows = kThreads / (DIM / 8) * P;
  const unsigned blocks = (a.rows + kRows - 1) / kRows;
  if (APPEND) {
    size_t smem = 0;
    if (a.positions != nullptr) smem = size_t(std::min(kRows, kRows / a.c.kv_heads + 2)) * a.pairs * sizeof(float2);
    Kv4AppendKernel<T, DIM, P><<<blocks, kThreads, smem, st>>>(a);
    return CheckLaunch("Kv4AppendKernel");
  }
  Kv4GatherKernel<T, DIM, P><<<blocks, kThreads, 0, st>>>(a);
  return CheckLaunch("Kv4GatherKernel");
}
template <typename T, int DIM, bool APPEND> int LaunchDim(const RowArgs& a, cudaStream_t st) {
  // four passes where that still gives every SM four blocks
  constexpr int kPasses = APPEND ? 1 : 4;
  if (kPasses > 1 && a.rows >= uint32_t(kThreads / (DIM / 8)) * kPasses * 148 * 4) return LaunchPasses<T, DIM, kPasses, APPEND>(a, st);
  return LaunchPasses<T, DIM, 1, APPEND>(a, st);
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
  a.interleaved = p->interleaved != 0;
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
