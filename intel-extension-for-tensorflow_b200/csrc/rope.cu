// Rotary positions of queries and keys, alone (itexb_rope) or after a root-mean-square norm of each head
// (itexb_qk_norm_rope), and that one's gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps);  y = R(angle) (x r w)          R: rotation of pairs times mscale, identity behind it
//   gradient:  t = R^T g;  dw = sum t x r;  u = t w;  dx = r (u - x r mean(u x r))
//
// All three are bound by HBM: two (three) times the tensor's bytes, a handful of operations per element.  A row (one
// head of one token) is spread over the 4 - 32 threads that hold it in 16-byte pieces; each thread owns both elements of
// its pairs, so nothing is exchanged for the rotation and a call may work in place.  The angles do not depend on the
// head: a block takes consecutive rows and forms the cosines and sines of its few tokens once, in shared memory.
#include <algorithm>
#include <climits>

#include "decoder.h"

namespace itexb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxGradBlocks = 296;  // per side; partial weight gradients: four blocks per SM of a 148-SM device for both
enum { kRope = 0, kNorm = 1, kGrad = 2 };

struct Side {  // queries or keys
  const void* x; int64_t xt, xh;
  void* y; int64_t yt, yh;
  const void* g; int64_t gt, gh;
  const void* w;
  void* dw;
};
struct RopeArgs {
  Side side[2];
  int heads[2];
  FastDiv div_heads;      // kRope / kNorm: by q_heads + k_heads; kGrad: see div_side
  FastDiv div_side[2];
  uint32_t rows;          // kRope / kNorm: tokens * (q_heads + k_heads)
  int64_t tokens;
  int head_dim, pairs, items, tpr, rows_per_block, block_tokens;
  int interleaved, pos64, w_dtype;
  float mscale, sin_sign, eps;
  const void* positions;
  const double* inv_freq;
  float* partial;         // kGrad: [2][blocks][head_dim]
};

__device__ __forceinline__ float LoadW(const void* w, int dt, int i) {
  return dt == ITEXB_DT_FLOAT ? static_cast<const float*>(w)[i]
         : dt == ITEXB_DT_BFLOAT16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : __half2float(static_cast<const __half*>(w)[i]);
}

// cos, sin (times mscale) of the tokens of rows [row0, row1) -> table[token - first][pair]
__device__ __forceinline__ void FillTable(float2* table, const RopeArgs& a, uint32_t first, uint32_t tokens) {
  const int n = int(tokens) * a.pairs;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const double frac = TurnFraction(LoadIndex(a.positions, a.pos64, int64_t(first) + t), a.inv_freq[p]);
    float s, c;
    sincospif(2.f * float(frac), &s, &c);
    table[i] = make_float2(c * a.mscale, s * a.mscale * a.sin_sign);
  }
}

// Rotates one item: `u`, `v` are its two VEC-element pieces, `cs` the table entries of its first pair.
template <int VEC> __device__ __forceinline__ void Turn(float (&u)[VEC], float (&v)[VEC], const float2* cs, bool interleaved) {
  if (VEC > 1 && interleaved) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 p = cs[i], q = cs[VEC / 2 + i];
      const float a = u[2 * i], b = u[2 * i + 1], c = v[2 * i], d = v[2 * i + 1];
      u[2 * i] = a * p.x - b * p.y; u[2 * i + 1] = b * p.x + a * p.y;
      v[2 * i] = c * q.x - d * q.y; v[2 * i + 1] = d * q.x + c * q.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float2 p = cs[i];
      const float a = u[i], b = v[i];
      u[i] = a * p.x - b * p.y; v[i] = b * p.x + a * p.y;
    }
  }
}

// Item j of a row: its pieces start at elements o0 and o1; the first pairs / VEC items are rotated.
struct Item { int o0, o1; bool turned; };
template <int VEC> __device__ __forceinline__ Item ItemOf(int j, const RopeArgs& a) {
  const int nt = a.pairs / VEC;
  if (j < nt && !a.interleaved) return {j * VEC, a.pairs + j * VEC, true};
  return {2 * VEC * j, 2 * VEC * j + VEC, j < nt};   // interleaved pairs, or the elements behind the rotated ones
}

// The weights as fp32 in shared memory: [queries, keys][head_dim].
__device__ __forceinline__ void FillWeights(float* w, const RopeArgs& a) {
  for (int i = threadIdx.x; i < 2 * a.head_dim; i += kThreads) {
    const int side = i >= a.head_dim;
    if (a.side[side].w != nullptr) w[i] = LoadW(a.side[side].w, a.w_dtype, i - side * a.head_dim);
  }
}
template <int VEC> __device__ __forceinline__ void TimesWeights(float (&u)[VEC], float (&v)[VEC], const float* w, const Item& it) {
  float p[VEC], q[VEC];
  LoadVec<float, VEC>(w + it.o0, p);
  LoadVec<float, VEC>(w + it.o1, q);
#pragma unroll
  for (int i = 0; i < VEC; ++i) { u[i] *= p[i]; v[i] *= q[i]; }
}

// A thread's pieces of one row, as loaded.
template <typename T, int VEC, int NI> struct Pieces {
  Vec<T, VEC> u[NI], v[NI];
  __device__ __forceinline__ void Load(const T* x, int in_row, bool on, const RopeArgs& a) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int j = in_row + n * a.tpr;
      if (on && j < a.items) {
        const Item it = ItemOf<VEC>(j, a);
        u[n] = *reinterpret_cast<const Vec<T, VEC>*>(x + it.o0);
        v[n] = *reinterpret_cast<const Vec<T, VEC>*>(x + it.o1);
      }
    }
  }
  __device__ __forceinline__ void Floats(int n, float (&fu)[VEC], float (&fv)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { fu[i] = ToFloat(u[n].v[i]); fv[i] = ToFloat(v[n].v[i]); }
  }
};

// A block's rows are taken in P passes whose loads are all issued before the table is formed: long calls keep 4 x 32 bytes
// per thread in flight (norms and rotation of 8192 tokens, 168 MB: 55 us with one pass per block).  Short ones take one pass
// per block and so reach more SMs.
template <typename T, int VEC, int NI, int MODE, int P>
__global__ void __launch_bounds__(kThreads) RopeKernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float4 s_mem[];
  float* s_w = reinterpret_cast<float*>(s_mem);                              // kNorm
  float2* s_table = reinterpret_cast<float2*>(s_w + (MODE == kNorm ? 2 * a.head_dim : 0));
  const int group = threadIdx.x / a.tpr, in_row = threadIdx.x - group * a.tpr;
  const int groups = kThreads / a.tpr;
  const uint32_t row0 = blockIdx.x * uint32_t(a.rows_per_block);
  const uint32_t row1 = min(a.rows, row0 + uint32_t(a.rows_per_block));
  const uint32_t first = QuickDiv(row0, a.div_heads);
  const uint32_t heads = uint32_t(a.heads[0] + a.heads[1]);
  Pieces<T, VEC, NI> x[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * groups + group;
    if (row < row1) {
      const uint32_t token = QuickDiv(row, a.div_heads);
      const int head = int(row - token * heads);
      const int is_k = head >= a.heads[0];
      const Side& s = a.side[is_k];
      x[p].Load(static_cast<const T*>(s.x) + int64_t(token) * s.xt + int64_t(head - (is_k ? a.heads[0] : 0)) * s.xh, in_row, true, a);
    }
  }
  FillTable(s_table, a, first, QuickDiv(row1 - 1, a.div_heads) - first + 1);
  if (MODE == kNorm) FillWeights(s_w, a);
  __syncthreads();
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t row = row0 + p * groups + group;
    const bool on = row < row1;
    if (P > 1 && row0 + p * groups >= row1) break;
    const uint32_t token = QuickDiv(on ? row : row0, a.div_heads);
    const int head = int((on ? row : row0) - token * heads);
    const int is_k = head >= a.heads[0];
    const Side& s = a.side[is_k];
    float r = 1.f;
    if (MODE == kNorm) {
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if (on && in_row + n * a.tpr < a.items) {
          float u[VEC], v[VEC];
          x[p].Floats(n, u, v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum = fmaf(u[i], u[i], fmaf(v[i], v[i], sum));
        }
      }
      for (int o = a.tpr >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = rsqrtf(sum / float(a.head_dim) + a.eps);
    }
    T* y = static_cast<T*>(s.y) + int64_t(token) * s.yt + int64_t(head - (is_k ? a.heads[0] : 0)) * s.yh;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int j = in_row + n * a.tpr;
      if (on && j < a.items) {
        const Item it = ItemOf<VEC>(j, a);
        float u[VEC], v[VEC];
        x[p].Floats(n, u, v);
        if (MODE == kNorm) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) { u[i] *= r; v[i] *= r; }
          TimesWeights<VEC>(u, v, s_w + is_k * a.head_dim, it);
        }
        if (it.turned) Turn<VEC>(u, v, s_table + (token - first) * a.pairs + j * VEC, a.interleaved);
        StoreVec<T, VEC>(y + it.o0, u);
        StoreVec<T, VEC>(y + it.o1, v);
      }
    }
  }
}

// blockIdx.y chooses queries or keys; blocks walk the row tiles with a fixed stride, so the partial sums of the weight
// gradient, and with them its bits, depend on the shape alone.  The next tile's loads are issued before this one's work.
template <typename T, int VEC, int NI>
__global__ void __launch_bounds__(kThreads) NormRopeGradKernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float4 s_mem[];
  float* s_w = reinterpret_cast<float*>(s_mem);
  float2* s_table = reinterpret_cast<float2*>(s_w + 2 * a.head_dim);
  const int which = blockIdx.y;
  const Side& s = a.side[which];
  const uint32_t heads = uint32_t(a.heads[which]);
  const uint32_t rows = uint32_t(a.tokens) * heads;
  const int group = threadIdx.x / a.tpr, in_row = threadIdx.x - group * a.tpr;
  const int groups = kThreads / a.tpr;
  const uint32_t stride = gridDim.x * uint32_t(groups);
  float du[NI][VEC], dv[NI][VEC];
#pragma unroll
  for (int n = 0; n < NI; ++n)
#pragma unroll
    for (int i = 0; i < VEC; ++i) du[n][i] = dv[n][i] = 0.f;
  FillWeights(s_w, a);
  Pieces<T, VEC, NI> x, g;
  auto load = [&](uint32_t row) {
    if (row < rows) {
      const uint32_t token = QuickDiv(row, a.div_side[which]);
      const int64_t h = row - token * heads;
      x.Load(static_cast<const T*>(s.x) + int64_t(token) * s.xt + h * s.xh, in_row, true, a);
      g.Load(static_cast<const T*>(s.g) + int64_t(token) * s.gt + h * s.gh, in_row, true, a);
    }
  };
  load(blockIdx.x * uint32_t(groups) + group);
  for (uint32_t row0 = blockIdx.x * uint32_t(groups); row0 < rows; row0 += stride) {
    const uint32_t row1 = min(rows, row0 + uint32_t(groups));
    const uint32_t first = QuickDiv(row0, a.div_side[which]);
    __syncthreads();
    FillTable(s_table, a, first, QuickDiv(row1 - 1, a.div_side[which]) - first + 1);
    __syncthreads();
    const uint32_t row = row0 + group;
    const bool on = row < row1;
    const uint32_t token = QuickDiv(on ? row : row0, a.div_side[which]);
    const int64_t h = (on ? row : row0) - token * heads;
    T* y = static_cast<T*>(s.y) + int64_t(token) * s.yt + h * s.yh;
    const Pieces<T, VEC, NI> cx = x, cg = g;
    load(row + stride);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if (on && in_row + n * a.tpr < a.items) {
        float u[VEC], v[VEC];
        cx.Floats(n, u, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum = fmaf(u[i], u[i], fmaf(v[i], v[i], sum));
      }
    }
    for (int o = a.tpr >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float r = rsqrtf(sum / float(a.head_dim) + a.eps);
    float gu[NI][VEC], gv[NI][VEC];
    float dot = 0.f;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int j = in_row + n * a.tpr;
      if (on && j < a.items) {
        const Item it = ItemOf<VEC>(j, a);
        float u[VEC], v[VEC];
        cx.Floats(n, u, v);
        cg.Floats(n, gu[n], gv[n]);
        if (it.turned) Turn<VEC>(gu[n], gv[n], s_table + (token - first) * a.pairs + j * VEC, a.interleaved);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          u[i] *= r;
          v[i] *= r;
          du[n][i] = fmaf(gu[n][i], u[i], du[n][i]);
          dv[n][i] = fmaf(gv[n][i], v[i], dv[n][i]);
        }
        TimesWeights<VEC>(gu[n], gv[n], s_w + which * a.head_dim, it);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dot = fmaf(gu[n][i], u[i], fmaf(gv[n][i], v[i], dot));
      }
    }
    for (int o = a.tpr >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    dot /= float(a.head_dim);
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int j = in_row + n * a.tpr;
      if (on && j < a.items) {
        const Item it = ItemOf<VEC>(j, a);
        float u[VEC], v[VEC];
        cx.Floats(n, u, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          gu[n][i] = r * (gu[n][i] - u[i] * r * dot);
          gv[n][i] = r * (gv[n][i] - v[i] * r * dot);
        }
        StoreVec<T, VEC>(y + it.o0, gu[n]);
        StoreVec<T, VEC>(y + it.o1, gv[n]);
      }
    }
  }
  // the block's partial sums: rows of one position in the row tile are added in the order of their thread groups
  __syncthreads();
  float* acc = reinterpret_cast<float*>(s_mem);  // [groups][head_dim]
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int j = in_row + n * a.tpr;
    if (j < a.items) {
      const Item it = ItemOf<VEC>(j, a);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        acc[group * a.head_dim + it.o0 + i] = du[n][i];
        acc[group * a.head_dim + it.o1 + i] = dv[n][i];
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.head_dim; c += kThreads) {
    float sum = 0.f;
    for (int i = 0; i < groups; ++i) sum += acc[i * a.head_dim + c];
    a.partial[(size_t(which) * gridDim.x + blockIdx.x) * a.head_dim + c] = sum;
  }
}

// Column sums of the partial weight gradients, in 64 bits: 32 columns a block, 32 warps that take up to 10 terms each.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) WeightGradKernel(const __grid_constant__ RopeArgs a, int blocks) {
  __shared__ double s_sum[kSumThreads / 32][33];
  const int which = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double sum = 0.0;
  if (c < a.head_dim)
#pragma unroll 10
    for (int b = warp; b < blocks; b += kSumThreads / 32) sum += double(a.partial[(size_t(which) * blocks + b) * a.head_dim + c]);
  s_sum[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && c < a.head_dim) {
    for (int w = 1; w < kSumThreads / 32; ++w) sum += s_sum[w][lane];
    void* dw = a.side[which].dw;
    if (a.w_dtype == ITEXB_DT_FLOAT) static_cast<float*>(dw)[c] = float(sum);
    else if (a.w_dtype == ITEXB_DT_BFLOAT16) static_cast<__nv_bfloat16*>(dw)[c] = __double2bfloat16(sum);
    else static_cast<__half*>(dw)[c] = __double2half(sum);
  }
}

bool Fits(const void* p, int64_t st, int64_t sh, int esz, int vec) {
  const int64_t b = int64_t(esz) * vec;
  return reinterpret_cast<uintptr_t>(p) % size_t(b) == 0 && (st * esz) % b == 0 && (sh * esz) % b == 0;
}

int CheckRope(const itexb_rope_params_t* p, const char* what) {
  ITEXB_REQUIRE(p->dtype == ITEXB_DT_FLOAT || p->dtype == ITEXB_DT_BFLOAT16 || p->dtype == ITEXB_DT_HALF, ITEXB_INVALID_ARGUMENT,
                "%s: unsupported type %s", what, DtypeName(p->dtype));
  ITEXB_REQUIRE(p->positions_dtype == ITEXB_DT_INT32 || p->positions_dtype == ITEXB_DT_INT64, ITEXB_INVALID_ARGUMENT,
                "%s: positions must be int32 or int64, got %s", what, DtypeName(p->positions_dtype));
  ITEXB_REQUIRE(p->tokens >= 0 && p->q_heads > 0 && p->k_heads >= 0, ITEXB_INVALID_ARGUMENT, "%s: bad shape", what);
  ITEXB_REQUIRE(p->head_dim >= 2 && p->head_dim <= 512 && p->head_dim % 2 == 0, ITEXB_INVALID_ARGUMENT,
                "%s: head_dim must be even and at most 512, got %d", what, p->head_dim);
  ITEXB_REQUIRE(p->rotary_dim >= 0 && p->rotary_dim <= p->head_dim && p->rotary_dim % 2 == 0, ITEXB_INVALID_ARGUMENT,
                "%s: rotary_dim must be even and at most head_dim, got %d", what, p->rotary_dim);
  ITEXB_REQUIRE(p->tokens <= INT_MAX / (int64_t(p->q_heads) + p->k_heads), ITEXB_INVALID_ARGUMENT, "%s: 2^31 rows or more", what);
  if (p->tokens == 0) return ITEXB_OK;
  ITEXB_REQUIRE(p->q && p->q_out && (p->k_heads == 0 || (p->k && p->k_out)), ITEXB_INVALID_ARGUMENT, "%s: NULL tensor", what);
  ITEXB_REQUIRE(p->positions && (p->inv_freq || p->rotary_dim == 0), ITEXB_INVALID_ARGUMENT, "%s: NULL positions or frequencies", what);
  return ITEXB_OK;
}

void Fill(RopeArgs& a, const itexb_rope_params_t* p) {
  a.side[0] = {p->q, p->q_token_stride, p->q_head_stride, p->q_out, p->q_out_token_stride, p->q_out_head_stride, nullptr, 0, 0, nullptr, nullptr};
  a.side[1] = {p->k, p->k_token_stride, p->k_head_stride, p->k_out, p->k_out_token_stride, p->k_out_head_stride, nullptr, 0, 0, nullptr, nullptr};
  a.heads[0] = p->q_heads;
  a.heads[1] = p->k_heads;
  a.tokens = p->tokens;
  a.rows = uint32_t(p->tokens * (p->q_heads + p->k_heads));
  a.div_heads = MakeFastDiv(uint32_t(p->q_heads + p->k_heads));
  a.div_side[0] = MakeFastDiv(uint32_t(p->q_heads));
  a.div_side[1] = MakeFastDiv(uint32_t(std::max(1, p->k_heads)));
  a.head_dim = p->head_dim;
  a.pairs = p->rotary_dim / 2;
  a.interleaved = p->interleaved != 0;
  a.pos64 = p->positions_dtype == ITEXB_DT_INT64;
  a.mscale = p->mscale;
  a.sin_sign = p->inverse ? -1.f : 1.f;
  a.positions = p->positions;
  a.inv_freq = p->inv_freq;
}

// The widest piece (16 bytes, 4 elements, one) that divides the row's parts and its addresses.
int PickVec(const RopeArgs& a, int esz, bool grad) {
  for (int vec : {16 / esz, 4}) {
    if (a.pairs % vec != 0 || (a.head_dim / 2 - a.pairs) % vec != 0) continue;
    bool ok = true;
    for (int i = 0; i < (a.heads[1] > 0 ? 2 : 1); ++i) {
      const Side& s = a.side[i];
      ok = ok && Fits(s.x, s.xt, s.xh, esz, vec) && Fits(s.y, s.yt, s.yh, esz, vec) && (!grad || Fits(s.g, s.gt, s.gh, esz, vec));
    }
    if (ok) return vec;
  }
  return 1;
}

int GradBlocks(int64_t tokens, int q_heads, int k_heads, int rows_per_block) {
  const int64_t most = tokens * std::max(q_heads, k_heads);
  return int(std::max<int64_t>(1, std::min<int64_t>(kMaxGradBlocks, (most + rows_per_block - 1) / rows_per_block)));
}

template <typename T, int VEC, int NI, int MODE, int P> int RunPasses(RopeArgs& a, size_t weights, cudaStream_t st) {
  const int heads = a.heads[0] + a.heads[1];
  a.rows_per_block = kThreads / a.tpr * P;
  const size_t smem = weights + size_t(std::min(a.rows_per_block, a.rows_per_block / heads + 2)) * a.pairs * sizeof(float2);
  auto kernel = RopeKernel<T, VEC, NI, MODE, P>;
  if (smem > 48 * 1024) ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  kernel<<<(a.rows + a.rows_per_block - 1) / a.rows_per_block, kThreads, smem, st>>>(a);
  return CheckLaunch("RopeKernel");
}

template <typename T, int VEC, int NI, int MODE> int Run(RopeArgs& a, cudaStream_t st) {
  a.items = a.head_dim / (2 * VEC);
  a.tpr = 1;
  while (a.tpr < 32 && a.tpr < a.items) a.tpr *= 2;
  const int groups = kThreads / a.tpr;
  const size_t weights = size_t(2) * a.head_dim * sizeof(float);
  if constexpr (MODE == kGrad) {
    const int least = std::min(a.heads[0], a.heads[1] > 0 ? a.heads[1] : a.heads[0]);
    const size_t smem = std::max(weights + size_t(std::min(groups, groups / least + 2)) * a.pairs * sizeof(float2), size_t(groups) * a.head_dim * sizeof(float));
    auto kernel = NormRopeGradKernel<T, VEC, NI>;
    if (smem > 48 * 1024) ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    const int sides = a.heads[1] > 0 ? 2 : 1;
    const int blocks = GradBlocks(a.tokens, a.heads[0], a.heads[1], groups);
    kernel<<<dim3(blocks, sides), kThreads, smem, st>>>(a);
    ITEXB_RETURN_IF_ERROR(CheckLaunch("NormRopeGradKernel"));
    WeightGradKernel<<<dim3((a.head_dim + 31) / 32, sides), kSumThreads, 0, st>>>(a, blocks);
    return CheckLaunch("WeightGradKernel");
  } else {
    // four passes where that still gives every SM four blocks, and where the pieces fit the registers
    constexpr int kPasses = NI == 1 && MODE == kRope ? 4 : 1;
    if (kPasses > 1 && a.rows >= uint32_t(groups) * kPasses * 148 * 4) return RunPasses<T, VEC, NI, MODE, kPasses>(a, MODE == kNorm ? weights : 0, st);
    return RunPasses<T, VEC, NI, MODE, 1>(a, MODE == kNorm ? weights : 0, st);
  }
}

template <typename T, int MODE> int Pick(RopeArgs& a, cudaStream_t st) {
  const int vec = PickVec(a, sizeof(T), MODE == kGrad);
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return Run<T, 8, 1, MODE>(a, st);
  }
  if (vec == 4) return a.head_dim <= 256 ? Run<T, 4, 1, MODE>(a, st) : Run<T, 4, 2, MODE>(a, st);
  return Run<T, 1, 8, MODE>(a, st);
}
template <int MODE> int Dispatch(RopeArgs& a, int dtype, cudaStream_t st) {
  if (dtype == ITEXB_DT_FLOAT) return Pick<float, MODE>(a, st);
  if (dtype == ITEXB_DT_BFLOAT16) return Pick<__nv_bfloat16, MODE>(a, st);
  return Pick<__half, MODE>(a, st);
}

int CheckNorm(const itexb_qk_norm_rope_params_t* p, const char* what) {
  ITEXB_RETURN_IF_ERROR(CheckRope(&p->r, what));
  ITEXB_REQUIRE(p->w_dtype == ITEXB_DT_FLOAT || p->w_dtype == ITEXB_DT_BFLOAT16 || p->w_dtype == ITEXB_DT_HALF, ITEXB_INVALID_ARGUMENT,
                "%s: unsupported weight type %s", what, DtypeName(p->w_dtype));
  ITEXB_REQUIRE(p->r.inverse == 0, ITEXB_INVALID_ARGUMENT, "%s: inverse does not apply", what);
  ITEXB_REQUIRE(p->epsilon >= 0.f, ITEXB_INVALID_ARGUMENT, "%s: epsilon must not be negative", what);
  ITEXB_REQUIRE(p->q_weight && (p->r.k_heads == 0 || p->k_weight), ITEXB_INVALID_ARGUMENT, "%s: NULL weight", what);
  return ITEXB_OK;
}

}  // namespace
}  // namespace itexb

using namespace itexb;

extern "C" int itexb_rope(const itexb_rope_params_t* p, itexb_stream_t stream) {
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "rope: NULL params");
  ITEXB_RETURN_IF_ERROR(CheckRope(p, "rope"));
  if (p->tokens == 0) return ITEXB_OK;
  RopeArgs a{};
  Fill(a, p);
  return Dispatch<kRope>(a, p->dtype, AsCuda(stream));
}

extern "C" int itexb_qk_norm_rope(const itexb_qk_norm_rope_params_t* p, itexb_stream_t stream) {
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "qk_norm_rope: NULL params");
  ITEXB_RETURN_IF_ERROR(CheckNorm(p, "qk_norm_rope"));
  if (p->r.tokens == 0) return ITEXB_OK;
  RopeArgs a{};
  Fill(a, &p->r);
  a.side[0].w = p->q_weight;
  a.side[1].w = p->k_weight;
  a.w_dtype = p->w_dtype;
  a.eps = p->epsilon;
  return Dispatch<kNorm>(a, p->r.dtype, AsCuda(stream));
}

extern "C" size_t itexb_qk_norm_rope_grad_workspace_bytes(int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t head_dim) {
  if (tokens <= 0 || q_heads <= 0 || k_heads < 0 || head_dim <= 0) return 0;
  return size_t(2) * size_t(GradBlocks(tokens, q_heads, k_heads, 1)) * size_t(head_dim) * sizeof(float);
}

extern "C" int itexb_qk_norm_rope_grad(const itexb_qk_norm_rope_grad_params_t* p, itexb_stream_t stream) {
  const char* what = "qk_norm_rope_grad";
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "%s: NULL params", what);
  const itexb_qk_norm_rope_params_t& n = p->n;
  ITEXB_RETURN_IF_ERROR(CheckNorm(&n, what));
  ITEXB_REQUIRE(p->d_q_weight && (n.r.k_heads == 0 || p->d_k_weight), ITEXB_INVALID_ARGUMENT, "%s: NULL weight gradient", what);
  cudaStream_t st = AsCuda(stream);
  if (n.r.tokens == 0) {  // sums over nothing
    const size_t bytes = size_t(n.r.head_dim) * DtypeSize(n.w_dtype);
    ITEXB_CUDA(cudaMemsetAsync(p->d_q_weight, 0, bytes, st));
    if (n.r.k_heads > 0) ITEXB_CUDA(cudaMemsetAsync(p->d_k_weight, 0, bytes, st));
    return ITEXB_OK;
  }
  ITEXB_REQUIRE(p->q_grad && (n.r.k_heads == 0 || p->k_grad) && p->workspace, ITEXB_INVALID_ARGUMENT, "%s: NULL gradient or workspace", what);
  RopeArgs a{};
  Fill(a, &n.r);
  a.sin_sign = -1.f;  // the rotation's transpose
  a.side[0].w = n.q_weight;
  a.side[1].w = n.k_weight;
  a.side[0].dw = p->d_q_weight;
  a.side[1].dw = p->d_k_weight;
  a.side[0].g = p->q_grad; a.side[0].gt = p->q_grad_token_stride; a.side[0].gh = p->q_grad_head_stride;
  a.side[1].g = p->k_grad; a.side[1].gt = p->k_grad_token_stride; a.side[1].gh = p->k_grad_head_stride;
  a.w_dtype = n.w_dtype;
  a.eps = n.epsilon;
  a.partial = static_cast<float*>(p->workspace);
  return Dispatch<kGrad>(a, n.r.dtype, st);
}
