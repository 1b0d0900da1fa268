// Rotary positions of queries and keys, alone (itexb_rope) or after a root-mean-square norm of each head
// (itexb_qk_norm_rope), and that one's gradient.
//
//   r = 1 / sqrt(mean(x^2) + eps);  y = R(angle) (x r w)          R: rotation of pairs times mscale, identity behind it
//   gradient:  t = R^T g;  dw = sum t x r;  u = t w;  dx = r (u - x r mean(u x r))
//
// All three are bound by HBM: two (three) times the tensor's bytes, a handful of operations per element.  A row (one
// head of one token) is spread over the 4 - 32 threads that hold it in 16-byte pieces; each thread owns both elements of
// its pairs, so nothing is exchanged for the rotation and a call may work in place.  The angles do not depend on the
// head: a block takes consecutive tokens, forms their cosines and sines once in shared memory and walks over their rows,
// with the next four rows per thread on their way to shared memory (gradient: two of each tensor).  At 4 x 16 KB per block
// that keeps ~100 KB in flight on an SM with a third of the registers that loads to registers would take.
// Measured: rotation of 16384 tokens, 32 + 8 heads of 128, fp16 (336 MB), 58 us, 5.8 TB/s; norms and rotation of 8192 such
// tokens, bf16 (168 MB), 37 us, 4.5 TB/s (53 us when every block formed tables and weights for 32 rows); the gradient of
// 6143 tokens with 16 + 16 heads of 64, bf16 (76 MB), 23 us + 4 us for the sums of the weights' gradients.
#include <algorithm>
#include <climits>

#include "decoder.h"

namespace itexb {
namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;
constexpr int kPerSm = 3;              // blocks on an SM at a time (4, with fewer registers, measured the same)
constexpr int kGradBlocks = 2 * kSms;
constexpr int kTableBytes = 32 * 1024; // cosines and sines of a block's tokens
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
  FastDiv div_heads;      // by q_heads + k_heads
  FastDiv div_side[2];    // by q_heads, by k_heads
  FastDiv div_pairs;
  int64_t tokens;
  int head_dim, pairs, items, tpr, table_tokens;
  int interleaved, pos64, w_dtype;
  float mscale, sin_sign, eps, inv_dim;
  const void* positions;
  const double* inv_freq;
  float* partial;         // kGrad: [2][blocks][head_dim]
};

__device__ __forceinline__ float LoadW(const void* w, int dt, int i) {
  return dt == ITEXB_DT_FLOAT ? static_cast<const float*>(w)[i]
         : dt == ITEXB_DT_BFLOAT16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : __half2float(static_cast<const __half*>(w)[i]);
}

// Place of element i of a vector that threads read in pieces of VEC floats: for pieces of 8 all first halves lie before all
// second halves, so that the 16-byte reads of neighbouring threads are neighbours too (no bank conflicts).
template <int VEC> __device__ __forceinline__ int Plane(int i, int n) { return VEC == 8 ? ((i >> 2) & 1) * (n / 2) + (i >> 3) * 4 + (i & 3) : i; }
template <int VEC> __device__ __forceinline__ void LoadPlane(const float* v, int i, int n, float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    float lo[4], hi[4];
    LoadVec<float, 4>(v + (i >> 1), lo);
    LoadVec<float, 4>(v + n / 2 + (i >> 1), hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) { f[k] = lo[k]; f[4 + k] = hi[k]; }
  } else {
    LoadVec<float, VEC>(v + i, f);
  }
}

// cos and sin (times mscale) of `tokens` tokens from `first` on -> cs[token][2][pair]
template <int VEC> __device__ __forceinline__ void FillTable(float* cs, const RopeArgs& a, uint32_t first, uint32_t tokens) {
  const int n = int(tokens) * a.pairs;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = QuickDiv(i, a.div_pairs), p = i - t * a.pairs;
    const double frac = TurnFraction(LoadIndex(a.positions, a.pos64, int64_t(first) + t), a.inv_freq[p]);
    float s, c;
    sincospif(2.f * float(frac), &s, &c);
    float* to = cs + t * 2 * a.pairs + (a.interleaved ? p : Plane<VEC>(p, a.pairs));
    to[0] = c * a.mscale;
    to[a.pairs] = s * a.mscale * a.sin_sign;
  }
}

// Rotates item j of a token with the cosines and sines `cs`.
template <int VEC> __device__ __forceinline__ void Turn(float (&u)[VEC], float (&v)[VEC], const float* cs, int j, const RopeArgs& a) {
  if constexpr (VEC == 1) {
    const float x = u[0], y = v[0], c = cs[j], s = cs[a.pairs + j];
    u[0] = x * c - y * s;
    v[0] = y * c + x * s;
  } else if (a.interleaved) {   // each piece holds whole pairs
    constexpr int H = VEC / 2;
    float c[2][H], s[2][H];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      LoadVec<float, H>(cs + k * (a.pairs / 2) + j * H, c[k]);
      LoadVec<float, H>(cs + a.pairs + k * (a.pairs / 2) + j * H, s[k]);
    }
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const F2 x = Fma2(Make2(-u[2 * i + 1], u[2 * i]), Make2(s[0][i], s[0][i]), Mul2(Make2(u[2 * i], u[2 * i + 1]), Make2(c[0][i], c[0][i])));
      const F2 y = Fma2(Make2(-v[2 * i + 1], v[2 * i]), Make2(s[1][i], s[1][i]), Mul2(Make2(v[2 * i], v[2 * i + 1]), Make2(c[1][i], c[1][i])));
      u[2 * i] = X(x); u[2 * i + 1] = Y(x);
      v[2 * i] = X(y); v[2 * i + 1] = Y(y);
    }
  } else {
    float c[VEC], s[VEC];
    LoadPlane<VEC>(cs, j * VEC, a.pairs, c);
    LoadPlane<VEC>(cs + a.pairs, j * VEC, a.pairs, s);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const F2 x = Make2(u[i], u[i + 1]), y = Make2(v[i], v[i + 1]), cc = Make2(c[i], c[i + 1]), ss = Make2(s[i], s[i + 1]);
      const F2 nx = Sub2(Mul2(x, cc), Mul2(y, ss)), ny = Fma2(x, ss, Mul2(y, cc));
      u[i] = X(nx); u[i + 1] = Y(nx);
      v[i] = X(ny); v[i + 1] = Y(ny);
    }
  }
}
// sum + u . v
template <int VEC> __device__ __forceinline__ float Dot(const float (&u)[VEC], const float (&v)[VEC], float sum) {
  if constexpr (VEC == 1) return fmaf(u[0], v[0], sum);
  else {
    F2 x = Make2(sum, 0.f);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) x = Fma2(Make2(u[i], u[i + 1]), Make2(v[i], v[i + 1]), x);
    return X(x) + Y(x);
  }
}
template <int VEC> __device__ __forceinline__ void AddProduct(float (&to)[VEC], const float (&u)[VEC], const float (&v)[VEC]) {
  if constexpr (VEC == 1) to[0] = fmaf(u[0], v[0], to[0]);
  else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const F2 x = Fma2(Make2(u[i], u[i + 1]), Make2(v[i], v[i + 1]), Make2(to[i], to[i + 1]));
      to[i] = X(x); to[i + 1] = Y(x);
    }
  }
}
template <int VEC> __device__ __forceinline__ void AddScaled(float (&to)[VEC], const float (&u)[VEC], float by) {
  float all[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) all[i] = by;
  AddProduct<VEC>(to, u, all);
}
template <int VEC> __device__ __forceinline__ void Times(float (&u)[VEC], const float (&by)[VEC]) {
  if constexpr (VEC == 1) u[0] *= by[0];
  else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const F2 x = Mul2(Make2(u[i], u[i + 1]), Make2(by[i], by[i + 1]));
      u[i] = X(x); u[i + 1] = Y(x);
    }
  }
}
template <int VEC> __device__ __forceinline__ void Scale(float (&u)[VEC], float by) {
  float all[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) all[i] = by;
  Times<VEC>(u, all);
}

// Item j of a row: its pieces start at elements o0 and o1; the first pairs / VEC items are rotated.  Neighbouring items'
// pieces are neighbours in memory: 16-byte accesses a piece apart would move every 32-byte sector twice.
struct Item { int o0, o1; bool turned; };
template <int VEC> __device__ __forceinline__ Item ItemOf(int j, const RopeArgs& a) {
  const int nt = a.pairs / VEC;
  if (VEC == 1 && a.interleaved && j < nt) return {2 * j, 2 * j + 1, true};
  if (j < nt) return {j * VEC, a.pairs + j * VEC, true};
  return {2 * a.pairs + (j - nt) * VEC, a.pairs + a.head_dim / 2 + (j - nt) * VEC, false};   // behind the rotated ones
}

// The weights as fp32 in shared memory: [queries, keys][head_dim], in Plane order.
template <int VEC> __device__ __forceinline__ void FillWeights(float* w, const RopeArgs& a) {
  for (int i = threadIdx.x; i < 2 * a.head_dim; i += kThreads) {
    const int side = i >= a.head_dim, e = i - side * a.head_dim;
    if (a.side[side].w != nullptr) w[side * a.head_dim + Plane<VEC>(e, a.head_dim)] = LoadW(a.side[side].w, a.w_dtype, e);
  }
}
// Pieces times the weights times r.
template <int VEC> __device__ __forceinline__ void TimesWeights(float (&u)[VEC], float (&v)[VEC], const float* w, const Item& it, int dim, float r) {
  float p[VEC], q[VEC];
  LoadPlane<VEC>(w, it.o0, dim, p);   // pieces start at multiples of VEC
  LoadPlane<VEC>(w, it.o1, dim, q);
  Scale<VEC>(u, r);
  Scale<VEC>(v, r);
  Times<VEC>(u, p);
  Times<VEC>(v, q);
}

// A thread's pieces of one row.
template <typename T, int VEC, int NI> struct Pieces {
  Vec<T, VEC> u[NI], v[NI];
  __device__ __forceinline__ void Floats(int n, float (&fu)[VEC], float (&fv)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { fu[i] = ToFloat(u[n].v[i]); fv[i] = ToFloat(v[n].v[i]); }
  }
};

// The pieces of D coming rows, copied to shared memory while the rows before them are worked on.  A thread reads only what
// it has copied itself, so a ring needs no barrier: Start(s), CommitCopies() for each row; WaitCopies() and Take() when its turn comes.
template <typename T, int VEC, int NI, int D> struct Ring {
  using Piece = Vec<T, VEC>;
  static constexpr int kBytes = D * 2 * NI * kThreads * int(sizeof(Piece));
  Piece* mine;
  __device__ __forceinline__ Ring(void* at) : mine(static_cast<Piece*>(at) + threadIdx.x) {}
  __device__ __forceinline__ void Start(int d, const T* x, int in_row, const RopeArgs& a) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int j = in_row + n * a.tpr;
      if (j < a.items) {
        const Item it = ItemOf<VEC>(j, a);
        CopyAhead(mine + (d * 2 * NI + 2 * n) * kThreads, reinterpret_cast<const Piece*>(x + it.o0));
        CopyAhead(mine + (d * 2 * NI + 2 * n + 1) * kThreads, reinterpret_cast<const Piece*>(x + it.o1));
      }
    }
  }
  __device__ __forceinline__ Pieces<T, VEC, NI> Take(int d) const {
    Pieces<T, VEC, NI> x;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      x.u[n] = mine[(d * 2 * NI + 2 * n) * kThreads];
      x.v[n] = mine[(d * 2 * NI + 2 * n + 1) * kThreads];
    }
    return x;
  }
};
// A block's equal part of the tokens, at most as many as its table holds.
template <typename T, int VEC, int NI, int MODE, int D>
__global__ void __launch_bounds__(kThreads, kPerSm) RopeKernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float4 s_mem[];
  Ring<T, VEC, NI, D> ring(s_mem);
  float* s_w = reinterpret_cast<float*>(s_mem) + Ring<T, VEC, NI, D>::kBytes / 4;   // kNorm
  float* s_table = s_w + (MODE == kNorm ? 2 * a.head_dim : 0);
  const int group = threadIdx.x / a.tpr, in_row = threadIdx.x - group * a.tpr;
  const uint32_t groups = kThreads / a.tpr, heads = uint32_t(a.heads[0] + a.heads[1]);
  const uint32_t t0 = uint32_t(a.tokens * blockIdx.x / gridDim.x), t1 = uint32_t(a.tokens * (blockIdx.x + 1) / gridDim.x);
  const uint32_t passes = ((t1 - t0) * heads + groups - 1) / groups;
  Walk now(t0, group, groups, heads, a.div_heads), next = now;
  auto load = [&](int d) {
    if (next.token < t1) {
      const int is_k = int(next.head) >= a.heads[0];
      const Side& s = a.side[is_k];
      ring.Start(d, static_cast<const T*>(s.x) + int64_t(next.token) * s.xt + int64_t(int(next.head) - (is_k ? a.heads[0] : 0)) * s.xh, in_row, a);
    }
    CommitCopies();
    next.Next();
  };
#pragma unroll
  for (int d = 0; d < D; ++d) load(d);
  FillTable<VEC>(s_table, a, t0, t1 - t0);
  if (MODE == kNorm) FillWeights<VEC>(s_w, a);
  __syncthreads();
  for (uint32_t pass = 0; pass < passes; pass += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (pass + d >= passes) break;
      const bool on = now.token < t1;
      const int is_k = int(now.head) >= a.heads[0];
      const Side& s = a.side[is_k];
      WaitCopies<D - 1>();
      const Pieces<T, VEC, NI> x = ring.Take(d);
      float r = 1.f;
      if (MODE == kNorm) {
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          if (on && in_row + n * a.tpr < a.items) {
            float u[VEC], v[VEC];
            x.Floats(n, u, v);
            sum = Dot<VEC>(u, u, Dot<VEC>(v, v, sum));
          }
        }
        for (int o = a.tpr >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
      }
      T* y = static_cast<T*>(s.y) + int64_t(now.token) * s.yt + int64_t(int(now.head) - (is_k ? a.heads[0] : 0)) * s.yh;
      const float* cs = s_table + (now.token - t0) * 2 * a.pairs;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int j = in_row + n * a.tpr;
        if (on && j < a.items) {
          const Item it = ItemOf<VEC>(j, a);
          float u[VEC], v[VEC];
          x.Floats(n, u, v);
          if (MODE == kNorm) TimesWeights<VEC>(u, v, s_w + is_k * a.head_dim, it, a.head_dim, r);
          if (it.turned) Turn<VEC>(u, v, cs, j, a);
          StoreVec<T, VEC>(y + it.o0, u);
          StoreVec<T, VEC>(y + it.o1, v);
        }
      }
      now.Next();
      load(d);
    }
  }
}

// As above, first for the queries and then for the keys, whose weight gradients each thread sums over its rows: the blocks
// and their parts depend on the shape alone, and with them the bits of those sums.
template <typename T, int VEC, int NI, int D>
__global__ void __launch_bounds__(kThreads, 2) NormRopeGradKernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ float4 s_mem[];
  using Rows = Ring<T, VEC, NI, D>;
  Rows x_ring(s_mem), g_ring(reinterpret_cast<char*>(s_mem) + Rows::kBytes);
  float* acc = reinterpret_cast<float*>(s_mem);  // [groups][head_dim], in the rings' place when they are empty
  float* s_w = acc + 2 * Rows::kBytes / 4;
  float* s_table = s_w + 2 * a.head_dim;
  const int group = threadIdx.x / a.tpr, in_row = threadIdx.x - group * a.tpr;
  const int groups = kThreads / a.tpr;
  const uint32_t b0 = uint32_t(a.tokens * blockIdx.x / gridDim.x), b1 = uint32_t(a.tokens * (blockIdx.x + 1) / gridDim.x);
  const bool refill = b1 - b0 > uint32_t(a.table_tokens);
  FillWeights<VEC>(s_w, a);
  for (int which = 0; which < (a.heads[1] > 0 ? 2 : 1); ++which) {
    const Side& s = a.side[which];
    const uint32_t heads = uint32_t(a.heads[which]);
    float du[NI][VEC], dv[NI][VEC];
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
    for (int i = 0; i < VEC; ++i) du[n][i] = dv[n][i] = 0.f;
    for (uint32_t t0 = b0; t0 < b1; t0 += uint32_t(a.table_tokens)) {
      const uint32_t t1 = min(b1, t0 + uint32_t(a.table_tokens));
      const uint32_t passes = ((t1 - t0) * heads + groups - 1) / groups;
      Walk now(t0, group, groups, heads, a.div_side[which]), next = now;
      auto load = [&](int d) {
        if (next.token < t1) {
          x_ring.Start(d, static_cast<const T*>(s.x) + int64_t(next.token) * s.xt + int64_t(next.head) * s.xh, in_row, a);
          g_ring.Start(d, static_cast<const T*>(s.g) + int64_t(next.token) * s.gt + int64_t(next.head) * s.gh, in_row, a);
        }
        CommitCopies();
        next.Next();
      };
#pragma unroll
      for (int d = 0; d < D; ++d) load(d);
      if (which == 0 || refill) {
        __syncthreads();
        FillTable<VEC>(s_table, a, t0, t1 - t0);
        __syncthreads();
      }
      for (uint32_t pass = 0; pass < passes; pass += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
          if (pass + d >= passes) break;
          const bool on = now.token < t1;
          T* y = static_cast<T*>(s.y) + int64_t(now.token) * s.yt + int64_t(now.head) * s.yh;
          const float* cs = s_table + (now.token - t0) * 2 * a.pairs;
          WaitCopies<D - 1>();
          const Pieces<T, VEC, NI> x = x_ring.Take(d), g = g_ring.Take(d);
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < NI; ++n) {
            if (on && in_row + n * a.tpr < a.items) {
              float u[VEC], v[VEC];
              x.Floats(n, u, v);
              sum = Dot<VEC>(u, u, Dot<VEC>(v, v, sum));
            }
          }
          for (int o = a.tpr >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float r = rsqrtf(fmaf(sum, a.inv_dim, a.eps));
          float gu[NI][VEC], gv[NI][VEC];
          float dot = 0.f;
#pragma unroll
          for (int n = 0; n < NI; ++n) {
            const int j = in_row + n * a.tpr;
            if (on && j < a.items) {
              const Item it = ItemOf<VEC>(j, a);
              float u[VEC], v[VEC];
              x.Floats(n, u, v);
              g.Floats(n, gu[n], gv[n]);
              if (it.turned) Turn<VEC>(gu[n], gv[n], cs, j, a);
              Scale<VEC>(u, r);
              Scale<VEC>(v, r);
              AddProduct<VEC>(du[n], gu[n], u);
              AddProduct<VEC>(dv[n], gv[n], v);
              TimesWeights<VEC>(gu[n], gv[n], s_w + which * a.head_dim, it, a.head_dim, r);   // r u
              dot = Dot<VEC>(gu[n], u, Dot<VEC>(gv[n], v, dot));
            }
          }
          for (int o = a.tpr >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
          dot *= -a.inv_dim;
#pragma unroll
          for (int n = 0; n < NI; ++n) {
            const int j = in_row + n * a.tpr;
            if (on && j < a.items) {
              const Item it = ItemOf<VEC>(j, a);
              float u[VEC], v[VEC];
              x.Floats(n, u, v);
              Scale<VEC>(u, r);
              Scale<VEC>(v, r);
              AddScaled<VEC>(gu[n], u, dot);
              AddScaled<VEC>(gv[n], v, dot);
              StoreVec<T, VEC>(y + it.o0, gu[n]);
              StoreVec<T, VEC>(y + it.o1, gv[n]);
            }
          }
          now.Next();
          load(d);
        }
      }
    }
    // the block's partial sums, added in the order of its thread groups
    WaitCopies<0>();
    __syncthreads();
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
    __syncthreads();
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
  a.div_heads = MakeFastDiv(uint32_t(p->q_heads + p->k_heads));
  a.div_side[0] = MakeFastDiv(uint32_t(p->q_heads));
  a.div_side[1] = MakeFastDiv(uint32_t(std::max(1, p->k_heads)));
  a.head_dim = p->head_dim;
  a.inv_dim = 1.f / float(p->head_dim);
  a.pairs = p->rotary_dim / 2;
  a.div_pairs = MakeFastDiv(uint32_t(std::max(1, a.pairs)));
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

int GradBlocks(int64_t tokens) { return int(std::min<int64_t>(kGradBlocks, tokens)); }

template <typename T, int VEC, int NI, int MODE> int Run(RopeArgs& a, cudaStream_t st) {
  a.items = a.head_dim / (2 * VEC);
  a.tpr = 1;
  while (a.tpr < 32 && a.tpr < a.items) a.tpr *= 2;
  const size_t per_token = size_t(std::max(1, a.pairs)) * 2 * sizeof(float);
  const int64_t most = int64_t(kTableBytes / per_token);
  const size_t weights = size_t(2) * a.head_dim * sizeof(float);
  constexpr int D = NI == 1 ? 4 : 2;   // rows in flight per thread: 3 measured the same, 6 took 41 us instead of 39 (norms, 8192 tokens)
  const auto launch = [&](auto kernel, int64_t blocks, size_t ring, const char* what) -> int {
    a.table_tokens = int(std::min<int64_t>(most, (a.tokens + blocks - 1) / blocks));
    const size_t smem = ring + (MODE == kRope ? 0 : weights) + a.table_tokens * per_token;
    if (smem > 48 * 1024) ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    kernel<<<unsigned(blocks), kThreads, smem, st>>>(a);
    return CheckLaunch(what);
  };
  if constexpr (MODE == kGrad) {
    constexpr int kHalf = (D + 1) / 2;
    const int blocks = GradBlocks(a.tokens);
    ITEXB_RETURN_IF_ERROR(launch(NormRopeGradKernel<T, VEC, NI, kHalf>, blocks, 2 * Ring<T, VEC, NI, kHalf>::kBytes, "NormRopeGradKernel"));
    WeightGradKernel<<<dim3((a.head_dim + 31) / 32, a.heads[1] > 0 ? 2 : 1), kSumThreads, 0, st>>>(a, blocks);
    return CheckLaunch("WeightGradKernel");
  } else {
    // Equal parts for whole waves of blocks.  More waves even out the SMs' different distances to memory, fewer pay less for
    // the blocks' starts, which cost more with weights: measured at 1, 2, 4 and 8 waves, rotation of 16384 tokens takes 68,
    // 62, 58 and 59 us (37 tokens a block to 5), norms and rotation of 8192 tokens 39, 41, 44 and 51 us (18 to 2).
    constexpr int kLeast = MODE == kNorm ? 16 : 8;   // tokens a block has at least before there is a second wave
    const int64_t wave = kPerSm * kSms, waves = std::max((a.tokens + wave * most - 1) / (wave * most), a.tokens / (wave * kLeast));
    return launch(RopeKernel<T, VEC, NI, MODE, D>, std::min(a.tokens, wave * std::max<int64_t>(1, waves)), Ring<T, VEC, NI, D>::kBytes, "RopeKernel");
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
  return size_t(2) * size_t(GradBlocks(tokens)) * size_t(head_dim) * sizeof(float);
}

extern "C" int itexb_qk_norm_rope_grad(const itexb_qk_norm_rope_grad_params_t* p, itexb_stream_t stream) {
  const char* what = "qk_norm_rope_grad";
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "%s: NULL params", what);
  const itexb_qk_norm_rope_params_t& n = p->n;
  ITEXB_RETURN_IF_ERROR(CheckNorm(&n, what));
  ITEXB_REQUIRE(p->d_q_weight && (n.r.k_heads == 0 || p->d_k_weight), ITEXB_INVALID_ARGUMENT, "%s: NULL weight gradient", what);
  cudaStream_t st = AsCuda(stream);
  ITEXB_REQUIRE(n.r.tokens == 0 || (p->q_grad && (n.r.k_heads == 0 || p->k_grad) && p->workspace), ITEXB_INVALID_ARGUMENT,
                "%s: NULL gradient or workspace", what);
  // sums over nothing
  const size_t bytes = size_t(n.r.head_dim) * DtypeSize(n.w_dtype);
  if (p->d_k_weight && (n.r.tokens == 0 || n.r.k_heads == 0)) ITEXB_CUDA(cudaMemsetAsync(p->d_k_weight, 0, bytes, st));
  if (n.r.tokens == 0) {
    ITEXB_CUDA(cudaMemsetAsync(p->d_q_weight, 0, bytes, st));
    return ITEXB_OK;
  }
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
