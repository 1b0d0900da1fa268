// Attention over the 4-bit paged cache (itexb_kv4_attention).
//
//   out = sum_j softmax_j(scale * q . k_j) v_j,  k_j, v_j = lo + step * code, j over the visible rows
//
// One block per query row and head: its four warps take the visible rows in turn, a lane holds head_dim / 32 elements
// and the running maximum, sum and output are kept in fp32 and joined at the end.
#include <algorithm>
#include <climits>

#include "kv4.h"

namespace itexb {
namespace {

struct AttnArgs {
  Kv4View c;
  const void* q; int64_t qt, qh;
  void* out; int64_t ot, oh;
  const int32_t* table; int64_t table_stride;
  const int32_t* kept;
  const int32_t* q_starts;
  int32_t* status_word;
  int64_t total_rows;
  int table_cols, num_seqs, q_heads, share, causal, window, max_new, max_kept;
  float scale_log2;      // scale * log2(e)
};

struct Seq { int64_t row0; int nnew, kept; };

// Lengths of sequence b, cut to the launch's bounds; what is cut off is reported.
__device__ __forceinline__ Seq SeqOf(const AttnArgs& a, int b, bool report) {
  Seq s;
  int64_t n = a.max_new;
  s.row0 = int64_t(b) * a.max_new;
  if (a.q_starts != nullptr) {
    s.row0 = a.q_starts[b];
    n = int64_t(a.q_starts[b + 1]) - s.row0;
  }
  const int64_t most = min(int64_t(a.max_kept), int64_t(a.table_cols) * a.c.page_size);
  int64_t kept = a.kept[b];
  const bool bad = n < 0 || n > a.max_new || s.row0 < 0 || s.row0 + n > a.total_rows || kept < 0 || kept > most;
  if (bad) {
    if (report) ReportIndex(a.status_word);
    if (s.row0 < 0 || s.row0 > a.total_rows) n = 0;
    n = max(int64_t(0), min(min(n, int64_t(a.max_new)), a.total_rows - s.row0));
    kept = max(int64_t(0), min(kept, most));
  }
  s.nnew = int(n);
  s.kept = int(kept);
  return s;
}

template <typename T, int DIM>
__global__ void __launch_bounds__(128) Kv4AttentionKernel(const __grid_constant__ AttnArgs a) {
  constexpr int E = DIM / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Seq s = SeqOf(a, b, threadIdx.x == 0 && i == 0 && h == 0);
  if (i >= s.nnew) return;
  const int kvh = h / a.share;
  const int64_t place = int64_t(s.kept) - s.nnew + i;
  const int end = a.causal ? int(max(int64_t(0), min(int64_t(s.kept), place + 1))) : s.kept;
  const int begin = a.window > 0 ? int(max(int64_t(0), place - a.window + 1)) : 0;
  const T* q = static_cast<const T*>(a.q) + (s.row0 + i) * a.qt + int64_t(h) * a.qh;
  float qv[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { qv[e] = ToFloat(q[lane * E + e]) * a.scale_log2; o[e] = 0.f; }
  float m = -INFINITY, l = 0.f;
  for (int j = begin + warp; j < end; j += 4) {
    const uint32_t col = QuickDiv(uint32_t(j), a.c.div_page);
    const int page = a.table[int64_t(b) * a.table_stride + col];
    if (page < 0 || page >= a.c.num_pages) {
      if (lane == 0) ReportIndex(a.status_word);
      continue;
    }
    const int64_t off = j - int(col) * a.c.page_size;
    const int64_t ci = int64_t(page) * a.c.cp + int64_t(kvh) * a.c.ch + off * a.c.ct + lane * E / 2;
    const int64_t pi = int64_t(page) * a.c.pp + int64_t(kvh) * a.c.ph + off * a.c.pt + lane * E / a.c.group;
    const float2 kp = __half22float2(a.c.k_params[pi]), vp = __half22float2(a.c.v_params[pi]);
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) dot = fmaf(qv[e], fmaf(float((a.c.k_codes[ci + e / 2] >> (4 * (e & 1))) & 15), kp.y, kp.x), dot);
    for (int t = 16; t > 0; t >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, t);
    const float top = fmaxf(m, dot);
    const float old = m == -INFINITY ? 0.f : exp2f(m - top), p = top == -INFINITY ? 0.f : exp2f(dot - top);
    l = l * old + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, fmaf(float((a.c.v_codes[ci + e / 2] >> (4 * (e & 1))) & 15), vp.y, vp.x), o[e] * old);
    m = top;
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  __syncthreads();
  float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float w[4], sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) { w[k] = s_m[k] == -INFINITY ? (isnan(s_l[k]) ? s_l[k] : 0.f) : exp2f(s_m[k] - top); sum = fmaf(s_l[k], w[k], sum); }
  T* out = static_cast<T*>(a.out) + (s.row0 + i) * a.ot + int64_t(h) * a.oh;
  for (int d = threadIdx.x; d < DIM; d += 128) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) v = fmaf(s_o[k][d], w[k], v);
    out[d] = FromFloat<T>(sum == 0.f ? 0.f : v / sum);
  }
}

int CheckAttention(const itexb_kv4_attention_params_t* p, AttnArgs* a) {
  const char* what = "kv4_attention";
  ITEXB_REQUIRE(p != nullptr, ITEXB_INVALID_ARGUMENT, "%s: NULL params", what);
  ITEXB_RETURN_IF_ERROR(CheckKv4(p->cache, what, &a->c));
  ITEXB_REQUIRE(p->dtype == ITEXB_DT_BFLOAT16 || p->dtype == ITEXB_DT_HALF, ITEXB_INVALID_ARGUMENT, "%s: unsupported type %s", what,
                DtypeName(p->dtype));
  ITEXB_REQUIRE(p->num_seqs >= 0 && p->q_heads > 0 && p->q_heads % p->cache.kv_heads == 0, ITEXB_INVALID_ARGUMENT,
                "%s: q_heads must be a multiple of kv_heads, got %d and %d", what, p->q_heads, p->cache.kv_heads);
  ITEXB_REQUIRE(p->max_new >= 0 && p->max_kept >= 0 && p->window >= 0 && p->total_rows >= 0 && p->table_cols >= 0, ITEXB_INVALID_ARGUMENT,
                "%s: negative bound", what);
  ITEXB_REQUIRE(p->num_seqs <= 65535 && p->q_heads <= 65535, ITEXB_INVALID_ARGUMENT, "%s: more than 65535 sequences or heads", what);
  ITEXB_REQUIRE(int64_t(p->max_new) * p->q_heads < (int64_t(1) << 31), ITEXB_INVALID_ARGUMENT, "%s: 2^31 query rows of a sequence or more", what);
  a->q = p->q; a->qt = p->q_token_stride; a->qh = p->q_head_stride;
  a->out = p->out; a->ot = p->out_token_stride; a->oh = p->out_head_stride;
  a->table = p->block_table; a->table_stride = p->table_stride; a->table_cols = p->table_cols;
  a->kept = p->kept; a->q_starts = p->q_starts; a->status_word = p->status_word;
  a->total_rows = p->total_rows;
  a->num_seqs = p->num_seqs; a->q_heads = p->q_heads; a->share = p->q_heads / p->cache.kv_heads;
  a->causal = p->causal != 0; a->window = p->window; a->max_new = p->max_new; a->max_kept = p->max_kept;
  a->scale_log2 = p->scale * 1.4426950408889634f;
  return ITEXB_OK;
}

}  // namespace
}  // namespace itexb

using namespace itexb;

extern "C" size_t itexb_kv4_attention_workspace_bytes(const itexb_kv4_attention_params_t*) { return 0; }

extern "C" int itexb_kv4_attention(const itexb_kv4_attention_params_t* p, itexb_stream_t stream) {
  AttnArgs a{};
  ITEXB_RETURN_IF_ERROR(CheckAttention(p, &a));
  if (p->num_seqs == 0 || p->max_new == 0 || p->total_rows == 0) return ITEXB_OK;
  ITEXB_REQUIRE(p->q && p->out && p->kept && (p->block_table || p->table_cols == 0), ITEXB_INVALID_ARGUMENT, "kv4_attention: NULL tensor");
  cudaStream_t st = AsCuda(stream);
  const dim3 grid(p->max_new, p->q_heads, p->num_seqs);
#define ITEXB_ATTN(T)                                                                            \
  do {                                                                                           \
    if (p->cache.head_dim == 64) Kv4AttentionKernel<T, 64><<<grid, 128, 0, st>>>(a);             \
    else if (p->cache.head_dim == 128) Kv4AttentionKernel<T, 128><<<grid, 128, 0, st>>>(a);      \
    else Kv4AttentionKernel<T, 256><<<grid, 128, 0, st>>>(a);                                    \
  } while (0)
  if (p->dtype == ITEXB_DT_BFLOAT16) ITEXB_ATTN(__nv_bfloat16);
  else ITEXB_ATTN(__half);
#undef ITEXB_ATTN
  return CheckLaunch("Kv4AttentionKernel");
}
