// What the kernels of itexb_kv4_attention share.
#ifndef ITEXB_CSRC_KV4_ATTENTION_H_
#define ITEXB_CSRC_KV4_ATTENTION_H_

#include "kv4.h"

namespace itexb {

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
  int q_aligned;           // q's rows are 16-byte aligned
  float scale_log2;        // scale * log2(e)
  FastDiv div_share;
};

constexpr int kMostKept = 0x7fffffff - 4096;   // tokens of a sequence

struct Seq { int64_t row0; int nnew, kept; };

// Lengths of sequence b, cut to the launch's bounds; what is cut off is reported.
__device__ __forceinline__ Seq SeqOf(const AttnArgs& a, int b, bool report) {
  Seq s;
  int64_t n = a.max_new;
  s.row0 = int64_t(b) * a.max_new;
  if (a.q_starts != nullptr) {
    s.row0 = __ldg(a.q_starts + b);
    n = int64_t(__ldg(a.q_starts + b + 1)) - s.row0;
  }
  // tiles are rounded up in 32 bits behind the last token
  const int64_t most = min(min(int64_t(a.max_kept), int64_t(a.table_cols) * a.c.page_size), int64_t(kMostKept));
  int64_t kept = __ldg(a.kept + b);
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

// Visible rows [begin, end) of new token i.
__device__ __forceinline__ int RowBegin(const AttnArgs& a, const Seq& s, int i) {
  return a.window > 0 ? int(max(int64_t(0), int64_t(s.kept) - s.nnew + i - a.window + 1)) : 0;
}
__device__ __forceinline__ int RowEnd(const AttnArgs& a, const Seq& s, int i) {
  return a.causal ? max(0, s.kept - s.nnew + i + 1) : s.kept;   // i < nnew: at most kept
}

__device__ __forceinline__ float Exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// Two elements of a query row (bf16 or half).
__device__ __forceinline__ float2 QueryPair(uint32_t w, bool bf16) {
  return bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// The same times a power of two (or its negative, or zero), as halves; for halves it is 1.
__device__ __forceinline__ uint32_t QueryHalf2(uint32_t w, bool bf16, float by) {
  uint32_t r;
  if (bf16) {
    const F2 x = Mul2(Make2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), Make2(by, by));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(Y(x)), "f"(X(x)));
  } else {
    uint32_t by2;
    asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(by2) : "f"(by));
    asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(by2));
  }
  return r;
}
// The larger magnitudes of two pairs of bf16 or halves (their bits order like their values; NaN counts as large).
__device__ __forceinline__ uint32_t MaxBits2(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }

size_t StepsWorkspace(const AttnArgs& a);
int LaunchSteps(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st);
size_t PrefillWorkspace(const AttnArgs& a);
int LaunchPrefill(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st);

}  // namespace itexb

#endif  // ITEXB_CSRC_KV4_ATTENTION_H_
