// Attention of few query rows over the 4-bit paged cache: decoding steps, drafted tokens.
//
// Bound: the cache's bytes (head_dim 128, groups of 64: 144 bytes per token and head, keys and values), as long as turning
// codes into operands stays cheap.  The codes themselves are multiplied, and the groups' ranges enter behind the products:
//     q . k_t = sum_g step_tg (sum_{d in g} q_d c_td) + lo_tg (sum_{d in g} q_d)
//     o_d     = sum_t (p_t step_tg) (c_td - 8) + sum_t p_t (lo_tg + 8 step_tg)
// A code becomes a half by or-ing it into the low mantissa bits of a constant where it lies: 1024 + c at bits 0-3, 64 + c at
// bits 4-7.  The keys' products take the constants along and their share, constant * sum q, is taken back in fp32.  The
// values' constants are subtracted before the product (exact), because there the sums run over all tokens: left in, they
// cost an 128 Ki context three digits.  Codes count from the middle of their range so that the rounding of (p step) is
// relative to what a value differs from it.
// q enters as half: for bf16 inputs each row is scaled by a power of two to at most 2, so that elements within 2^-14 of the
// row's largest stay exact and the others are off by 2^-25 of it.  p is kept at most 4 (see kRescale), p * step is then
// below 2^15.1 for every step a half can hold; small products lose bits only where they are 2^-11 of the largest or less.
//
// A warp owns tiles of 16 tokens and keeps its own running maximum, so warps meet only at the end of a block's chunk of
// tokens.  Both products run on mma.m16n8k16 with the cache as the 16-row operand (16 tokens, 16 channels) and up to
// 8 query rows of the key/value head as the 8 columns: S^T = K q^T, O^T += V^T P^T; the weights turn from the first one's
// accumulator layout into the second one's operand by an 8 x 8 transpose each.  Tensor cores of the tcgen05 kind want 64 or
// more rows, of which a decoding step has 1 to 8, and operands in shared memory; here the tensor work is a small part of
// the issue slots.  The order of channels inside a product is free, so lanes take them as the codes lie in a word.
// Tiles come in through per-warp rings of cp.async copies (three tiles in flight per warp, sixteen or more warps per SM); the
// 16-byte pieces are permuted so that both products read them without bank conflicts.
// A context is cut into chunks of up to 2048 tokens, one block each; their partial results are joined by a second kernel.
#include <algorithm>

#include "kv4_attention.h"

namespace itexb {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;                       // tokens
constexpr int kStages = 4;
constexpr int kMaxChunk = kTile * kWarps * 32;  // a lane of each warp holds the page of one of its tiles
constexpr float kRescale = 4.f;                 // scores may pass the running maximum by 4 before it moves,
constexpr float kShift = 2.f;                   // so weights are 2^(score - maximum - 2), at most 4
constexpr float kNone = -INFINITY;

struct StepArgs {
  AttnArgs a;
  int chunk;           // tokens, a multiple of kTile * kWarps
  int chunks;          // per sequence at most
  int row_tiles;
  float* part_o;       // [seqs][kv_heads][max_new * share][chunks][head_dim], null: one chunk, write the output
  float2* part_ml;     // ... (maximum, sum)
  int bf16;            // type of q and out, else half
};

template <int DIM> __device__ __forceinline__ uint32_t PieceAt(int row, int piece) {  // byte offset of a 16-byte piece in a tile
  if (DIM == 64) return uint32_t((row >> 2) * 128 + ((((row & 3) * 2 + piece) ^ (((row >> 2) & 1) * 2)) * 16));
  if (DIM == 128) return uint32_t((row >> 1) * 128 + ((((row & 1) * 4 + piece) ^ (((row >> 1) & 3) * 2)) * 16));
  return uint32_t(row * 128 + ((piece ^ (((row & 1) * 4) ^ (((row >> 1) & 1) * 2) ^ (((row >> 2) & 1) * 4))) * 16));
}

template <int BYTES> __device__ __forceinline__ void CpAsync(uint32_t dst, const void* src) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

__device__ __forceinline__ void Mma(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// The codes of a word's nibbles 0 and 4 as 1024 + c, of 1 and 5 as 64 + c (pairs of halves); nibbles 2, 6, 3, 7: of w >> 8.
__device__ __forceinline__ uint32_t AndOr(uint32_t x, uint32_t mask, uint32_t constant) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(constant));
  return r;
}
__device__ __forceinline__ uint32_t EvenCodes(uint32_t w) { return AndOr(w, 0x000F000Fu, 0x64006400u); }
__device__ __forceinline__ uint32_t OddCodes(uint32_t w) { return AndOr(w, 0x00F000F0u, 0x54005400u); }
__device__ __forceinline__ uint32_t AddHalf2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("add.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
// c - 8 from the above
__device__ __forceinline__ uint32_t EvenCentred(uint32_t w) { return AddHalf2(EvenCodes(w), 0xE408E408u); }   // - 1032
__device__ __forceinline__ uint32_t OddCentred(uint32_t w) { return AddHalf2(OddCodes(w), 0xD480D480u); }    // - 72
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Pairs of fp32 values handled by one instruction; each is rounded as alone.
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 Make2(float x, float y) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ F2 Same2(float x) { return Make2(x, x); }
__device__ __forceinline__ float X(F2 a) { float x, y; asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); return x; }
__device__ __forceinline__ float Y(F2 a) { float x, y; asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v)); return y; }
__device__ __forceinline__ F2 Fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
__device__ __forceinline__ F2 Mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ F2 Add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }

// Partial results of four warps (or of several chunks) with maxima m and sums l: what the part's values are weighed with.
__device__ __forceinline__ float PartWeight(float m, float l, float top) { return m == kNone ? (isnan(l) ? l : 0.f) : Exp2(m - top); }

__device__ __forceinline__ void StoreOut(const AttnArgs& a, int bf16, int64_t at, float v) {
  if (bf16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// PAGE16: pages hold a multiple of 16 tokens, so a tile lies in one page.
template <int DIM, int GROUP, int NT, bool PAGE16>
__global__ void __launch_bounds__(kThreads) StepsKernel(const __grid_constant__ StepArgs s) {
  constexpr int NG = DIM / GROUP;
  constexpr int kRow = DIM / 2, kPieces = DIM / 32;
  constexpr int kCodes = kTile * kRow, kPars = kTile * NG * 4;
  constexpr int kStage = 2 * kCodes + 2 * kPars;
  constexpr int kW = GROUP / 32;                 // words of codes per lane, group and row (keys); halves (values)
  const AttnArgs& a = s.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_ok[kWarps][kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;
  const int kvh = int(blockIdx.y) / s.row_tiles, rt = int(blockIdx.y) - kvh * s.row_tiles, b = blockIdx.z;
  const Seq q = SeqOf(a, b, threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0);
  const int rows = q.nnew * a.share, row0 = rt * 8 * NT;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (row0 >= rows) return;
  // the tokens that some row of this block sees, and those that all of them see
  const int i_first = int(QuickDiv(uint32_t(row0), a.div_share)), i_last = int(QuickDiv(uint32_t(min(rows, row0 + 8 * NT) - 1), a.div_share));
  const int seq_begin = RowBegin(a, q, 0) & ~(kTile - 1);   // of the sequence's first row: chunks are laid out from here
  const int block_begin = RowBegin(a, q, i_first), all_begin = RowBegin(a, q, i_last), all_end = RowEnd(a, q, i_first);
  const int begin = seq_begin + int(blockIdx.x) * s.chunk;
  const int end = min(begin + s.chunk, RowEnd(a, q, i_last));
  const int ntiles = end > begin ? (end - begin + kTile - 1) / kTile : 0;
  if (ntiles == 0 && (blockIdx.x > 0 || s.part_o != nullptr)) {
    // the joining kernel reads every chunk of the sequence's rows
    if (s.part_o != nullptr && begin < RowEnd(a, q, q.nnew - 1)) {
      const int n = min(8 * NT, rows - row0);
      const int64_t at = ((int64_t(b) * a.c.kv_heads + kvh) * (int64_t(a.max_new) * a.share) + row0) * s.chunks + blockIdx.x;
      if (int(threadIdx.x) < n) s.part_ml[at + int64_t(threadIdx.x) * s.chunks] = make_float2(kNone, 0.f);
      for (int x = threadIdx.x; x < n * DIM; x += kThreads) s.part_o[(at + int64_t(x / DIM) * s.chunks) * DIM + x % DIM] = 0.f;
    }
    return;
  }

  // ---- query rows as the 8-column operand; per group the sums sum q and the constants' share in the products
  uint32_t qf[NT][DIM / 16][2];
  F2 qs[NT][NG], qc[NT][NG], scale[NT];  // of columns 2c, 2c + 1
  int lo[NT][2], hi[NT][2];              // visible tokens of those columns
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int rr = row0 + nt * 8 + r;
    const bool on = rr < rows;
    const int i = int(QuickDiv(uint32_t(on ? rr : row0), a.div_share)), h = (on ? rr : row0) - i * a.share;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (q.row0 + i) * a.qt + int64_t(kvh * a.share + h) * a.qh;
    union Piece { uint4 v; uint32_t u[4]; uint16_t e[8]; } x[NG][kW];
    float most = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        const int d = g * GROUP + c * (GROUP / 4) + w * 8;
        if (!on) x[g][w].v = make_uint4(0, 0, 0, 0);
        else if (a.q_aligned) x[g][w].v = *reinterpret_cast<const uint4*>(src + d);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) x[g][w].e[e] = src[d + e];
        if (s.bf16)
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(__uint_as_float(uint32_t(x[g][w].e[e]) << 16)));
      }
    float down = 1.f, up = a.scale_log2;     // powers of two: q * down is exact
    if (s.bf16) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int e = min(max(int(__float_as_uint(most) >> 23), 1), 253);
      if (most > 0.f && most < INFINITY) {
        down = __uint_as_float(uint32_t(254 - e) << 23);
        up = __uint_as_float(uint32_t(e) << 23) * a.scale_log2;
      }
    }
    scale[nt] = Make2(__shfl_sync(0xffffffffu, up, (2 * c) * 4), __shfl_sync(0xffffffffu, up, (2 * c + 1) * 4));
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f, share = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        Piece& y = x[g][w];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (s.bf16) y.e[e] = __half_as_ushort(__float2half_rn(__uint_as_float(uint32_t(y.e[e]) << 16) * down));
          const float f = __half2float(__ushort_as_half(y.e[e]));
          sum += f;
          share += f * ((e & 1) ? 64.f : 1024.f);
        }
        // a word's codes come out in pairs (j, j + 4)
        const int ks = (g * kW + w) * 2;
        qf[nt][ks][0] = __byte_perm(y.u[0], y.u[2], 0x5410);
        qf[nt][ks][1] = __byte_perm(y.u[0], y.u[2], 0x7632);
        qf[nt][ks + 1][0] = __byte_perm(y.u[1], y.u[3], 0x5410);
        qf[nt][ks + 1][1] = __byte_perm(y.u[1], y.u[3], 0x7632);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      share += __shfl_xor_sync(0xffffffffu, share, 1);
      share += __shfl_xor_sync(0xffffffffu, share, 2);
      qs[nt][g] = Make2(__shfl_sync(0xffffffffu, sum, (2 * c) * 4), __shfl_sync(0xffffffffu, sum, (2 * c + 1) * 4));
      qc[nt][g] = Make2(-__shfl_sync(0xffffffffu, share, (2 * c) * 4), -__shfl_sync(0xffffffffu, share, (2 * c + 1) * 4));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int ii = int(QuickDiv(uint32_t(min(rows - 1, row0 + nt * 8 + 2 * c + e)), a.div_share));  // a column without a row: any bounds
      lo[nt][e] = RowBegin(a, q, ii);
      hi[nt][e] = RowEnd(a, q, ii);
    }
  }

  // ---- tiles: w, w + 4, ...
  uint8_t* ring = smem + warp * (kStages * kStage);
  const uint32_t ring_addr = uint32_t(__cvta_generic_to_shared(ring));
  const int mine = ntiles > warp ? (ntiles - warp + kWarps - 1) / kWarps : 0;
  const int32_t* table = a.table + int64_t(b) * a.table_stride;
  int my_page = -1;
  if (PAGE16 && lane < mine) {
    my_page = __ldg(table + QuickDiv(uint32_t(begin + (warp + lane * kWarps) * kTile), a.c.div_page));
    if (my_page < 0 || my_page >= a.c.num_pages) {
      ReportIndex(a.status_word);
      my_page = -1;
    }
  }
  const uint8_t* kcodes = a.c.k_codes + int64_t(kvh) * a.c.ch;
  const uint8_t* vcodes = a.c.v_codes + int64_t(kvh) * a.c.ch;
  const int64_t lane_at = int64_t(lane / kPieces) * a.c.ct + (lane % kPieces) * 16;   // this lane's first piece in a tile
  const int64_t lane_step = int64_t(32 / kPieces) * a.c.ct;
  const __half2* pars = (lane < 16 ? a.c.k_params : a.c.v_params) + int64_t(kvh) * a.c.ph;

  auto issue = [&](int n) {
    const int stage = n & (kStages - 1);
    const int j0 = begin + (warp + n * kWarps) * kTile;
    const uint32_t dst = ring_addr + stage * kStage;
    if (PAGE16) {
      const int page = __shfl_sync(0xffffffffu, my_page, n);
      if (page >= 0) {
        const int off = j0 - int(QuickDiv(uint32_t(j0), a.c.div_page)) * a.c.page_size;
        int64_t from = int64_t(page) * a.c.cp + int64_t(off) * a.c.ct + lane_at;
#pragma unroll
        for (int x = 0; x < kPieces * kTile; x += 32) {
          const int row = (x + lane) / kPieces, piece = (x + lane) % kPieces;
          CpAsync<16>(dst + PieceAt<DIM>(row, piece), kcodes + from);
          CpAsync<16>(dst + kCodes + PieceAt<DIM>(row, piece), vcodes + from);
          from += lane_step;
        }
        const __half2* p = pars + int64_t(page) * a.c.pp + int64_t(off + (lane & 15)) * a.c.pt;
        const uint32_t pd = dst + 2 * kCodes + lane * (NG * 4);   // keys' rows, then values'
        if (NG <= 4) CpAsync<(NG > 4 ? 4 : NG) * 4>(pd, p);
        else { CpAsync<16>(pd, p); CpAsync<16>(pd + 16, p + 4); }
      }
      if (lane == 0) s_ok[warp][stage] = page >= 0 ? 0xffffu : 0u;
    } else {
      int page = -1, off = 0;
      const int j = j0 + (lane & 15);
      if (j >= block_begin && j < end) {
        const int col = int(QuickDiv(uint32_t(j), a.c.div_page));
        off = j - col * a.c.page_size;
        page = __ldg(table + col);
        if (page < 0 || page >= a.c.num_pages) {
          ReportIndex(a.status_word);
          page = -1;
        }
      }
      const uint32_t ok = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;
#pragma unroll
      for (int x = 0; x < kPieces * kTile; x += 32) {
        const int row = (x + lane) / kPieces, piece = (x + lane) % kPieces;
        const int pg = __shfl_sync(0xffffffffu, page, row), of = __shfl_sync(0xffffffffu, off, row);
        if (pg >= 0) {
          const int64_t from = int64_t(pg) * a.c.cp + int64_t(of) * a.c.ct + piece * 16;
          CpAsync<16>(dst + PieceAt<DIM>(row, piece), kcodes + from);
          CpAsync<16>(dst + kCodes + PieceAt<DIM>(row, piece), vcodes + from);
        }
      }
      if (page >= 0) {
        const __half2* p = pars + int64_t(page) * a.c.pp + int64_t(off) * a.c.pt;
        const uint32_t pd = dst + 2 * kCodes + lane * (NG * 4);
        if (NG <= 4) CpAsync<(NG > 4 ? 4 : NG) * 4>(pd, p);
        else { CpAsync<16>(pd, p); CpAsync<16>(pd + 16, p + 4); }
      }
      if (lane == 0) s_ok[warp][stage] = ok;
    }
  };

  float o[NT][DIM / 16][4];
  F2 zsum[NT][NG], l[NT];
  float m[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 0; x < DIM / 16; ++x) o[nt][x][0] = o[nt][x][1] = o[nt][x][2] = o[nt][x][3] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) zsum[nt][g] = Same2(0.f);
    m[nt][0] = m[nt][1] = kNone;
    l[nt] = Same2(0.f);
  }

#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) {
    if (n < mine) issue(n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int n = 0; n < mine; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    if (n + kStages - 1 < mine) issue(n + kStages - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const int stage = n & (kStages - 1);
    const uint8_t* st = ring + stage * kStage;
    const int j0 = begin + (warp + n * kWarps) * kTile;
    const uint32_t ok = s_ok[warp][stage];

    // ---- scores of tokens r, r + 8 and columns 2c, 2c + 1
    F2 t[NT][2];
    const __half2* kp = reinterpret_cast<const __half2*>(st + 2 * kCodes);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t w0[kW], w1[kW];
      const int byte = g * (GROUP / 2) + c * (GROUP / 8);
      const uint8_t* from = st + PieceAt<DIM>(r, byte / 16) + byte % 16;
      if (kW == 1) { w0[0] = *reinterpret_cast<const uint32_t*>(from); w1[0] = *reinterpret_cast<const uint32_t*>(from + 8 * kRow); }
      else if (kW == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(from), y = *reinterpret_cast<const uint2*>(from + 8 * kRow);
        w0[0] = x.x; w0[kW - 1] = x.y; w1[0] = y.x; w1[kW - 1] = y.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(from), y = *reinterpret_cast<const uint4*>(from + 8 * kRow);
        w0[0] = x.x; w0[1 % kW] = x.y; w0[2 % kW] = x.z; w0[3 % kW] = x.w;
        w1[0] = y.x; w1[1 % kW] = y.y; w1[2 % kW] = y.z; w1[3 % kW] = y.w;
      }
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t u0 = half ? w0[w] >> 8 : w0[w], u1 = half ? w1[w] >> 8 : w1[w];
          const uint32_t x[4] = {EvenCodes(u0), EvenCodes(u1), OddCodes(u0), OddCodes(u1)};
          const int ks = (g * kW + w) * 2 + half;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Mma(acc[nt], x, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
      const float2 p0 = __half22float2(kp[r * NG + g]), p1 = __half22float2(kp[(r + 8) * NG + g]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const F2 l0 = Same2(p0.x), l1 = Same2(p1.x);
        const F2 base0 = g == 0 ? Mul2(l0, qs[nt][g]) : Fma2(l0, qs[nt][g], t[nt][0]);
        const F2 base1 = g == 0 ? Mul2(l1, qs[nt][g]) : Fma2(l1, qs[nt][g], t[nt][1]);
        t[nt][0] = Fma2(Same2(p0.y), Add2(Make2(acc[nt][0], acc[nt][1]), qc[nt][g]), base0);
        t[nt][1] = Fma2(Same2(p1.y), Add2(Make2(acc[nt][2], acc[nt][3]), qc[nt][g]), base1);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) { t[nt][0] = Mul2(t[nt][0], scale[nt]); t[nt][1] = Mul2(t[nt][1], scale[nt]); }

    // ---- masks: only tiles that not every row sees whole
    const bool partial = j0 < all_begin || j0 + kTile > all_end || ok != 0xffffu;
    uint32_t seen = 0xffffffffu;     // bit 4 nt + 2 * (token r + 8) + column
    if (partial) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int in = r + 8 * k, j = j0 + in;
          const bool there = ((ok >> in) & 1u) != 0u;
          float v[2] = {X(t[nt][k]), Y(t[nt][k])};
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!there || j < lo[nt][e] || j >= hi[nt][e]) {
              seen &= ~(1u << (4 * nt + 2 * k + e));
              v[e] = kNone;
            }
          t[nt][k] = Make2(v[0], v[1]);
        }
    }
    // ---- the running maximum, moved only when a score passes it by more than kRescale
    bool above = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      above = above || fmaxf(X(t[nt][0]), X(t[nt][1])) > m[nt][0] + kRescale || fmaxf(Y(t[nt][0]), Y(t[nt][1])) > m[nt][1] + kRescale;
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = e ? fmaxf(Y(t[nt][0]), Y(t[nt][1])) : fmaxf(X(t[nt][0]), X(t[nt][1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top, m[nt][e]);
          f[e] = top == kNone ? 1.f : Exp2(m[nt][e] - top);
          m[nt][e] = top;
        }
        const F2 f2 = Make2(f[0], f[1]);
        l[nt] = Mul2(l[nt], f2);
#pragma unroll
        for (int g = 0; g < NG; ++g) zsum[nt][g] = Mul2(zsum[nt][g], f2);
#pragma unroll
        for (int x = 0; x < DIM / 16; ++x) { o[nt][x][0] *= f[0]; o[nt][x][1] *= f[1]; o[nt][x][2] *= f[0]; o[nt][x][3] *= f[1]; }
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const F2 down = Make2(m[nt][0] == kNone ? 0.f : -kShift - m[nt][0], m[nt][1] == kNone ? 0.f : -kShift - m[nt][1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const F2 d = Add2(t[nt][k], down);
        t[nt][k] = Make2(Exp2(X(d)), Exp2(Y(d)));
        l[nt] = Add2(l[nt], t[nt][k]);
      }
    }

    // ---- values: weights times the group's steps as the 8-column operand, codes of 16 channels as rows
    const uint8_t* sv = st + kCodes;
    const __half2* vp = reinterpret_cast<const __half2*>(st + 2 * kCodes + kPars);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 p0 = __half22float2(vp[r * NG + g]), p1 = __half22float2(vp[(r + 8) * NG + g]);
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const F2 mid0 = Same2(fmaf(8.f, p0.y, p0.x)), mid1 = Same2(fmaf(8.f, p1.y, p1.x));
        F2 w0 = Mul2(t[nt][0], Same2(p0.y)), w1 = Mul2(t[nt][1], Same2(p1.y));
        if (partial) {  // an unseen row's lo and step may be anything
          const uint32_t b = seen >> (4 * nt);
          w0 = Make2(b & 1u ? X(w0) : 0.f, b & 2u ? Y(w0) : 0.f);
          w1 = Make2(b & 4u ? X(w1) : 0.f, b & 8u ? Y(w1) : 0.f);
          const F2 z0 = Mul2(t[nt][0], mid0), z1 = Mul2(t[nt][1], mid1);
          zsum[nt][g] = Add2(zsum[nt][g], Add2(Make2(b & 1u ? X(z0) : 0.f, b & 2u ? Y(z0) : 0.f), Make2(b & 4u ? X(z1) : 0.f, b & 8u ? Y(z1) : 0.f)));
        } else {
          zsum[nt][g] = Fma2(t[nt][0], mid0, Fma2(t[nt][1], mid1, zsum[nt][g]));
        }
        b0[nt] = Transpose8x8(PackHalf(X(w0), Y(w0)));
        b1[nt] = Transpose8x8(PackHalf(X(w1), Y(w1)));
      }
      const int byte = g * (GROUP / 2) + r * (GROUP / 16);
      const uint8_t* fa = sv + PieceAt<DIM>(2 * c, byte / 16) + byte % 16;
      const uint8_t* fb = sv + PieceAt<DIM>(2 * c + 1, byte / 16) + byte % 16;
      uint32_t x[4][kW > 1 ? kW / 2 : 1];   // tokens 2c, 2c + 1, 2c + 8, 2c + 9
      if (kW == 1) {
        x[0][0] = *reinterpret_cast<const uint16_t*>(fa); x[1][0] = *reinterpret_cast<const uint16_t*>(fb);
        x[2][0] = *reinterpret_cast<const uint16_t*>(fa + 8 * kRow); x[3][0] = *reinterpret_cast<const uint16_t*>(fb + 8 * kRow);
      } else if (kW == 2) {
        x[0][0] = *reinterpret_cast<const uint32_t*>(fa); x[1][0] = *reinterpret_cast<const uint32_t*>(fb);
        x[2][0] = *reinterpret_cast<const uint32_t*>(fa + 8 * kRow); x[3][0] = *reinterpret_cast<const uint32_t*>(fb + 8 * kRow);
      } else {
        const uint2 x0 = *reinterpret_cast<const uint2*>(fa), x1 = *reinterpret_cast<const uint2*>(fb);
        const uint2 x2 = *reinterpret_cast<const uint2*>(fa + 8 * kRow), x3 = *reinterpret_cast<const uint2*>(fb + 8 * kRow);
        constexpr int k1 = kW > 2 ? 1 : 0;
        x[0][0] = x0.x; x[0][k1] = x0.y; x[1][0] = x1.x; x[1][k1] = x1.y;
        x[2][0] = x2.x; x[2][k1] = x2.y; x[3][0] = x3.x; x[3][k1] = x3.y;
      }
#pragma unroll
      for (int hh = 0; hh < kW; ++hh) {
        // four codes of each of two tokens, token pairs in the word's halves
        const uint32_t sel = (hh & 1) ? 0x7632 : 0x5410;
        const uint32_t u = __byte_perm(x[0][hh / 2], x[1][hh / 2], sel), v = __byte_perm(x[2][hh / 2], x[3][hh / 2], sel);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t uk = k ? u >> 8 : u, vk = k ? v >> 8 : v;
          const uint32_t y[4] = {EvenCentred(uk), OddCentred(uk), EvenCentred(vk), OddCentred(vk)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Mma(o[nt][(g * kW + hh) * 2 + k], y, b0[nt], b1[nt]);
        }
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();   // the rings become the warps' results

  // ---- join the warps
  constexpr int kRows = 8 * NT;
  float* s_o = reinterpret_cast<float*>(smem);                       // [warps][rows][DIM]
  float2* s_ml = reinterpret_cast<float2*>(s_o + kWarps * kRows * DIM);  // [warps][rows]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = e ? Y(l[nt]) : X(l[nt]);
      for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int row = warp * kRows + nt * 8 + 2 * c + e;
      if (r == 0) s_ml[row] = make_float2(m[nt][e], sum);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float z = e ? Y(zsum[nt][g]) : X(zsum[nt][g]);
        for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
#pragma unroll
        for (int x = 0; x < GROUP / 16; ++x) {
          const int d = g * GROUP + r * (GROUP / 8) + x * 2;
          *reinterpret_cast<float2*>(s_o + row * DIM + d) = make_float2(o[nt][g * (GROUP / 16) + x][e] + z, o[nt][g * (GROUP / 16) + x][e + 2] + z);
        }
      }
    }
  __syncthreads();
  const int64_t part_row = (int64_t(b) * a.c.kv_heads + kvh) * (int64_t(a.max_new) * a.share) + row0;
  for (int x = threadIdx.x; x < min(kRows, rows - row0) * (DIM / 2); x += kThreads) {
    const int row = x / (DIM / 2), d = 2 * (x - row * (DIM / 2));
    float top = kNone;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * kRows + row].x);
    float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = s_ml[w * kRows + row];
      const float f = PartWeight(ml.x, ml.y, top);
      const float2 v = *reinterpret_cast<const float2*>(s_o + (w * kRows + row) * DIM + d);
      sum = fmaf(ml.y, f, sum);
      v0 = fmaf(v.x, f, v0);
      v1 = fmaf(v.y, f, v1);
    }
    if (s.part_o != nullptr) {
      const int64_t at = (part_row + row) * s.chunks + blockIdx.x;
      *reinterpret_cast<float2*>(s.part_o + at * DIM + d) = make_float2(v0, v1);
      if (d == 0) s.part_ml[at] = make_float2(top, sum);
    } else {
      const int rr = row0 + row, i = int(QuickDiv(uint32_t(rr), a.div_share)), h = kvh * a.share + rr - i * a.share;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      StoreOut(a, s.bf16, (q.row0 + i) * a.ot + int64_t(h) * a.oh + d, v0 * inv);
      StoreOut(a, s.bf16, (q.row0 + i) * a.ot + int64_t(h) * a.oh + d + 1, v1 * inv);
    }
  }
}

// Joins the chunks of one query row: WARPS warps take them in turn, the parts are then added in the warps' order.
template <int DIM, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) JoinKernel(const __grid_constant__ StepArgs s) {
  constexpr int E = DIM / 32;
  constexpr int kBlockRows = WARPS == 1 ? 4 : 1;
  __shared__ float s_o[WARPS == 1 ? 1 : WARPS][WARPS == 1 ? 1 : DIM];
  __shared__ float s_l[WARPS];
  const AttnArgs& a = s.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = WARPS == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int max_rows = a.max_new * a.share;
  const int rr = int(blockIdx.x) * kBlockRows + (WARPS == 1 ? int(threadIdx.x >> 5) : 0), kvh = blockIdx.y, b = blockIdx.z;
  if (rr >= max_rows) return;
  const Seq q = SeqOf(a, b, false);
  if (rr >= q.nnew * a.share) return;
  const int i = int(QuickDiv(uint32_t(rr), a.div_share)), h = kvh * a.share + rr - i * a.share;
  const int begin = RowBegin(a, q, 0) & ~(kTile - 1), end = RowEnd(a, q, q.nnew - 1);
  const int chunks = end > begin ? (end - begin + s.chunk - 1) / s.chunk : 0;
  const int64_t at = ((int64_t(b) * a.c.kv_heads + kvh) * max_rows + rr) * s.chunks;
  float top = kNone;
  for (int x = lane; x < chunks; x += 32) top = fmaxf(top, s.part_ml[at + x].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  float o[E], sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int x = warp; x < chunks; x += WARPS) {
    const float2 ml = s.part_ml[at + x];
    float v[E];
    LoadVec<float, E>(s.part_o + (at + x) * DIM + lane * E, v);
    const float f = PartWeight(ml.x, ml.y, top);
    sum = fmaf(ml.y, f, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], f, o[e]);
  }
  const int64_t out = (q.row0 + i) * a.ot + int64_t(h) * a.oh;
  if (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) s_l[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += s_l[w];
    for (int d = threadIdx.x; d < DIM; d += WARPS * 32) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += s_o[w][d];
      StoreOut(a, s.bf16, out + d, sum == 0.f ? 0.f : v / sum);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) StoreOut(a, s.bf16, out + lane * E + e, sum == 0.f ? 0.f : o[e] / sum);
  }
}

struct Plan { int nt, row_tiles, chunk, chunks; };

Plan PlanSteps(const AttnArgs& a) {
  Plan p;
  const int rows = a.max_new * a.share;
  p.nt = rows > 8 && a.c.head_dim < 256 ? 2 : 1;   // 16 columns of 256 channels would not fit a thread's registers
  p.row_tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
  // tokens that the widest sequence's chunks cover
  int64_t span = std::min<int64_t>(a.max_kept, int64_t(a.table_cols) * a.c.page_size);
  if (a.window > 0) span = std::min<int64_t>(span, int64_t(a.window) + a.max_new + kTile);
  const int64_t units = int64_t(a.num_seqs) * a.c.kv_heads * p.row_tiles;
  const int64_t step = kTile * kWarps;
  const int64_t want = (span * units + 148 * 4 - 1) / (148 * 4);
  p.chunk = int(std::min<int64_t>(kMaxChunk, std::max<int64_t>(2 * step, (want + step - 1) / step * step)));
  p.chunks = int(std::max<int64_t>(1, (span + p.chunk - 1) / p.chunk));
  return p;
}

int64_t PartRows(const AttnArgs& a, const Plan& p) { return int64_t(a.num_seqs) * a.q_heads * a.max_new * p.chunks; }

template <typename K> int Prepare(K kernel, size_t smem) {
  if (smem > 48 * 1024) ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  return ITEXB_OK;
}

template <int DIM, int GROUP, int NT, bool PAGE16> int LaunchKernel(const StepArgs& s, cudaStream_t st) {
  constexpr size_t kStage = 2 * kTile * (DIM / 2) + 2 * kTile * (DIM / GROUP) * 4;
  constexpr size_t kRing = kWarps * kStages * kStage, kJoin = size_t(kWarps) * 8 * NT * (DIM * 4 + 8);
  constexpr size_t kSmem = kRing > kJoin ? kRing : kJoin;
  auto kernel = StepsKernel<DIM, GROUP, NT, PAGE16>;
  ITEXB_RETURN_IF_ERROR(Prepare(kernel, kSmem));
  kernel<<<dim3(s.chunks, s.a.c.kv_heads * s.row_tiles, s.a.num_seqs), kThreads, kSmem, st>>>(s);
  return CheckLaunch("StepsKernel");
}
template <int DIM, int WARPS> int LaunchJoin(const StepArgs& s, cudaStream_t st) {
  const int rows = s.a.max_new * s.a.share;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(WARPS == 1 ? (rows + 3) / 4 : rows, s.a.c.kv_heads, s.a.num_seqs);
  cfg.blockDim = dim3(WARPS == 1 ? 128 : WARPS * 32);
  cfg.stream = st;
  // starts while the last blocks of the steps run; it waits for their results itself
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ITEXB_CUDA(cudaLaunchKernelEx(&cfg, JoinKernel<DIM, WARPS>, s));
  return CheckLaunch("JoinKernel");
}
template <int DIM, int GROUP, int NT> int LaunchPage(const StepArgs& s, cudaStream_t st) {
  if (s.a.c.page_size % kTile == 0) return LaunchKernel<DIM, GROUP, NT, true>(s, st);
  return LaunchKernel<DIM, GROUP, NT, false>(s, st);
}
template <int DIM, int GROUP> int LaunchGroup(const StepArgs& s, int nt, cudaStream_t st) {
  if constexpr (GROUP <= DIM) {
    if constexpr (DIM < 256) {
      ITEXB_RETURN_IF_ERROR((nt == 1 ? LaunchPage<DIM, GROUP, 1>(s, st) : LaunchPage<DIM, GROUP, 2>(s, st)));
    } else {
      ITEXB_RETURN_IF_ERROR((LaunchPage<DIM, GROUP, 1>(s, st)));
    }
    if (s.part_o == nullptr) return ITEXB_OK;
    return s.chunks > 8 ? LaunchJoin<DIM, 8>(s, st) : LaunchJoin<DIM, 1>(s, st);
  } else {
    return SetError(ITEXB_INTERNAL, "kv4_attention: group above head_dim");
  }
}
template <int DIM> int LaunchDim(const StepArgs& s, int nt, cudaStream_t st) {
  if (s.a.c.group == 32) return LaunchGroup<DIM, 32>(s, nt, st);
  if (s.a.c.group == 64) return LaunchGroup<DIM, 64>(s, nt, st);
  return LaunchGroup<DIM, 128>(s, nt, st);
}
int LaunchType(const StepArgs& s, int nt, cudaStream_t st) {
  if (s.a.c.head_dim == 64) return LaunchDim<64>(s, nt, st);
  if (s.a.c.head_dim == 128) return LaunchDim<128>(s, nt, st);
  return LaunchDim<256>(s, nt, st);
}

}  // namespace

size_t StepsWorkspace(const AttnArgs& a) {
  const Plan p = PlanSteps(a);
  return p.chunks == 1 ? 0 : size_t(PartRows(a, p)) * (size_t(a.c.head_dim) * sizeof(float) + sizeof(float2));
}

int LaunchSteps(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st) {
  const Plan p = PlanSteps(a);
  ITEXB_REQUIRE(int64_t(a.c.kv_heads) * p.row_tiles <= 65535, ITEXB_INVALID_ARGUMENT, "kv4_attention: too many query rows");
  StepArgs s{};
  s.a = a;
  s.chunk = p.chunk;
  s.chunks = p.chunks;
  s.row_tiles = p.row_tiles;
  if (p.chunks > 1) {
    s.part_o = static_cast<float*>(workspace);
    s.part_ml = reinterpret_cast<float2*>(s.part_o + PartRows(a, p) * a.c.head_dim);
  }
  s.bf16 = dtype == ITEXB_DT_BFLOAT16;
  return LaunchType(s, p.nt, st);
}

}  // namespace itexb
