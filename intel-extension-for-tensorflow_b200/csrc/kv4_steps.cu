// Attention of few query rows over the 4-bit paged cache: decoding steps, drafted tokens.
//
// Bound: the cache's bytes (head_dim 128, groups of 64: 144 bytes per token and head, keys and values), as long as turning
// codes into operands stays cheap.  The codes themselves are multiplied, and the groups' ranges enter behind the products:
//     q . k_t = sum_g step_tg (sum_{d in g} q_d c_td) + lo_tg (sum_{d in g} q_d)
//     o_d     = sum_t (p_t step_tg) (c_td - 8) + sum_t p_t (lo_tg + 8 step_tg)
// A code needs no conversion: masked out where it lies, the word's low byte of each half reads as a subnormal half,
// c 2^-24 at bits 0-3 and 16 c 2^-24 at bits 4-7, which the tensor cores multiply exactly.  That is one mask per two codes
// and one shift per four.  The 16 is taken out of q beforehand and out of the output afterwards, the 2^24 is part of the scale.
// Codes count from the middle of their range (8 sum p step, by the same rounded weights, comes off at the end), so that
// the rounding of (p step) is relative to what a value differs from it.
// (A constant's mantissa or-ed around the code, 1024 + c, costs as much, and taking the constant out again either three
// digits, in sums over 128 Ki tokens, or an addition per two codes.)
// q enters as half: each row is scaled by a power of two to between 2^14 and 2^15, so that elements of 2^-24 of the row's largest
// and more stay exact (odd channels, over 16) and the others are off by 2^-35 of it.  p is kept at most 4 (see kRescale); p * step is a half
// times a power of two per group of channels that follows the largest step the warp has seen (see kLimitField): steps of any size
// fit, and a product is off by 2^-11 of itself or 2^-25 of the largest, 2^-40 of it where steps are alike.
//
// A warp owns tiles of 16 tokens and keeps its own running maximum, so warps meet only at the end of a block's part.  Both
// products run on mma.m16n8k16 with the cache as the 16-row operand (16 tokens, 16 channels) and up to 8 query rows of the
// key/value head as the 8 columns: S^T = K q^T, O^T += V^T P^T; the weights turn from the first one's accumulator layout into
// the second one's operand by an 8 x 8 transpose each.  Tensor cores of the tcgen05 kind want 64 or more rows, of which a
// decoding step has 1 to 8, and operands in shared memory; here the tensor work is a small part of the issue slots.  The
// order of channels inside a product is free, so lanes take them as the codes lie in a word.
// Tiles come in through per-warp rings of cp.async copies (three tiles in flight per warp, sixteen or more warps per SM); the
// 16-byte pieces are permuted so that both products read them without bank conflicts.
// The grid is one wave of resident blocks.  The tiles of all sequences and heads form one list, sequence after sequence, of
// which every block takes an equal, contiguous part; a (sequence, head) that ends inside a block's part is written by it, the
// others are joined from at most one result per block by a second kernel.  (One block per 2048 tokens instead left a fifth of
// the machine idle behind the longest contexts, and smaller chunks cost more at their ends than they evened out.)
// Measured, single tokens, 32 / 8 heads of 128, groups of 64: 64 sequences up to 8192 (421 MB) 104 us, 4.0 TB/s; bound by issue slots (58 % busy) and the dependent steps of a tile with three warps per scheduler.
#include <algorithm>

#include "kv4_attention.h"

namespace itexb {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTile = 16;                       // tokens
constexpr int kMaxBlocks = 740;                 // five per SM of a 148-SM device
constexpr int kLeastTiles = 8;                  // of a block's part, where there is little work: 5 sequences of up to 700
                                                // tokens take 14.4 us on the device with 4 or 8, 14.6 with 16
constexpr float kRescale = 4.f;                 // scores may pass the running maximum by 4 before it moves,
constexpr float kShift = 2.f;                   // so weights are 2^(score - maximum - 2), at most 4
constexpr float kNone = -3.0e38f;               // the maximum of no scores or products
constexpr float kFarthest = 2.9e38f;            // magnitude of a maximum of some scores at most

// Limits of a group's steps, as the word (lo, step) of a step they stay below: 2^26 times a half's exponent bits, so with 2^E the
// limit, its steps are multiplied by 2^(13 - E), products with weights up to 4 are below 2^15.  A step that reaches the limit moves
// it to 8 to 16 times the largest step.
constexpr uint32_t kLimitField = 26, kLimitMost = 31u << kLimitField;   // 2^16: no step reaches it
__device__ __forceinline__ float LiftOf(uint32_t limit) { return __uint_as_float((155u << 23) - (limit >> 3)); }        // 2^(13 - E)
__device__ __forceinline__ float UnitOf(uint32_t limit) { return __uint_as_float((123u << 23) + (limit >> 3)); }        // 2^24 / 2^(13 - E)
__device__ __forceinline__ float Dropped(uint32_t from, uint32_t to) { return __uint_as_float((127u << 23) - ((to - from) >> 3)); }

struct StepArgs {
  AttnArgs a;
  int row_tiles, units;      // 8 NT query rows each; units of a sequence: kv_heads * row_tiles
  int bf16;                  // type of q and out, else half
  float* part_o;             // [blocks][2][8 NT][head_dim]: a unit begun by an earlier block, a unit left to the next one
  float2* part_ml;           // [blocks][2][8 NT] (maximum, sum)
  int64_t* list;             // [2 + seqs]: tiles in all, blocks at work, tiles before each sequence
};

// Tiles that the new tokens of a sequence see.
__device__ __forceinline__ int SeqTiles(const AttnArgs& a, const Seq& q) {
  if (q.nnew == 0) return 0;
  const int begin = RowBegin(a, q, 0) & ~(kTile - 1), end = RowEnd(a, q, q.nnew - 1);
  return end > begin ? (end - begin + kTile - 1) / kTile : 0;
}
__device__ __forceinline__ int64_t BlockStart(int64_t total, int64_t blocks, int64_t block) { return total * block / blocks; }

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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <int WORDS> __device__ __forceinline__ void Lds(uint32_t (&w)[WORDS], const uint8_t* at) {
  if constexpr (WORDS == 1) w[0] = *reinterpret_cast<const uint32_t*>(at);
  else if constexpr (WORDS == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    w[0] = x.x; w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(at + 4 * i);
      w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
    }
  }
}
__device__ __forceinline__ float2 Pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ void MmaFromZero(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// The codes of a word's nibbles 0 and 4 as halves c 2^-24, of 1 and 5 as 16 c 2^-24; nibbles 2, 6, 3, 7: of w >> 8.
__device__ __forceinline__ uint32_t EvenCodes(uint32_t w) { return w & 0x000F000Fu; }
__device__ __forceinline__ uint32_t OddCodes(uint32_t w) { return w & 0x00F000F0u; }
constexpr uint32_t kMiddle = 0x00080008u;      // the code 8
constexpr float kUnit = 16777216.f;            // 2^24
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Partial results of four warps (or of several blocks) with maxima m and sums l: what the part's values are weighed with.
__device__ __forceinline__ float PartWeight(float m, float l, float top) { return m <= kNone ? (isnan(l) ? l : 0.f) : Exp2(m - top); }

__device__ __forceinline__ void StoreOut(const AttnArgs& a, int bf16, int64_t at, float v) {
  if (bf16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(a.out)[at] = __float2half_rn(v);
}

// PAGE16: pages hold a multiple of 16 tokens, so a tile lies in one page.
// (The comparisons here and below are of before steps were scaled, which costs each side 1 to 3 %.)
// At least so many blocks share an SM (registers).  head_dim 64 with 4 and with 5 (spills): 35, 47 us for 24 sequences of 3000 with
// 5 tokens each; with 3 and with 4 where a tile of rows has 16 (12 tokens each): 50, 52.
template <int DIM, int GROUP, int NT> constexpr int kShareSm = DIM == 64 ? (NT == 1 ? 4 : 3) : DIM == 128 ? (NT == 1 ? 3 : 2) : 2;
// Tiles a warp works on at a time.  Two give each other something to do and share the bookkeeping, but cost registers and so
// warps.  Measured with one and with two: head_dim 128, 64 sequences up to 8192 110, 103 us, one of 131072 48, 44; head_dim 64,
// 24 sequences of 3000 with 5 tokens each 35, 39 us (groups of 64: 31, 36), 64 sequences with one each 72, 76.
template <int DIM, int NT> constexpr int kTogether = DIM == 128 && NT == 1 ? 2 : 1;
template <int DIM, int NT> constexpr int kStagesOf = kTogether<DIM, NT> == 2 ? 3 : 4;

template <int DIM, int GROUP, int NT, bool PAGE16>
__global__ void __launch_bounds__(kThreads, kShareSm<DIM, GROUP, NT>) StepsKernel(const __grid_constant__ StepArgs s) {
  constexpr int NG = DIM / GROUP;
  constexpr int kRow = DIM / 2, kPieces = DIM / 32;
  constexpr int kCodes = kTile * kRow, kPars = kTile * NG * 4;
  constexpr int TT = kTogether<DIM, NT>, kStages = kStagesOf<DIM, NT>;
  constexpr int kTileBytes = 2 * kCodes + 2 * kPars, kStage = TT * kTileBytes;
  constexpr int kW = GROUP / 32;                 // words of codes per lane, group and row (keys); halves (values)
  const AttnArgs& a = s.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_ok[kWarps][kStages];          // rows of a tile that are there
  __shared__ longlong2 s_from[kWarps][32];            // PAGE16: where the next tiles' codes and params begin, from a page on
  __shared__ int64_t s_sum[kWarps];
  __shared__ int64_t s_pos, s_stop, s_rest;           // place in the list, its end for this block; tiles of sequence s_seq before it
  __shared__ int s_seq;
  __shared__ Seq s_q;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, c = lane & 3;

  // Launched programmatically: what the previous kernel of the stream wrote is visible from here on.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // ---- this block's part of the list of tiles
  {
    const int per = (a.num_seqs + kThreads - 1) / kThreads;
    const int b0 = min(a.num_seqs, int(threadIdx.x) * per), b1 = min(a.num_seqs, b0 + per);
    Seq one{};              // of sequence b0: the only one of this thread where there are at most 128
    int64_t sum = 0;
    for (int x = b0; x < b1; ++x) {
      const Seq q = SeqOf(a, x, blockIdx.x == 0);
      if (x == b0) one = q;
      sum += int64_t(SeqTiles(a, q)) * s.units;
    }
    int64_t before = sum;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, before, x);
      if (lane >= x) before += y;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
    }
    before -= sum;
    const int64_t blocks = max(int64_t(1), min(int64_t(gridDim.x), total / kLeastTiles));
    const int64_t pos = BlockStart(total, blocks, blockIdx.x);
    const int64_t stop = blockIdx.x < blocks ? BlockStart(total, blocks, blockIdx.x + 1) : pos;
    if (threadIdx.x == 0) { s_pos = pos; s_stop = stop; }
    const bool mine = pos >= before && pos < before + sum;
    if (mine || blockIdx.x == 0) {
      if (threadIdx.x == 0 && blockIdx.x == 0) { s.list[0] = total; s.list[1] = blocks; }   // for the joining kernel
      int64_t at = before;
      for (int x = b0; x < b1; ++x) {
        const Seq q = x == b0 ? one : SeqOf(a, x, false);
        const int64_t n = int64_t(SeqTiles(a, q)) * s.units;
        if (blockIdx.x == 0) s.list[2 + x] = at;
        if (mine && pos >= at && pos < at + n) {
          s_seq = x;
          s_q = q;
          s_rest = pos - at;
        }
        at += n;
      }
    }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  constexpr int kCopies = kPieces * kTile / 32;
  uint32_t put[kCopies];
#pragma unroll
  for (int x = 0; x < kCopies; ++x) put[x] = PieceAt<DIM>((x * 32 + lane) / kPieces, (x * 32 + lane) % kPieces);
  const uint32_t put_pars = 2 * kCodes + lane * (NG * 4);   // keys' rows, then values'
  const int64_t lane_step = int64_t(32 / kPieces) * a.c.ct;
  const uint32_t ring = warp * (kStages * kStage), ring_addr = uint32_t(__cvta_generic_to_shared(smem)) + ring;

  while (s_pos < s_stop) {
  const int b = s_seq;
  const Seq q = s_q;
  const int tiles = SeqTiles(a, q);      // not 0
  const int64_t rest = s_rest;
  const int unit = int(rest / tiles);
  const int tile0 = int(rest - int64_t(unit) * tiles), tile1 = int(min(int64_t(tiles), tile0 + (s_stop - s_pos)));
  __syncthreads();
  if (threadIdx.x == 0) {
    s_pos += tile1 - tile0;
    s_rest = rest + (tile1 - tile0);
    if (s_rest == int64_t(tiles) * s.units && s_pos < s_stop) {   // on to the next sequence that has any
      int x = b + 1;
      Seq next = SeqOf(a, x, false);
      while (SeqTiles(a, next) == 0) next = SeqOf(a, ++x, false);
      s_seq = x;
      s_q = next;
      s_rest = 0;
    }
  }
  const int kvh = unit / s.row_tiles, rt = unit - kvh * s.row_tiles;
  const int rows = q.nnew * a.share, row0 = rt * 8 * NT;
  if (row0 >= rows) {   // a sequence shorter than the longest has fewer row tiles
    __syncthreads();
    continue;
  }
  // the tokens that some row of this unit sees, and those that all of them see
  const int i_first = int(QuickDiv(uint32_t(row0), a.div_share)), i_last = int(QuickDiv(uint32_t(min(rows, row0 + 8 * NT) - 1), a.div_share));
  const int some_begin = RowBegin(a, q, i_first), some_end = RowEnd(a, q, i_last);
  const int all_begin = RowBegin(a, q, i_last), all_end = RowEnd(a, q, i_first);
  const int begin = (RowBegin(a, q, 0) & ~(kTile - 1)) + tile0 * kTile;
  const int ntiles = tile1 - tile0;

  // ---- steps of TT tiles: w, w + 4, ...
  const int nsteps = (ntiles + TT - 1) / TT;
  const int mine = nsteps > warp ? (nsteps - warp + kWarps - 1) / kWarps : 0;
  const int32_t* table = a.table + int64_t(b) * a.table_stride;
  const uint8_t* kcodes = a.c.k_codes + int64_t(kvh) * a.c.ch;
  const uint8_t* vcodes = a.c.v_codes + int64_t(kvh) * a.c.ch;
  const uint8_t* pars = reinterpret_cast<const uint8_t*>((lane < 16 ? a.c.k_params : a.c.v_params) + int64_t(kvh) * a.c.ph);
  if (PAGE16) {  // this lane's first piece of a tile, its row's params
    kcodes += int64_t(lane / kPieces) * a.c.ct + (lane % kPieces) * 16;
    vcodes += int64_t(lane / kPieces) * a.c.ct + (lane % kPieces) * 16;
    pars += int64_t(lane & 15) * a.c.pt * 4;
  }
  uint32_t there = 0;   // PAGE16: of the next 32 tiles, those whose page exists and that some row sees

  auto issue = [&](int n, int stage) {
    const uint32_t to = ring_addr + stage * kStage;
    uint32_t rows_there = 0;
    if (PAGE16) {
      constexpr int kAhead = 32 / TT;
      if (n % kAhead == 0) {   // a lane looks up the page of one of the next 32 tiles
        __syncwarp();
        longlong2 from = make_longlong2(0, 0);
        bool ok = false;
        const int tile = (warp + (n + lane / TT) * kWarps) * TT + lane % TT, j0 = begin + tile * kTile;
        if (tile < ntiles && j0 + kTile > some_begin && j0 < some_end) {
          const int col = int(QuickDiv(uint32_t(j0), a.c.div_page)), off = j0 - col * a.c.page_size;
          const int page = __ldg(table + col);
          ok = page >= 0 && page < a.c.num_pages;
          if (ok) from = make_longlong2(int64_t(page) * a.c.cp + int64_t(off) * a.c.ct, (int64_t(page) * a.c.pp + int64_t(off) * a.c.pt) * 4);
          else ReportIndex(a.status_word);
        }
        s_from[warp][lane] = from;
        there = __ballot_sync(0xffffffffu, ok);
        __syncwarp();
      }
#pragma unroll
      for (int h = 0; h < TT; ++h) {
        const int at = (n % kAhead) * TT + h;
        if ((there >> at) & 1u) {
          const uint32_t dst = to + h * kTileBytes;
          const longlong2 from = s_from[warp][at];
          const uint8_t *k = kcodes + from.x, *v = vcodes + from.x, *p = pars + from.y;
#pragma unroll
          for (int x = 0; x < kCopies; ++x) {
            CpAsync<16>(dst + put[x], k);
            CpAsync<16>(dst + kCodes + put[x], v);
            k += lane_step;
            v += lane_step;
          }
          if (NG <= 4) CpAsync<(NG > 4 ? 4 : NG) * 4>(dst + put_pars, p);
          else { CpAsync<16>(dst + put_pars, p); CpAsync<16>(dst + put_pars + 16, p + 16); }
          rows_there |= 0xffffu << (16 * h);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < TT; ++h) {
        const uint32_t dst = to + h * kTileBytes;
        const int tile = (warp + n * kWarps) * TT + h;
        int page = -1, off = 0;
        const int j = begin + tile * kTile + (lane & 15);
        if (tile < ntiles && j >= some_begin && j < some_end) {
          const int col = int(QuickDiv(uint32_t(j), a.c.div_page));
          off = j - col * a.c.page_size;
          page = __ldg(table + col);
          if (page < 0 || page >= a.c.num_pages) {
            ReportIndex(a.status_word);
            page = -1;
          }
        }
        rows_there |= (__ballot_sync(0xffffffffu, page >= 0) & 0xffffu) << (16 * h);
#pragma unroll
        for (int x = 0; x < kCopies; ++x) {
          const int row = (x * 32 + lane) / kPieces, piece = (x * 32 + lane) % kPieces;
          const int pg = __shfl_sync(0xffffffffu, page, row), of = __shfl_sync(0xffffffffu, off, row);
          if (pg >= 0) {
            const int64_t from = int64_t(pg) * a.c.cp + int64_t(of) * a.c.ct + piece * 16;
            CpAsync<16>(dst + put[x], kcodes + from);
            CpAsync<16>(dst + kCodes + put[x], vcodes + from);
          }
        }
        if (page >= 0) {
          const uint8_t* p = pars + (int64_t(page) * a.c.pp + int64_t(off) * a.c.pt) * 4;
          if (NG <= 4) CpAsync<(NG > 4 ? 4 : NG) * 4>(dst + put_pars, p);
          else { CpAsync<16>(dst + put_pars, p); CpAsync<16>(dst + put_pars + 16, p + 16); }
        }
      }
    }
    if (lane == 0) s_ok[warp][stage] = rows_there;
  };

#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) {
    if (n < mine) issue(n, n);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // ---- query rows as the 8-column operand, and their sums per group times 2^-24
  uint32_t qf[NT][DIM / 16][2];
  F2 qs[NT][NG], scale[NT];              // of columns 2c, 2c + 1
  int lo[NT][2], hi[NT][2];              // visible tokens of those columns
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int rr = row0 + nt * 8 + r;
    const bool on = rr < rows;
    const int i = int(QuickDiv(uint32_t(on ? rr : row0), a.div_share)), h = (on ? rr : row0) - i * a.share;
    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (q.row0 + i) * a.qt + int64_t(kvh * a.share + h) * a.qh;
    union Piece { uint4 v; uint32_t u[4]; uint16_t e[8]; } x[NG][kW];
    uint32_t bits = 0;
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
#pragma unroll
        for (int e = 0; e < 4; ++e) bits = MaxBits2(x[g][w].u[e], bits);
      }
    // q * down is exact but for underflow; scores are (codes' product) * up, up > 0
    float down = a.scale_log2 < 0.f ? -1.f : (a.scale_log2 == 0.f ? 0.f : 1.f), up = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
    bits = MaxBits2(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = MaxBits2(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    const float2 most2 = QueryPair(bits, s.bf16);
    const float most = most2.x > most2.y ? most2.x : most2.y;      // NaN: nothing to scale
    if (most > 0.f && most < INFINITY) {
      const int e = max(int(__float_as_uint(most) >> 23), 15);
      down *= __uint_as_float(uint32_t(268 - e) << 23);            // 2^(14 - exponent)
      up = fmaxf(up * __uint_as_float(uint32_t(e - 14) << 23), 1e-37f);
    }
    up = fminf(up * kUnit, -kNone);
    scale[nt] = Make2(__shfl_sync(0xffffffffu, up, (2 * c) * 4), __shfl_sync(0xffffffffu, up, (2 * c + 1) * 4));
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        Piece& y = x[g][w];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 in = QueryPair(y.u[e], s.bf16);
          y.u[e] = PackHalf(in.x * down, in.y * down);
          const float2 f = Pair(y.u[e]);
          sum += f.x + f.y;
          asm("mul.f16x2 %0, %0, %1;" : "+r"(y.u[e]) : "r"(0x2C003C00u));   // odd channels by 1/16
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
      sum *= 1.f / kUnit;
      qs[nt][g] = Make2(__shfl_sync(0xffffffffu, sum, (2 * c) * 4), __shfl_sync(0xffffffffu, sum, (2 * c + 1) * 4));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int ii = int(QuickDiv(uint32_t(min(rows - 1, row0 + nt * 8 + 2 * c + e)), a.div_share));  // a column without a row: any bounds
      lo[nt][e] = RowBegin(a, q, ii);
      hi[nt][e] = RowEnd(a, q, ii);
    }
  }

  float o[NT][DIM / 16][4], middle[NT][NG][4];   // sums times 2^-24 and the group's lift; the odd channels' (2, 3) are 16 times as large
  F2 zsum[NT][NG], l[NT];
  uint32_t limit[NG];          // of the steps of values; the o and middle of a group are times LiftOf it
  F2 under[NT];                // -(running maximum) of the products: taken off before they are scaled, which is exact for scores of any size
#pragma unroll
  for (int g = 0; g < NG; ++g) limit[g] = 0u;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int x = 0; x < DIM / 16; ++x) o[nt][x][0] = o[nt][x][1] = o[nt][x][2] = o[nt][x][3] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      zsum[nt][g] = Same2(0.f);
      middle[nt][g][0] = middle[nt][g][1] = middle[nt][g][2] = middle[nt][g][3] = 0.f;
    }
    under[nt] = Same2(-kNone);
    l[nt] = Same2(0.f);
  }

  // where this lane reads in a tile; a group further is another piece of the same row (an xor, see PieceAt)
  const uint32_t key_at = PieceAt<DIM>(r, c * (GROUP / 8) / 16) + c * (GROUP / 8) % 16;
  const uint32_t value_at0 = kCodes + PieceAt<DIM>(2 * c, r * (GROUP / 16) / 16) + r * (GROUP / 16) % 16;
  const uint32_t value_at1 = kCodes + PieceAt<DIM>(2 * c + 1, r * (GROUP / 16) / 16) + r * (GROUP / 16) % 16;
  const uint32_t pars_at = 2 * kCodes + r * (NG * 4);
  // Moves the limits of groups whose finite steps reach them.
  auto raise = [&](auto part, const uint32_t st, const int j0, const uint32_t ok) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t most = 0;
#pragma unroll
      for (int x = 0; x < 2 * TT; ++x) {
        const int in = (x >> 1) * kTile + (x & 1) * 8 + r, j = j0 + in;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + st + (x >> 1) * kTileBytes + pars_at + kPars + (x & 1) * (8 * NG * 4) + 4 * g) & 0x7fffffffu;
        if (w < kLimitMost && (!decltype(part)::value || (((ok >> in) & 1u) != 0u && j >= some_begin && j < some_end))) most = max(most, w);
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 4));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
      const uint32_t to = most >= limit[g] ? min((most >> kLimitField) + 4u, 31u) << kLimitField : limit[g];
      const float f = Dropped(limit[g], to);
      limit[g] = to;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        middle[nt][g][0] *= f; middle[nt][g][1] *= f;
#pragma unroll
        for (int x = g * (GROUP / 16); x < (g + 1) * (GROUP / 16); ++x) { o[nt][x][0] *= f; o[nt][x][1] *= f; o[nt][x][2] *= f; o[nt][x][3] *= f; }
      }
    }
  };
  auto compute = [&](auto part, const uint32_t st, const int j0, const uint32_t ok) {
    float t[TT][NT][4];
    uint32_t seen = 0xffffffffu;     // bit 16 h + 4 nt + 2 * (token r + 8) + column
#pragma unroll
    for (int h = 0; h < TT; ++h) {
    const uint32_t sh = st + h * kTileBytes;
    // ---- scores of tokens r, r + 8 and columns 2c, 2c + 1
    uint32_t kp0[NG], kp1[NG];
    Lds<NG>(kp0, smem + sh + pars_at);
    Lds<NG>(kp1, smem + sh + pars_at + 8 * NG * 4);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t w0[kW], w1[kW];
      const uint8_t* from = smem + ((sh + key_at) ^ (g * (GROUP / 2)));
      Lds<kW>(w0, from);
      Lds<kW>(w1, from + 8 * kRow);
      float acc[NT][4];
#pragma unroll
      for (int w = 0; w < kW; ++w) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t u0 = half ? w0[w] >> 8 : w0[w], u1 = half ? w1[w] >> 8 : w1[w];
          const uint32_t x[4] = {EvenCodes(u0), EvenCodes(u1), OddCodes(u0), OddCodes(u1)};
          const int ks = (g * kW + w) * 2 + half;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (w == 0 && half == 0) MmaFromZero(acc[nt], x, qf[nt][ks][0], qf[nt][ks][1]);
            else Mma(acc[nt], x, qf[nt][ks][0], qf[nt][ks][1]);
          }
        }
      }
      const float2 p0 = Pair(kp0[g]), p1 = Pair(kp1[g]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float qsum = e & 1 ? Y(qs[nt][g]) : X(qs[nt][g]);
          const float2 p = e < 2 ? p0 : p1;
          t[h][nt][e] = fmaf(p.y, acc[nt][e], g == 0 ? p.x * qsum : fmaf(p.x, qsum, t[h][nt][e]));
        }
    }

    // ---- masks
    if constexpr (decltype(part)::value) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int in = r + 8 * k, j = j0 + h * kTile + in;
          const bool there = ((ok >> (16 * h + in)) & 1u) != 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!there || j < lo[nt][e] || j >= hi[nt][e]) {
              seen &= ~(1u << (16 * h + 4 * nt + 2 * k + e));
              t[h][nt][2 * k + e] = -INFINITY;
            }
        }
    }
    }
    // ---- the running maximum, moved only when a score passes it by more than kRescale
    F2 d[TT][NT][2];
    float over = -INFINITY;
#pragma unroll
    for (int h = 0; h < TT; ++h)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          d[h][nt][k] = Fma2(Add2(Make2(t[h][nt][2 * k], t[h][nt][2 * k + 1]), under[nt]), scale[nt], Same2(-kShift));
          over = fmaxf(over, fmaxf(X(d[h][nt][k]), Y(d[h][nt][k])));
        }
    if (__any_sync(0xffffffffu, over > kRescale - kShift)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2], to[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float was = e ? Y(under[nt]) : X(under[nt]);
          float top = -INFINITY;
#pragma unroll
          for (int h = 0; h < TT; ++h) top = fmaxf(top, fmaxf(t[h][nt][e], t[h][nt][e + 2]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          to[e] = fminf(was, -top);
          f[e] = Exp2((to[e] - was) * (e ? Y(scale[nt]) : X(scale[nt])));
        }
        under[nt] = Make2(to[0], to[1]);
        const F2 f2 = Make2(f[0], f[1]);
        l[nt] = Mul2(l[nt], f2);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          zsum[nt][g] = Mul2(zsum[nt][g], f2);
          middle[nt][g][0] *= f[0]; middle[nt][g][1] *= f[1];   // all its rows are alike; (2, 3) are never read
        }
#pragma unroll
        for (int x = 0; x < DIM / 16; ++x) { o[nt][x][0] *= f[0]; o[nt][x][1] *= f[1]; o[nt][x][2] *= f[0]; o[nt][x][3] *= f[1]; }
#pragma unroll
        for (int h = 0; h < TT; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            d[h][nt][k] = Fma2(Add2(Make2(t[h][nt][2 * k], t[h][nt][2 * k + 1]), under[nt]), scale[nt], Same2(-kShift));
      }
    }
#pragma unroll
    for (int h = 0; h < TT; ++h)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[h][nt][e] = Exp2(e & 1 ? Y(d[h][nt][e >> 1]) : X(d[h][nt][e >> 1]));
        l[nt] = Add2(l[nt], Add2(Make2(t[h][nt][0], t[h][nt][1]), Make2(t[h][nt][2], t[h][nt][3])));
      }

    // ---- steps of values, of tokens that some row sees, against the limits
    uint32_t most[NG];
#pragma unroll
    for (int h = 0; h < TT; ++h) {
      bool in0 = true, in1 = true;
      if constexpr (decltype(part)::value) {
        const int j = j0 + h * kTile + r;
        in0 = ((ok >> (16 * h + r)) & 1u) != 0u && j >= some_begin && j < some_end;
        in1 = ((ok >> (16 * h + r + 8)) & 1u) != 0u && j + 8 >= some_begin && j + 8 < some_end;
      }
      uint32_t vp0[NG], vp1[NG];
      Lds<NG>(vp0, smem + st + h * kTileBytes + pars_at + kPars);
      Lds<NG>(vp1, smem + st + h * kTileBytes + pars_at + kPars + 8 * NG * 4);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t x = max(in0 ? vp0[g] : 0u, in1 ? vp1[g] : 0u);
        most[g] = h == 0 ? x : max(most[g], x);
      }
    }
    bool reached = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) reached = reached || most[g] >= limit[g];
    if (__any_sync(0xffffffffu, reached)) raise(part, st, j0, ok);
#pragma unroll
    for (int h = 0; h < TT; ++h) {
    const uint32_t sh = st + h * kTileBytes;
    // ---- values: weights times the group's steps as the 8-column operand, codes of 16 channels as rows
    uint32_t vp0[NG], vp1[NG];
    Lds<NG>(vp0, smem + sh + pars_at + kPars);
    Lds<NG>(vp1, smem + sh + pars_at + kPars + 8 * NG * 4);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float2 p0 = Pair(vp0[g]), p1 = Pair(vp1[g]);
      const float lift = LiftOf(limit[g]), step0 = p0.y * lift, step1 = p1.y * lift;
      uint32_t b0[NT], b1[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mid[2] = {fmaf(8.f, p0.y, p0.x), fmaf(8.f, p1.y, p1.x)};
        float w[4];
        if constexpr (decltype(part)::value) {  // an unseen row's lo and step may be anything
          float z[2] = {X(zsum[nt][g]), Y(zsum[nt][g])};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool on = ((seen >> (16 * h + 4 * nt + e)) & 1u) != 0u;
            w[e] = on ? t[h][nt][e] * (e < 2 ? step0 : step1) : 0.f;
            z[e & 1] = on ? fmaf(t[h][nt][e], mid[e >> 1], z[e & 1]) : z[e & 1];
          }
          zsum[nt][g] = Make2(z[0], z[1]);
        } else {
          const F2 t0 = Make2(t[h][nt][0], t[h][nt][1]), t1 = Make2(t[h][nt][2], t[h][nt][3]);
          const F2 w0 = Mul2(t0, Same2(step0)), w1 = Mul2(t1, Same2(step1));
          w[0] = X(w0); w[1] = Y(w0); w[2] = X(w1); w[3] = Y(w1);
          zsum[nt][g] = Fma2(t1, Same2(mid[1]), Fma2(t0, Same2(mid[0]), zsum[nt][g]));
        }
        b0[nt] = Transpose8x8(PackHalf(w[0], w[1]));
        b1[nt] = Transpose8x8(PackHalf(w[2], w[3]));
        const uint32_t eights[4] = {kMiddle, kMiddle, kMiddle, kMiddle};
        Mma(middle[nt][g], eights, b0[nt], b1[nt]);
      }
      const uint8_t *fa = smem + ((sh + value_at0) ^ (g * (GROUP / 2))), *fb = smem + ((sh + value_at1) ^ (g * (GROUP / 2)));
      uint32_t x[4][kW > 1 ? kW / 2 : 1];   // tokens 2c, 2c + 1, 2c + 8, 2c + 9
      if constexpr (kW == 1) {
        x[0][0] = *reinterpret_cast<const uint16_t*>(fa); x[1][0] = *reinterpret_cast<const uint16_t*>(fb);
        x[2][0] = *reinterpret_cast<const uint16_t*>(fa + 8 * kRow); x[3][0] = *reinterpret_cast<const uint16_t*>(fb + 8 * kRow);
      } else {
        Lds<kW / 2>(x[0], fa); Lds<kW / 2>(x[1], fb); Lds<kW / 2>(x[2], fa + 8 * kRow); Lds<kW / 2>(x[3], fb + 8 * kRow);
      }
#pragma unroll
      for (int hh = 0; hh < kW; ++hh) {
        // four codes of each of two tokens, token pairs in the word's halves
        const uint32_t sel = (hh & 1) ? 0x7632 : 0x5410;
        const uint32_t u = __byte_perm(x[0][hh / 2], x[1][hh / 2], sel), v = __byte_perm(x[2][hh / 2], x[3][hh / 2], sel);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t uk = k ? u >> 8 : u, vk = k ? v >> 8 : v;
          const uint32_t y[4] = {EvenCodes(uk), OddCodes(uk), EvenCodes(vk), OddCodes(vk)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) Mma(o[nt][(g * kW + hh) * 2 + k], y, b0[nt], b1[nt]);
        }
      }
    }
    }
  };

  for (int n = 0, stage = 0; n < mine; ++n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    if (n + kStages - 1 < mine) issue(n + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const uint32_t st = ring + stage * kStage;
    const int j0 = begin + (warp + n * kWarps) * (TT * kTile);
    const uint32_t ok = s_ok[warp][stage];
    constexpr uint32_t kAll = TT == 2 ? 0xffffffffu : 0xffffu;

    // two copies of the code: tiles that not every row sees whole carry masks
    if (ok == kAll && j0 >= all_begin && j0 + TT * kTile <= all_end) compute(std::false_type{}, st, j0, ok);
    else if (ok != 0u) compute(std::true_type{}, st, j0, ok);
    __syncwarp();
    stage = stage == kStages - 1 ? 0 : stage + 1;
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
      const float top = -(e ? Y(under[nt]) : X(under[nt]));
      if (r == 0) s_ml[row] = make_float2(top <= kNone ? kNone : fminf(fmaxf(top * (e ? Y(scale[nt]) : X(scale[nt])), -kFarthest), kFarthest), sum);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float unit = UnitOf(limit[g]);
        float z = e ? Y(zsum[nt][g]) : X(zsum[nt][g]);
        for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
#pragma unroll
        for (int x = 0; x < GROUP / 16; ++x) {
          const int d = g * GROUP + r * (GROUP / 8) + x * 2;
          const float *v = o[nt][g * (GROUP / 16) + x];
          *reinterpret_cast<float2*>(s_o + row * DIM + d) =
              make_float2(fmaf(v[e] - middle[nt][g][e], unit, z), fmaf(fmaf(v[e + 2], 0.0625f, -middle[nt][g][e]), unit, z));
        }
      }
    }
  __syncthreads();
  const bool whole = ntiles == tiles;
  const int64_t part = (int64_t(blockIdx.x) * 2 + (tile0 == 0)) * kRows;
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
    if (!whole) {
      *reinterpret_cast<float2*>(s.part_o + (part + row) * DIM + d) = make_float2(v0, v1);
      if (d == 0) s.part_ml[part + row] = make_float2(top, sum);
    } else {
      const int rr = row0 + row, i = int(QuickDiv(uint32_t(rr), a.div_share)), h = kvh * a.share + rr - i * a.share;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at = (q.row0 + i) * a.ot + int64_t(h) * a.oh + d;
      StoreOut(a, s.bf16, at, v0 * inv);
      StoreOut(a, s.bf16, at + 1, v1 * inv);
    }
  }
  __syncthreads();   // the results become rings again
  }
}

// Joins one query row of a unit that several blocks worked on: WARPS warps take the blocks' results in turn, the warps' sums
// are then added in their order.  Rows that see nothing are set to zero here.
template <int DIM, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) JoinKernel(const __grid_constant__ StepArgs s) {
  constexpr int E = DIM / 32;
  constexpr int kBlockRows = WARPS == 1 ? 4 : 1;
  __shared__ float s_o[WARPS == 1 ? 1 : WARPS][WARPS == 1 ? 1 : DIM];
  __shared__ float s_l[WARPS];
  const AttnArgs& a = s.a;
  const int warp = WARPS == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rr = int(blockIdx.x) * kBlockRows + (WARPS == 1 ? int(threadIdx.x >> 5) : 0), kvh = blockIdx.y, b = blockIdx.z;
  const Seq q = SeqOf(a, b, false);
  const int tiles = SeqTiles(a, q);
  asm volatile("griddepcontrol.wait;" ::: "memory");   // every block, so that this kernel does not end before the first one
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (rr >= q.nnew * a.share) return;
  const int row = rr % (8 * NT);
  int64_t c0 = 0, c1 = -1;
  if (tiles > 0) {
    const int64_t total = s.list[0], blocks = s.list[1];
    const int64_t x = s.list[2 + b] + (int64_t(kvh) * s.row_tiles + rr / (8 * NT)) * tiles;
    c0 = ((x + 1) * blocks - 1) / total;              // the block that holds tile x
    c1 = ((x + tiles) * blocks - 1) / total;
    if (c0 == c1) return;                             // it wrote the row
  }
  const int parts = int(c1 - c0) + 1;
  // the unit begins in block c0 (its second result) and goes on in the others (their first)
  auto at = [&](int i) { return ((c0 + i) * 2 + (i == 0)) * (8 * NT) + row; };
  float top = kNone;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, s.part_ml[at(i)].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  float o[E], sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = warp; i < parts; i += WARPS) {
    const float2 ml = s.part_ml[at(i)];
    float v[E];
    constexpr int kPiece = E < 4 ? E : 4;
#pragma unroll
    for (int e = 0; e < E; e += kPiece) {
      float x[kPiece];
      LoadVec<float, kPiece>(s.part_o + at(i) * DIM + lane * E + e, x);
#pragma unroll
      for (int k = 0; k < kPiece; ++k) v[e + k] = x[k];
    }
    const float f = PartWeight(ml.x, ml.y, top);
    sum = fmaf(ml.y, f, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(v[e], f, o[e]);
  }
  const int i = int(QuickDiv(uint32_t(rr), a.div_share)), h = kvh * a.share + rr - i * a.share;
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

struct Plan { int nt, row_tiles; int64_t tiles; };

Plan PlanSteps(const AttnArgs& a) {
  Plan p;
  const int rows = a.max_new * a.share;
  p.nt = rows > 8 && a.c.head_dim < 256 ? 2 : 1;   // 16 columns of 256 channels would not fit a thread's registers
  p.row_tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
  int64_t span = std::min<int64_t>(a.max_kept, int64_t(a.table_cols) * a.c.page_size);
  if (a.window > 0) span = std::min<int64_t>(span, int64_t(a.window) + a.max_new + kTile);
  p.tiles = (span + kTile - 1) / kTile * a.num_seqs * a.c.kv_heads * p.row_tiles;   // at most
  return p;
}

size_t PartBytes(const AttnArgs& a, const Plan& p) { return size_t(kMaxBlocks) * 2 * 8 * p.nt * (size_t(a.c.head_dim) * sizeof(float) + sizeof(float2)); }

template <int DIM, int GROUP, int NT, bool PAGE16> int LaunchKernel(const StepArgs& s, const Plan& p, cudaStream_t st, int* blocks) {
  constexpr size_t kStage = kTogether<DIM, NT> * (2 * kTile * (DIM / 2) + 2 * kTile * (DIM / GROUP) * 4);
  constexpr size_t kRing = kWarps * kStagesOf<DIM, NT> * kStage, kJoin = size_t(kWarps) * 8 * NT * (DIM * 4 + 8);
  constexpr size_t kSmem = kRing > kJoin ? kRing : kJoin;
  auto kernel = StepsKernel<DIM, GROUP, NT, PAGE16>;
  static std::atomic<int> resident{0};   // blocks per SM; the same for every device of this kind
  int per_sm = resident.load(std::memory_order_relaxed);
  if (kSmem > 48 * 1024) ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmem)));
  if (per_sm == 0) {
    ITEXB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, kSmem));
    resident.store(per_sm, std::memory_order_relaxed);
  }
  *blocks = int(std::min<int64_t>(std::min(kMaxBlocks, per_sm * SmCount()), std::max<int64_t>(1, p.tiles / kLeastTiles)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(*blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ITEXB_CUDA(cudaLaunchKernelEx(&cfg, kernel, s));
  return CheckLaunch("StepsKernel");
}
template <int DIM, int NT, int WARPS> int LaunchJoin(const StepArgs& s, cudaStream_t st) {
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
  ITEXB_CUDA(cudaLaunchKernelEx(&cfg, JoinKernel<DIM, NT, WARPS>, s));
  return CheckLaunch("JoinKernel");
}
template <int DIM, int GROUP, int NT> int LaunchPage(const StepArgs& s, const Plan& p, cudaStream_t st) {
  int blocks = 0;
  if (s.a.c.page_size % kTile == 0) ITEXB_RETURN_IF_ERROR((LaunchKernel<DIM, GROUP, NT, true>(s, p, st, &blocks)));
  else ITEXB_RETURN_IF_ERROR((LaunchKernel<DIM, GROUP, NT, false>(s, p, st, &blocks)));
  // more than 8 results per unit: a block of 8 warps adds them up, else a warp
  if (blocks > 8 * int64_t(s.a.num_seqs) * s.units) return LaunchJoin<DIM, NT, 8>(s, st);
  return LaunchJoin<DIM, NT, 1>(s, st);
}
template <int DIM, int GROUP> int LaunchGroup(const StepArgs& s, const Plan& p, cudaStream_t st) {
  if constexpr (GROUP > DIM) {
    return SetError(ITEXB_INTERNAL, "kv4_attention: group above head_dim");
  } else if constexpr (DIM < 256) {
    return p.nt == 1 ? LaunchPage<DIM, GROUP, 1>(s, p, st) : LaunchPage<DIM, GROUP, 2>(s, p, st);
  } else {
    return LaunchPage<DIM, GROUP, 1>(s, p, st);
  }
}
template <int DIM> int LaunchDim(const StepArgs& s, const Plan& p, cudaStream_t st) {
  if (s.a.c.group == 32) return LaunchGroup<DIM, 32>(s, p, st);
  if (s.a.c.group == 64) return LaunchGroup<DIM, 64>(s, p, st);
  return LaunchGroup<DIM, 128>(s, p, st);
}

}  // namespace

size_t StepsWorkspace(const AttnArgs& a) { return PartBytes(a, PlanSteps(a)) + (size_t(a.num_seqs) + 2) * sizeof(int64_t); }

int LaunchSteps(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st) {
  const Plan p = PlanSteps(a);
  StepArgs s{};
  s.a = a;
  s.row_tiles = p.row_tiles;
  s.units = a.c.kv_heads * p.row_tiles;
  s.bf16 = dtype == ITEXB_DT_BFLOAT16;
  s.part_o = static_cast<float*>(workspace);
  s.part_ml = reinterpret_cast<float2*>(s.part_o + size_t(kMaxBlocks) * 2 * 8 * p.nt * a.c.head_dim);
  s.list = reinterpret_cast<int64_t*>(static_cast<uint8_t*>(workspace) + PartBytes(a, p));
  if (a.c.head_dim == 64) return LaunchDim<64>(s, p, st);
  if (a.c.head_dim == 128) return LaunchDim<128>(s, p, st);
  return LaunchDim<256>(s, p, st);
}

}  // namespace itexb
