// Attention of many query rows over the 4-bit paged cache: prompts and their chunks.
//
// Bound: the tensor cores' 4 head_dim operations per (row, token) pair, and beside them the exponentials: 16 per clock and SM
// against the 32 pairs per clock that the two products of head_dim 128 allow.
//
// One block of 512 threads owns 256 query rows of one key/value head (new tokens times the query heads that share it; 128
// rows for head_dim 256) and walks the visible tokens in tiles of 128:
//   warp 0       issues tcgen05.mma (f16 operands, fp32 accumulators in tensor memory): S = q K^T and O += P V for the two
//                halves of 128 rows in turn, so that one half's products run under the other half's softmax
//   warp 1       allocates tensor memory: S of each half (128 columns; P overwrites it as halves), O of each half
//   warps 4-11   softmax, a thread per row: weights 2^(s - m + 7) straight from S with the maximum m of earlier tiles; only when
//                a row's weights of a tile add up to more than 2^15 is the maximum looked for, the accumulator rescaled and the
//                tile done again.  Weights go back to tensor memory as the second product's A operand
//   warps 12-15  a thread per token: page lookup, codes and params into registers one tile ahead, values lo + step * code as
//                halves into shared memory in the layout the tensor cores read (128-byte swizzle; keys K-major, values
//                MN-major: both are rows of channels)
// Halves hold a value to 2^-12 of itself; q enters scaled by a power of two per row (see kv4_steps.cu).  The order of
// channels is the codes' in a word, for q, keys and the output alike.
// Rows of the cache that no query may see are zeros here; a value group stored as NaN is zeros too and makes the rows that see
// it NaN at the end.  Every wait is bounded.
#include <algorithm>

#include "kv4_attention.h"

namespace itexb {
namespace {

constexpr int kThreads = 512;
constexpr int kTokens = 128;                 // per tile
constexpr int kRows = 128;                   // per half: lanes of tensor memory
constexpr float kUp = 7.f;                   // weights are 2^(score - maximum + 7),
constexpr float kLimit = 32768.f;            // and their sum over a tile at most 2^15, so that none overflows a half
constexpr float kNone = 3.0e38f;             // -maximum + 7 of no scores
constexpr long long kWaitCycles = 4000000000ll;   // about 2 s

template <int DIM> struct Shape {
  static constexpr int kHalves = DIM == 256 ? 1 : 2;       // of 128 rows
  static constexpr int kStages = DIM == 256 ? 1 : 2;       // tiles of keys, and of values
  static constexpr int kQBytes = kHalves * kRows * DIM * 2, kTileBytes = kTokens * DIM * 2;
  static constexpr int kSmem = kQBytes + 2 * kStages * kTileBytes;
  static constexpr int kOColumn = kHalves * 128;           // of the first half's O; S of half m starts at column 128 m
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
__device__ __forceinline__ void MmaSmem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void MmaTmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add)), "r"(0u)
      : "memory");
}
// Rows of 128 bytes in groups of eight, 1024 bytes apart, 128-byte swizzle.  `lead`: bytes between blocks of 64 channels where
// channels are the operand's outer dimension (values).
__device__ __forceinline__ uint64_t Desc(uint32_t at, uint32_t lead) {
  return uint64_t((at & 0x3ffffu) >> 4) | (uint64_t(lead >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ void TmemLoad32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
        "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
        "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                 "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                 "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]),
                 "+r"(v[31])::"memory");
}
__device__ __forceinline__ void TmemStore32(uint32_t at, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
      "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void TmemStoreDone() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct Shared {   // behind the operand tiles
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done[2], drained;
  uint32_t tmem;
  volatile int quit;
  int nan_values;          // some value group is stored as NaN
  uint32_t there[4][4];    // of the last four tiles: tokens that exist, 32 per word
};

// Byte offset of 16-byte piece `piece` of row `row` in a tile of rows of DIM halves: blocks of 64 channels, 128-byte swizzle.
__device__ __forceinline__ uint32_t PieceAt(int row, int piece) {
  return uint32_t(piece >> 3) * (128 * 128) + uint32_t(row) * 128 + uint32_t(((piece & 7) ^ (row & 7)) * 16);
}
__device__ __forceinline__ uint32_t AndOr(uint32_t x, uint32_t mask, uint32_t constant) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(constant));
  return r;
}
// lo + step * code for the codes at two nibbles of a word: the code's bits in the mantissa of 1024 (bits 0-3) or 64 (bits
// 4-7), the constant subtracted (exact), one rounding in the multiply-add.
__device__ __forceinline__ uint32_t Value2(uint32_t bits, uint32_t minus, uint32_t step2, uint32_t lo2) {
  uint32_t c, r;
  asm("add.f16x2 %0, %1, %2;" : "=r"(c) : "r"(bits), "r"(minus));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(c), "r"(step2), "r"(lo2));
  return r;
}
__device__ __forceinline__ uint4 Values8(uint32_t w, uint32_t step2, uint32_t lo2) {
  const uint32_t u = w >> 8;
  return make_uint4(Value2(AndOr(w, 0x000F000Fu, 0x64006400u), 0xE400E400u, step2, lo2), Value2(AndOr(w, 0x00F000F0u, 0x54005400u), 0xD400D400u, step2, lo2),
                    Value2(AndOr(u, 0x000F000Fu, 0x64006400u), 0xE400E400u, step2, lo2), Value2(AndOr(u, 0x00F000F0u, 0x54005400u), 0xD400D400u, step2, lo2));
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
  __device__ __forceinline__ void Store(uint8_t* tile, int row) const {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) {
      const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int piece = i * 4 + k;
        const uint32_t p = params[piece * 8 / GROUP];
        *reinterpret_cast<uint4*>(tile + PieceAt(row, piece)) = Values8(w[k], __byte_perm(p, p, 0x3232), __byte_perm(p, p, 0x1010));
      }
    }
  }
};
__device__ __forceinline__ bool NotFinite(uint32_t half2) { return (half2 & 0x7c00u) == 0x7c00u || (half2 & 0x7c000000u) == 0x7c000000u; }

struct PrefillArgs {
  AttnArgs a;
  int bf16;
};

template <int DIM, int GROUP>
__global__ void __launch_bounds__(kThreads, 1) PrefillKernel(const __grid_constant__ PrefillArgs s) {
  using H = Shape<DIM>;
  constexpr int M = H::kHalves, ST = H::kStages, NG = DIM / GROUP;
  const AttnArgs& a = s.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const s_q = smem;
  uint8_t* const s_k = smem + H::kQBytes;
  uint8_t* const s_v = s_k + ST * H::kTileBytes;
  Shared& sh = *reinterpret_cast<Shared*>(s_v + ST * H::kTileBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, b = blockIdx.z;
  if ((SmemAt(smem) & 1023u) != 0) {   // the swizzle needs it; refuse rather than compute garbage
    if (threadIdx.x == 0 && a.status_word != nullptr) atomicCAS(a.status_word, 0, ITEXB_STATUS_WAIT_EXPIRED);
    return;
  }
  const Seq q = SeqOf(a, b, threadIdx.x == 0 && blockIdx.x == 0 && kvh == 0);
  const int rows = q.nnew * a.share;
  const int blocks = (rows + M * kRows - 1) / (M * kRows);
  // the last rows see the most tokens: their blocks come first
  const int row0 = (blocks - 1 - int(blockIdx.x)) * (M * kRows);
  if (int(blockIdx.x) >= blocks) return;
  const int row1 = min(rows, row0 + M * kRows);
  const int halves = row1 - row0 > kRows ? 2 : 1;
  const int i_first = int(QuickDiv(uint32_t(row0), a.div_share)), i_last = int(QuickDiv(uint32_t(row1 - 1), a.div_share));
  const int some_begin = RowBegin(a, q, i_first), end = RowEnd(a, q, i_last), begin = some_begin & ~15;
  const int tiles = end > begin ? (end - begin + kTokens - 1) / kTokens : 0;

  if (threadIdx.x == 0) {
    BarInit(&sh.q_full, uint32_t(halves * kRows));
    for (int i = 0; i < 2; ++i) {
      BarInit(&sh.k_full[i], 128);
      BarInit(&sh.k_empty[i], 1);
      BarInit(&sh.v_full[i], 128);
      BarInit(&sh.v_empty[i], 1);
      BarInit(&sh.s_full[i], 2);      // the products' completion, and the issuer itself (for what it has seen others write)
      BarInit(&sh.p_full[i], kRows);
      BarInit(&sh.o_done[i], 2);
    }
    BarInit(&sh.drained, 1);
    sh.quit = 0;
    sh.nan_values = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SmemAt(&sh.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  FenceBefore();
  __syncthreads();
  FenceAfter();
  const uint32_t tmem = sh.tmem;
  volatile int* const quit = &sh.quit;

  if (warp == 0) {
    // ---------------- products ----------------
    if (lane == 0 && tiles > 0) {
      constexpr uint32_t kIdescS = (1u << 4) | (uint32_t(kTokens >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      constexpr uint32_t kIdescO = (1u << 4) | (1u << 16) | (uint32_t(DIM >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
      auto scores = [&](int m, int j) {
        const uint32_t qa = SmemAt(s_q) + m * (kRows * DIM * 2), ka = SmemAt(s_k) + (j % ST) * H::kTileBytes;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          const uint32_t off = (k / 4) * (128 * 128) + (k % 4) * 32;
          MmaSmem(tmem + m * 128, Desc(qa + off, 16), Desc(ka + off, 16), kIdescS, k > 0);
        }
        Commit(&sh.s_full[m]);
        BarArrive(&sh.s_full[m]);
        if (m == halves - 1) Commit(&sh.k_empty[j % ST]);
      };
      bool ok = BarWait(&sh.q_full, 0, quit, a.status_word) && BarWait(&sh.k_full[0], 0, quit, a.status_word);
      FenceAfter();
      for (int m = 0; m < halves && ok; ++m) scores(m, 0);
      for (int j = 0; j < tiles && ok; ++j) {
        for (int m = 0; m < halves && ok; ++m) {
          ok = BarWait(&sh.p_full[m], j & 1, quit, a.status_word) && (m > 0 || BarWait(&sh.v_full[j % ST], (j / ST) & 1, quit, a.status_word));
          if (!ok) break;
          FenceAfter();
          const uint32_t va = SmemAt(s_v) + (j % ST) * H::kTileBytes;
#pragma unroll
          for (int k = 0; k < kTokens / 16; ++k)
            MmaTmem(tmem + H::kOColumn + m * DIM, tmem + m * 128 + k * 8, Desc(va + k * 2048, 128 * 128), kIdescO, j > 0 || k > 0);
          Commit(&sh.o_done[m]);
          BarArrive(&sh.o_done[m]);
          if (m == halves - 1) Commit(&sh.v_empty[j % ST]);
          if (j + 1 < tiles) {
            ok = m > 0 || BarWait(&sh.k_full[(j + 1) % ST], ((j + 1) / ST) & 1, quit, a.status_word);
            // P is read from where the next S goes
            ok = ok && BarWait(&sh.o_done[m], j & 1, quit, a.status_word);
            if (!ok) break;
            FenceAfter();
            scores(m, j + 1);
          }
        }
      }
      // nothing in flight when tensor memory is given back
      Commit(&sh.drained);
      BarWait(&sh.drained, 0, nullptr, a.status_word);
    }
  } else if (warp >= 4 && warp < 4 + 4 * halves) {
    // ---------------- softmax ----------------
    const int m = (warp - 4) >> 2, in_half = (warp & 3) * 32 + lane;
    const int rr = row0 + m * kRows + in_half;
    const bool on = rr < row1;
    const int i = int(QuickDiv(uint32_t(on ? rr : row0), a.div_share)), h = (on ? rr : row0) - i * a.share;
    const int lo = on ? RowBegin(a, q, i) : 0, hi = on ? RowEnd(a, q, i) : 0;
    // tokens that all rows of this warp see
    const int w_first = int(QuickDiv(uint32_t(min(row1 - 1, row0 + m * kRows + (warp & 3) * 32)), a.div_share));
    const int w_last = int(QuickDiv(uint32_t(min(row1, row0 + m * kRows + (warp & 3) * 32 + 32) - 1), a.div_share));
    const int all_begin = RowBegin(a, q, max(w_first, w_last)), all_end = RowEnd(a, q, min(w_first, w_last));
    float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
    {
      // ---- the row of q: half, scaled, in the codes' order
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + (q.row0 + i) * a.qt + int64_t(kvh * a.share + h) * a.qh;
      union Piece { uint4 v; uint32_t u[4]; uint16_t e[8]; };
      auto piece = [&](int p) {
        Piece x;
        if (!on) x.v = make_uint4(0, 0, 0, 0);
        else if (a.q_aligned) x.v = __ldg(reinterpret_cast<const uint4*>(src) + p);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) x.e[e] = src[p * 8 + e];
        return x;
      };
      float down = a.scale_log2 < 0.f ? -1.f : (a.scale_log2 == 0.f ? 0.f : 1.f);
      if (s.bf16) {
        float most = 0.f;
#pragma unroll 4
        for (int p = 0; p < DIM / 8; ++p) {
          const Piece x = piece(p);
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(__uint_as_float(uint32_t(x.e[e]) << 16)));
        }
        const int e = min(max(int(__float_as_uint(most) >> 23), 1), 253);
        if (most > 0.f && most < INFINITY) {
          down *= __uint_as_float(uint32_t(254 - e) << 23);
          scale = fmaxf(scale * __uint_as_float(uint32_t(e) << 23), 1e-37f);
        }
      }
      uint8_t* const to = s_q + m * (kRows * DIM * 2);
#pragma unroll 4
      for (int p = 0; p < DIM / 8; ++p) {
        Piece x = piece(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float raw = s.bf16 ? __uint_as_float(uint32_t(x.e[e]) << 16) : __half2float(__ushort_as_half(x.e[e]));
          x.e[e] = __half_as_ushort(__float2half_rn(raw * down));
        }
        *reinterpret_cast<uint4*>(to + PieceAt(in_half, p)) =
            make_uint4(__byte_perm(x.u[0], x.u[2], 0x5410), __byte_perm(x.u[0], x.u[2], 0x7632), __byte_perm(x.u[1], x.u[3], 0x5410), __byte_perm(x.u[1], x.u[3], 0x7632));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      BarArrive(&sh.q_full);
    }
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + m * 128, o_at = tmem + lanes + H::kOColumn + m * DIM;
    float shift = kNone, total = 0.f;       // weights are 2^(score * scale + shift)
    bool ok = true;
    for (int j = 0; j < tiles && ok; ++j) {
      ok = BarWait(&sh.s_full[m], j & 1, quit, a.status_word);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      FenceAfter();
      const int j0 = begin + j * kTokens;
      const uint32_t* there = sh.there[j & 3];
      const bool partial = j0 < all_begin || j0 + kTokens > all_end || (there[0] & there[1] & there[2] & there[3]) != 0xffffffffu;
      uint32_t p[kTokens / 2];
      float sum = 0.f;
      auto weights = [&]() {
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          TmemLoad32(s_at + c * 32, v);
          if (partial) {
            const uint32_t word = there[c];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const int t = j0 + c * 32 + e;
              if (t < lo || t >= hi || ((word >> e) & 1u) == 0u) v[e] = 0xff800000u;
            }
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float x = Exp2(fmaf(__uint_as_float(v[e]), scale, shift)), y = Exp2(fmaf(__uint_as_float(v[e + 1]), scale, shift));
            part[0] += x;
            part[1] += y;
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p[c * 16 + e / 2]) : "f"(y), "f"(x));
          }
        }
        sum = part[0] + part[1];
      };
      weights();
      if (__any_sync(0xffffffffu, sum > kLimit)) {
        // a new maximum for the rows that passed it
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          TmemLoad32(s_at + c * 32, v);
          const uint32_t word = there[c];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int t = j0 + c * 32 + e;
            if (!partial || (t >= lo && t < hi && ((word >> e) & 1u) != 0u)) top = fmaxf(top, __uint_as_float(v[e]));
          }
        }
        const float to = fminf(shift, kUp - top * scale);
        const float f = Exp2(to - shift);
        shift = to;
        total *= f;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < DIM / 32; ++c) {
            uint32_t v[32];
            TmemLoad32(o_at + c * 32, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
            TmemStore32(o_at + c * 32, v);
          }
        }
        weights();
      }
      total += sum;
      TmemStore32(s_at, p);
      TmemStore32(s_at + 32, p + 32);
      TmemStoreDone();
      FenceBefore();
      BarArrive(&sh.p_full[m]);
    }
    if (tiles > 0 && ok) ok = __all_sync(0xffffffffu, BarWait(&sh.o_done[m], (tiles - 1) & 1, quit, a.status_word));
    if (ok) {
      FenceAfter();
      uint32_t nan_groups = 0;
      if (tiles > 0 && sh.nan_values != 0) {   // rare: find the value groups that are NaN among the tokens this row sees
        for (int t = lo; t < hi; ++t) {
          const int col = int(QuickDiv(uint32_t(t), a.c.div_page)), page = __ldg(a.table + int64_t(b) * a.table_stride + col);
          if (page < 0 || page >= a.c.num_pages) continue;
          const __half2* at = a.c.v_params + int64_t(page) * a.c.pp + int64_t(kvh) * a.c.ph + int64_t(t - col * a.c.page_size) * a.c.pt;
          for (int g = 0; g < NG; ++g) nan_groups |= uint32_t(NotFinite(__ldg(reinterpret_cast<const uint32_t*>(at + g)))) << g;
        }
      }
      __syncwarp();
      const float inv = total == 0.f ? 0.f : 1.f / total;
      const int64_t at = (q.row0 + i) * a.ot + int64_t(kvh * a.share + h) * a.oh;
      const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.ot & 7) == 0 && (a.oh & 7) == 0;
#pragma unroll 1
      for (int c = 0; c < DIM / 32; ++c) {
        uint32_t v[32];
        __syncwarp();
        if (tiles > 0) TmemLoad32(o_at + c * 32, v);
        else
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        const bool is_nan = (nan_groups >> (c * 32 / GROUP)) & 1u;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          union { uint4 x; uint16_t e[8]; } out;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int from = e < 4 ? 2 * e : 2 * (e - 4) + 1;   // back from the codes' order
            const float f = is_nan ? __uint_as_float(0x7fffffffu) : (total == 0.f ? 0.f : __uint_as_float(v[w * 8 + from]) * inv);
            out.e[e] = s.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f)) : __half_as_ushort(__float2half_rn(f));
          }
          if (on) {
            uint16_t* to = static_cast<uint16_t*>(a.out) + at + c * 32 + w * 8;
            if (wide) *reinterpret_cast<uint4*>(to) = out.x;
            else
#pragma unroll
              for (int e = 0; e < 8; ++e) to[e] = out.e[e];
          }
        }
      }
    }
    FenceBefore();
  } else if (warp >= 12) {
    // ---------------- codes to operands ----------------
    const int t = threadIdx.x - 12 * 32, w = warp - 12;
    const int32_t* table = a.table + int64_t(b) * a.table_stride;
    const uint8_t* kc = a.c.k_codes + int64_t(kvh) * a.c.ch;
    const uint8_t* vc = a.c.v_codes + int64_t(kvh) * a.c.ch;
    const __half2* kp = a.c.k_params + int64_t(kvh) * a.c.ph;
    const __half2* vp = a.c.v_params + int64_t(kvh) * a.c.ph;
    Row<DIM, GROUP> k, v;
    // the page of this thread's token of a tile, -1 where there is none
    auto page_of = [&](int j) {
      const int tok = begin + j * kTokens + t;
      if (j >= tiles || tok < some_begin || tok >= end) return -1;
      const int page = __ldg(table + QuickDiv(uint32_t(tok), a.c.div_page));
      if (page >= 0 && page < a.c.num_pages) return page;
      ReportIndex(a.status_word);
      return -1;
    };
    auto offset_of = [&](int j) {
      const int tok = begin + j * kTokens + t;
      return tok - int(QuickDiv(uint32_t(tok), a.c.div_page)) * a.c.page_size;
    };
    auto load = [&](Row<DIM, GROUP>& r, const uint8_t* codes, const __half2* params, int page, int j) {
      if (page < 0) { r.Clear(); return; }
      const int64_t off = offset_of(j);
      r.Load(codes + int64_t(page) * a.c.cp + off * a.c.ct, params + int64_t(page) * a.c.pp + off * a.c.pt);
    };
    int page = page_of(0), next = page_of(1);
    load(k, kc, kp, page, 0);
    load(v, vc, vp, page, 0);
    bool ok = true;
    for (int j = 0; j < tiles && ok; ++j) {
      const int after = page_of(j + 2);
      if (j >= ST) ok = BarWait(&sh.k_empty[j % ST], ((j / ST) - 1) & 1, quit, a.status_word);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      k.Store(s_k + (j % ST) * H::kTileBytes, t);
      const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
      if (lane == 0) sh.there[j & 3][w] = there;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      BarArrive(&sh.k_full[j % ST]);
      load(k, kc, kp, next, j + 1);
      if (j >= ST) ok = BarWait(&sh.v_empty[j % ST], ((j / ST) - 1) & 1, quit, a.status_word);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      bool bad = false;
#pragma unroll
      for (int g = 0; g < NG; ++g)
        if (NotFinite(v.params[g])) { v.params[g] = 0; bad = true; }
      if (bad) sh.nan_values = 1;
      v.Store(s_v + (j % ST) * H::kTileBytes, t);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      BarArrive(&sh.v_full[j % ST]);
      load(v, vc, vp, next, j + 1);
      page = next;
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

template <int DIM, int GROUP> int LaunchGroup(const PrefillArgs& s, cudaStream_t st) {
  using H = Shape<DIM>;
  constexpr int kSmem = H::kSmem + int(sizeof(Shared));
  auto kernel = PrefillKernel<DIM, GROUP>;
  ITEXB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int64_t rows = int64_t(s.a.max_new) * s.a.share;
  const dim3 grid(unsigned((rows + H::kHalves * kRows - 1) / (H::kHalves * kRows)), s.a.c.kv_heads, s.a.num_seqs);
  kernel<<<grid, kThreads, kSmem, st>>>(s);
  return CheckLaunch("PrefillKernel");
}
template <int DIM> int LaunchDim(const PrefillArgs& s, cudaStream_t st) {
  if (s.a.c.group == 32) return LaunchGroup<DIM, 32>(s, st);
  if (s.a.c.group == 64) return LaunchGroup<DIM, 64>(s, st);
  if constexpr (DIM >= 128) return LaunchGroup<DIM, 128>(s, st);
  return SetError(ITEXB_INTERNAL, "kv4_attention: group above head_dim");
}

}  // namespace

int LaunchPrefill(const AttnArgs& a, int dtype, cudaStream_t st) {
  PrefillArgs s{a, dtype == ITEXB_DT_BFLOAT16};
  if (a.c.head_dim == 64) return LaunchDim<64>(s, st);
  if (a.c.head_dim == 128) return LaunchDim<128>(s, st);
  return LaunchDim<256>(s, st);
}

}  // namespace itexb
