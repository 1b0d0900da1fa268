// itexb_kv4_attention: argument checks and the choice of kernel.
#include <cmath>

#include "kv4_attention.h"

using namespace itexb;

namespace {

// Rows that share their keys and values, above which the kernel of whole 128-token tiles is taken; the other reads the cache
// once for every 16 rows.  Measured (rows: one kernel, the other), 32 sequences of 4096 tokens, 32 / 8 heads of 128: 16 rows 75,
// 137 us; 24 rows 129, 137; 32 rows 132, 137; 64 rows 244, 138.  One sequence of 10240: 32 rows 31, 40 us; 64 rows 37, 40.
// head_dim 256: 32 rows 38, 53 us; 64 rows 58, 54; head_dim 64: 32 rows 30, 34 us; 64 rows 30, 34.
constexpr int kFewRows = 32;
bool IsPrefill(const AttnArgs& a) { return int64_t(a.max_new) * a.share > kFewRows; }

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
  a->q_aligned = reinterpret_cast<uintptr_t>(p->q) % 16 == 0 && p->q_token_stride % 8 == 0 && p->q_head_stride % 8 == 0;
  a->scale_log2 = p->scale * 1.4426950408889634f;
  ITEXB_REQUIRE(std::isfinite(a->scale_log2), ITEXB_INVALID_ARGUMENT, "%s: scale must be finite, got %g", what, double(p->scale));
  a->div_share = MakeFastDiv(uint32_t(a->share));
  return ITEXB_OK;
}

}  // namespace

extern "C" size_t itexb_kv4_attention_workspace_bytes(const itexb_kv4_attention_params_t* p) {
  AttnArgs a{};
  if (CheckAttention(p, &a) != ITEXB_OK || p->num_seqs == 0 || p->max_new == 0 || p->total_rows == 0) return 0;
  return IsPrefill(a) ? PrefillWorkspace(a) : StepsWorkspace(a);
}

extern "C" int itexb_kv4_attention(const itexb_kv4_attention_params_t* p, itexb_stream_t stream) {
  AttnArgs a{};
  ITEXB_RETURN_IF_ERROR(CheckAttention(p, &a));
  if (p->num_seqs == 0 || p->max_new == 0 || p->total_rows == 0) return ITEXB_OK;
  ITEXB_REQUIRE(p->q && p->out && p->kept && (p->block_table || p->table_cols == 0), ITEXB_INVALID_ARGUMENT, "kv4_attention: NULL tensor");
  const size_t need = IsPrefill(a) ? PrefillWorkspace(a) : StepsWorkspace(a);
  ITEXB_REQUIRE(p->workspace && p->workspace_bytes >= need && reinterpret_cast<uintptr_t>(p->workspace) % 16 == 0, ITEXB_INVALID_ARGUMENT,
                "kv4_attention: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need, p->workspace_bytes);
  if (IsPrefill(a)) return LaunchPrefill(a, p->dtype, p->workspace, AsCuda(stream));
  return LaunchSteps(a, p->dtype, p->workspace, AsCuda(stream));
}
