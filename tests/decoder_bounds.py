"""Attention over the 4-bit cache in 64 bits, with bounds that are as tight as the kernels' roundings are few.

Every term is a worst case, U = half a step of a half, 2^-11, unless said otherwise:
  output    half a step of its type
  weights   a weight is a half.  The few-row kernel (at most 32 query rows of a key/value head) multiplies it with a value's
            distance from the middle of its group's range, lo + 8 step, the middle itself being added in fp32; the many-row
            kernel with the value.
  values    a half, once, in the many-row kernel for bf16 queries and for groups whose products with codes could pass the largest half;
            otherwise exact or off by U^2
  scores    keys as the values; queries are off by 2^-24 of the row's largest magnitude; sums in fp32.  A score's error enters
            a weight and the sum it is divided by.
  sums      fp32: a product of a weight with at most 15 + 8 steps, or with a value, is off by 2^-23 of the running sum at each
            of (tokens / 64 + 16) additions one after another: 16 tokens an addition, four warps, and the joins."""
import math

import torch

import decoder_ref as R

HALF = 2.0 ** -11


def rows_of(cache, table_row, kept, head):
    """-> k, v, middle, step of one sequence's rows and head, float64 [kept, head_dim]."""
    j = torch.arange(kept, device=table_row.device)
    page, off = table_row.long()[j // cache.page_size], j % cache.page_size
    out = []
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        c, p = codes[page, head, off], params[page, head, off].double()
        lo, step = (p[..., i].repeat_interleave(cache.group, -1) for i in (0, 1))
        code = torch.stack([c & 15, c >> 4], -1).flatten(-2).double()
        out.append((lo + step * code, lo + 8.0 * step, step))
    return out[0][0], out[1][0], out[1][1], out[1][2]


def attention(cache, q, table, kept, starts, causal=True, window=0, scale=None):
    """-> dict of float64 tensors like q: out; its sums over tokens of p |v|, p |v - middle|, p step (their largest of any channel where
    only that is needed); dots [rows, heads, 1]: the largest scale * sum |q| |k| of a visible token."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    share = q.shape[1] // cache.kv_heads
    r = {n: torch.zeros(q.shape, dtype=torch.float64, device=q.device) for n in ("out", "v", "off", "step")}
    r["dots"] = torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device=q.device)
    r["wide"] = any(bool(((p[..., 1].abs() >= 2048) | (p[..., 0].abs() >= 32768)).any()) for p in (cache.k_params, cache.v_params))
    r["kept"], r["many"] = max(kept), max(b - a for a, b in zip(starts, starts[1:])) * share > 32
    for b, n_kept in enumerate(kept):
        a, e = starts[b], starts[b + 1]
        n = e - a
        if n == 0 or n_kept == 0:
            continue
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(n_kept, device=q.device)[None, :]
        place = n_kept - n + i
        seen = (j <= place) if causal else torch.ones((n, n_kept), dtype=torch.bool, device=q.device)
        if window:
            seen = seen & (j > place - window)
        for h in range(cache.kv_heads):
            k, v, mid, step = rows_of(cache, table[b].clamp_min(0), n_kept, h)
            for g in range(h * share, (h + 1) * share):
                x = q[a:e, g].double()
                p = torch.softmax((x @ k.T * scale).masked_fill(~seen, -math.inf), -1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                r["out"][a:e, g], r["v"][a:e, g], r["off"][a:e, g], r["step"][a:e, g] = p @ v, p @ v.abs(), p @ (v - mid).abs(), p @ step
                r["dots"][a:e, g, 0] = (x.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(-1)
    return r


def tolerance(r, dtype, score=None):
    """Bound of each output's error; score: of the scores' errors where it is known better than from `dots`."""
    one = r["many"] and (dtype == torch.bfloat16 or r["wide"])        # keys and values as one half each
    if score is None:
        score = r["dots"] * ((HALF if one else 2.0 ** -21) + 2.0 ** -16)
    far = r["v"] if r["many"] else r["off"]
    fp32 = (r["v"] + 23.0 * r["step"]) * (2.0 ** -23 * (r["kept"] / 64 + 16))
    return (R.U[dtype] * r["out"].abs() + R.TINY[dtype] + far * HALF + (r["v"] * HALF if one else r["v"] * 2.0 ** -20) + fp32
            + 2.0 * torch.expm1(score) * torch.maximum(r["v"], r["off"])) * (1.0 + 2.0 ** -6)


def check(got, r, rows=None, score=None, norm=None, context=None):
    """Every output within `tolerance`, and all together within `norm` of their 2-norm."""
    g, want, tol = (x[:rows] for x in (got.double(), r["out"], tolerance(r, got.dtype, score)))
    assert torch.isfinite(g).all(), context
    off = (g - want).abs()
    assert (off <= tol).all(), (context, float((off - tol).max()), float((off / tol.clamp_min(1e-300)).max()))
    if norm is not None:
        assert float((g - want).norm()) <= norm * float(want.norm()), (context, float((g - want).norm() / want.norm()))
