"""64-bit references of the decoder operators and the error bounds their tests use.

Bounds are worst cases added up from the roundings a kernel makes.  U[t] is half a step of a type relative to the value
(its unit roundoff)."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}     # half a subnormal step


def pairs_of(x, rot, interleaved):
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def put_pairs(x, a, b, rot, interleaved):
    y = x.clone()
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = a, b
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a, b
    return y


def rotate(x, positions, inv_freq, interleaved=False, mscale=1.0, sign=1.0):
    """x: float64 [tokens, heads, dim] -> (rotated, |a| + |b| of each element's pair times mscale)."""
    rot = 2 * inv_freq.numel()
    ang = sign * torch.outer(positions.double(), inv_freq)[:, None, :]
    c, s = ang.cos() * mscale, ang.sin() * mscale
    a, b = pairs_of(x, rot, interleaved)
    size = mscale * (a.abs() + b.abs())
    return (put_pairs(x, a * c - b * s, b * c + a * s, rot, interleaved), put_pairs(x.abs(), size, size, rot, interleaved))


# An fp32 rotation: the angle's fraction of a turn rounded to fp32 (2^-25 turns, 2^-22.3 rad), cos and sin off by up to 2 ulp,
# the product with mscale and three roundings: below 2^-21 of |a| + |b|.
ROT = 2.0 ** -21


def normed(x, w, eps):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w


def quantize(x, group):
    """The definition in 64 bits: values, lo, step (both as halves) of rows x [..., dim]."""
    g = x.double().unflatten(-1, (-1, group))
    lo = g.amin(-1).half()
    step = ((g.amax(-1) - lo.double()) / 15.0).clamp_min(0.0).half()
    return g, lo, step


def dequantize(codes, params):
    """fp32 values of cache rows: exact products (11 + 4 bits), one rounding of the sum."""
    v = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.float()
    return (v.unflatten(-1, (p.shape[-2], -1)) * p[..., 1:] + p[..., :1]).flatten(-2)


def cache_rows(cache, table_row, kept, head):
    """-> k, v and what the rounding of a weight may multiply: |v|, or v's distance from the middle of its group's range, lo + 8
    step, where the middle is added unrounded.  There the fp32 sums are of products with 128 + code and with 136, up to 143
    steps, taken from each other: two sums over the tokens of a warp (a quarter of them, 16 at a time, and the joins), each
    addition off by up to 2^-23 of the sum, in units of the weights' 2^-8: 143 * 2 * 2^-15 steps times their number.
    float64 [kept, dim] of one sequence and head."""
    j = torch.arange(kept, device=table_row.device)
    page, off = table_row.long()[j // cache.page_size], j % cache.page_size
    k, v = (dequantize(c[page, head, off], p[page, head, off]).double() for c, p in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)))
    pars = cache.v_params[page, head, off].double()
    lo, step = (pars[..., i].repeat_interleave(cache.group, -1) for i in (0, 1))
    return k, v, torch.maximum(v.abs(), (v - lo - 8.0 * step).abs()) + step * (143.0 * 2.0 ** -14 * (kept / 64 + 8))


def attention(cache, q, table, kept, starts, causal=True, window=0, scale=None, hidden=None):
    """-> (out, bound's parts A = sum p |what weights multiply| and D = scale * sum |q| |k| at its largest), float64; rows behind the last sequence NaN.
    hidden: bool [seqs, rows] of cache rows that do not count."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    share = q.shape[1] // cache.kv_heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    size, dots = torch.zeros_like(out), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device=q.device)
    for b, n_kept in enumerate(kept):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        i, j = torch.arange(n, device=q.device)[:, None], torch.arange(n_kept, device=q.device)[None, :]
        place = n_kept - n + i
        seen = (j <= place) if causal else torch.ones((n, n_kept), dtype=torch.bool, device=q.device)
        if window:
            seen = seen & (j > place - window)
        if hidden is not None:
            seen = seen & ~hidden[b, :n_kept]
        for h in range(cache.kv_heads):
            if n_kept == 0:
                out[lo:hi] = 0.0
                break
            clean = seen.any(0)[:, None]
            k, v, far = (torch.where(clean, x, 0.0) for x in cache_rows(cache, table[b].clamp_min(0), n_kept, h))
            for g in range(h * share, (h + 1) * share):
                x = q[lo:hi, g].double()
                a = (x @ k.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(a, -1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                out[lo:hi, g], size[lo:hi, g] = p @ v, p @ far
                dots[lo:hi, g, 0] = (x.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0).amax(-1)
    return out, size, dots


def check_attention(got, want, size, dots, rows, context):
    """Elementwise: the weights' rounding (bf16 at worst, 2^-8 of what a weight multiplies, see cache_rows), the values' (fp16, 2^-11), the output's, and twice a score's error
    (keys rounded to fp16, 2^-11, fp32 sums over the dimension, 2^-16) in the exponent, since it enters weights and their sum.
    In the 2-norm: the roundings are independent, each uniform within half a step (a factor 3^-1/2), so weights, output and
    scores add up to less than 6e-3 of the output for bf16 (2^-8 / 3^1/2 = 0.0023 each), where the scores stay moderate."""
    g, w, s, d = got[:rows].double(), want[:rows], size[:rows], dots[:rows]
    tol = U[got.dtype] * w.abs() + TINY[got.dtype] + s * (2.0 ** -8 + 2.0 ** -11 + 2.0 * d * (2.0 ** -11 + 2.0 ** -16))
    off = (g - w).abs()
    assert torch.isfinite(g).all(), context
    assert (off <= tol).all(), (context, float((off - tol).max()), float(off.max()))
    norm = float(w.norm())
    if norm > 0:
        assert float((g - w).norm()) <= 6e-3 * norm, (context, float((g - w).norm()) / norm)
