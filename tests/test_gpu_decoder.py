"""The decoder operators on the GPU against 64-bit references: rotary positions, per-head norms with the rotation and their
gradient, the 4-bit paged cache, attention over it, and a run of them as a decoder layer uses them."""
import importlib
import math

import pytest
import torch

import decoder_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K(itex):
    return importlib.import_module("itex_b200.kernels")


@pytest.fixture(scope="module")
def kv4(itex):
    return importlib.import_module("itex_b200.kv4")


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def within(got, want, tol):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= tol).all(), (float((off - tol).max()), float(off.max()))


def out_tol(want, dtype):
    return R.U[dtype] * want.abs() * (1 + 2.0 ** -7) + R.TINY[dtype]


# ------------------------------------------------------------------------------------------------------------- rope

SHAPES = [  # tokens, q heads, kv heads, dim, rotated
    (1, 1, 1, 64, 64), (3, 32, 8, 128, 128), (37, 5, 1, 80, 80), (70, 6, 2, 96, 48), (9, 2, 2, 256, 128), (130, 3, 1, 512, 512), (5, 3, 2, 10, 6),
    (4, 2, 1, 64, 0), (300, 1, 1, 128, 32), (8, 1, 2, 6, 2), (11, 3, 3, 512, 12)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rope(K, shape, interleaved, dtype):
    t, hq, hk, dim, rot = shape
    q, k = randn(1, t, hq, dim, dtype=dtype), randn(2, t, hk, dim, dtype=dtype)
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
    pos = (torch.arange(t, device="cuda") * 7919 + 1000003) % 1500000
    for inverse, mscale, idx in ((False, 1.0, torch.int64), (True, 1.25, torch.int32)):
        got = K.rope(q, pos.to(idx), freq, k=k, interleaved=interleaved, inverse=inverse, mscale=mscale)
        for x, y in zip((q, k), got):
            want, size = R.rotate(x.double(), pos, freq, interleaved, mscale, -1.0 if inverse else 1.0)
            within(y, want, size * R.ROT + out_tol(want, dtype))
            if rot < dim:
                assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("offset, pad", [(0, 0), (1, 0), (4, 4), (3, 5)])
def test_rope_strided_views_and_in_place(K, offset, pad):
    """Columns of a projection's output at any offset; in place; only the rotated columns change; k left out."""
    t, hq, hk, dim = 21, 4, 2, 64
    width = (hq + 2 * hk) * dim + pad
    buf = randn(3, t * width + 8, dtype=torch.bfloat16)
    qkv = buf[offset:offset + t * width].view(t, width)
    q, k = qkv[:, :hq * dim].unflatten(1, (hq, dim)), qkv[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim))
    before = buf.clone()
    freq, pos = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32), torch.arange(t, device="cuda") - 10
    want = [R.rotate(x.double(), pos, freq) for x in (q, k)]
    alone = K.rope(q, pos, freq)
    assert alone.is_contiguous()
    oq, ok = K.rope(q, pos, freq, k=k, out_q=q, out_k=k)
    assert oq.data_ptr() == q.data_ptr() and torch.equal(alone, q)
    for x, (w, size) in zip((q, k), want):
        within(x, w, size * R.ROT + out_tol(w, torch.bfloat16))
    rest = qkv[:, (hq + hk) * dim:]
    assert torch.equal(rest, before[offset:offset + t * width].view(t, width)[:, (hq + hk) * dim:])
    assert torch.equal(buf[:offset], before[:offset]) and torch.equal(buf[offset + t * width:], before[offset + t * width:])


def test_rope_is_its_own_inverse_and_its_gradient(K):
    t, h, dim = 12, 3, 64
    freq, pos = 100.0 ** (-torch.arange(20, dtype=torch.float64, device="cuda") / 20), torch.arange(t, device="cuda") * 31
    for interleaved in (False, True):
        x, g = randn(4, t, h, dim), randn(5, t, h, dim)
        back = K.rope(K.rope(x, pos, freq, interleaved=interleaved), pos, freq, interleaved=interleaved, inverse=True)
        size = R.rotate(x.double(), pos, freq, interleaved)[1]
        within(back, x.double(), 4 * R.ROT * size + 2 * R.U[torch.float32] * x.abs())
        # <g, R x> = <R^T g, x>: each side is off by ROT of the pairs' sizes
        m = 1.5
        left = (g.double() * K.rope(x, pos, freq, interleaved=interleaved, mscale=m).double()).sum()
        right = (x.double() * K.rope(g, pos, freq, interleaved=interleaved, mscale=m, inverse=True).double()).sum()
        bound = 3 * R.ROT * m * ((g.abs().double() * size).sum() + (x.abs().double() * R.rotate(g.double(), pos, freq, interleaved)[1]).sum())
        assert abs(float(left - right)) <= float(bound)


def test_rope_of_nothing(K):
    freq = torch.ones(4, dtype=torch.float64, device="cuda")
    q = torch.empty((0, 2, 8), device="cuda")
    assert K.rope(q, torch.empty(0, dtype=torch.int64, device="cuda"), freq).shape == (0, 2, 8)


# -------------------------------------------------------------------------------------------------------- norm + rope

@pytest.mark.parametrize("dtype, wtype", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_qk_norm_rope(K, shape, interleaved, dtype, wtype):
    t, hq, hk, dim, rot = shape
    q, k = randn(1, t, hq, dim, dtype=dtype) * 3, randn(2, t, hk, dim, dtype=dtype)
    k[0, 0] = 0                                               # a row of zeros: epsilon alone keeps it finite
    wq, wk = ((1 + 0.2 * randn(s, dim)).to(wtype) for s in (3, 4))
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
    pos = torch.arange(t, device="cuda") * 77
    got = K.qk_norm_rope(q, k, wq, wk, pos, freq, eps=1e-5, interleaved=interleaved, mscale=0.5)
    for x, w, y in zip((q, k), (wq, wk), got):
        n = R.normed(x.double(), w.double(), 1e-5)
        want, size = R.rotate(n, pos, freq, interleaved, 0.5)
        # the sum of squares in fp32: dim roundings, halved by the root; rsqrt 2 ulp, the two products
        within(y, want, size * (R.ROT + (dim / 2 + 8) * 2.0 ** -24) + out_tol(want, dtype))


@pytest.mark.parametrize("dtype, wtype", [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_qk_norm_rope_backward(K, shape, interleaved, dtype, wtype):
    t, hq, hk, dim, rot = shape
    eps, m = 1e-5, 0.75
    x = [randn(s, t, h, dim, dtype=dtype) for s, h in ((1, hq), (2, hk))]
    g = [randn(s, t, h, dim, dtype=dtype) for s, h in ((5, hq), (6, hk))]
    w = [(1 + 0.2 * randn(s, dim)).to(wtype) for s in (3, 4)]
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
    pos = torch.arange(t, device="cuda") * 77
    got = K.qk_norm_rope_backward(*g, *x, *w, pos, freq, eps=eps, interleaved=interleaved, mscale=m)
    again = K.qk_norm_rope_backward(*g, *x, *w, pos, freq, eps=eps, interleaved=interleaved, mscale=m)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for i in range(2):
        xd, gd, wd = x[i].double(), g[i].double(), w[i].double()
        xd.requires_grad_(), wd.requires_grad_()
        y = R.rotate(R.normed(xd, wd, eps), pos, freq, interleaved, m)[0]
        dx, dw = torch.autograd.grad(y, (xd, wd), gd)
        with torch.no_grad():
            r = (xd.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
            hat, size = (xd * r).abs(), R.rotate(gd, pos, freq, interleaved, m)[1]
            u = size * wd.abs()
            # t to ROT; r and the mean over dim elements in fp32
            bound = r * (u + hat * (u * hat).mean(-1, keepdim=True)) * (R.ROT + (2 * dim + 16) * 2.0 ** -24)
            within(got[i], dx, bound + out_tol(dx, dtype))
            # a thread adds at most 2 rows of these shapes, a block at most 128 partial sums; the rest is in 64 bits
            bound = (size * hat).sum((0, 1)) * (R.ROT + (dim / 2 + 160) * 2.0 ** -24)
            within(got[2 + i], dw, bound + out_tol(dw, wtype))


def test_qk_norm_rope_backward_against_differences(K):
    """(f(x + e d) - f(x - e d)) / 2e in 64 bits of the forward definition, against <gradient, d> of the kernel."""
    t, hq, hk, dim = 5, 3, 1, 64
    q, k, gq, gk = randn(1, t, hq, dim), randn(2, t, hk, dim), randn(3, t, hq, dim), randn(4, t, hk, dim)
    wq, wk = 1 + 0.2 * randn(5, dim), 1 + 0.2 * randn(6, dim)
    freq, pos = 1000.0 ** (-torch.arange(16, dtype=torch.float64, device="cuda") / 16), torch.arange(t, device="cuda") * 5
    dq, dk, dwq, dwk = K.qk_norm_rope_backward(gq, gk, q, k, wq, wk, pos, freq, eps=1e-3)
    for x, w, g, dx, dw, s in ((q, wq, gq, dq, dwq, 7), (k, wk, gk, dk, dwk, 8)):
        ex, ew = randn(s, *x.shape).double(), randn(s + 10, dim).double()

        def f(e):
            return (R.rotate(R.normed(x.double() + e * ex, w.double() + e * ew, 1e-3), pos, freq)[0] * g.double()).sum()

        want = float((f(1e-5) - f(-1e-5)) / 2e-5)
        got = float((dx.double() * ex).sum() + (dw.double() * ew).sum())
        size = float((dx.double() * ex).abs().sum() + (dw.double() * ew).abs().sum())
        # differences: e^2 f''' / 6 below 1e-8 of the terms' size, cancellation 2^-52 |f| / e below 1e-9; the kernel: fp32, below 2e-5
        assert abs(got - want) <= 3e-5 * size


@pytest.mark.parametrize("tokens, heads, dim, dtype", [(20011, 1, 256, torch.bfloat16), (10007, 1, 256, torch.float32), (4099, 3, 64, torch.float16)])
def test_long_calls(K, tokens, heads, dim, dtype):
    """Blocks of many tokens, several waves of them, tables formed in several turns: every row is right, and so are the sums."""
    freq = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device="cuda") * 2 / dim)
    pos = torch.randperm(tokens, device="cuda")
    q, k = randn(1, tokens, heads, dim, dtype=dtype), randn(2, tokens, heads, dim, dtype=dtype)
    w = [1 + 0.2 * randn(s, dim) for s in (3, 4)]
    g = [randn(s, tokens, heads, dim, dtype=dtype) for s in (5, 6)]
    turned = K.rope(q, pos, freq, k=k)
    grads = K.qk_norm_rope_backward(*g, q, k, *w, pos, freq, eps=1e-5)
    for i, (x, y) in enumerate(zip((q, k), turned)):
        want, size = R.rotate(x.double(), pos, freq)
        within(y, want, size * R.ROT + out_tol(want, dtype))
        xd, wd = x.double(), w[i].double()
        r = (xd.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
        hat = xd * r
        t, size = R.rotate(g[i].double(), pos, freq, sign=-1.0)
        u, ub = t * wd, size * wd.abs()
        dx = r * (u - hat * (u * hat).mean(-1, keepdim=True))
        bound = r * (ub + hat.abs() * (ub * hat.abs()).mean(-1, keepdim=True)) * (R.ROT + (2 * dim + 16) * 2.0 ** -24)
        within(grads[i], dx, bound + out_tol(dx, dtype))
        # fp32: a thread's rows (at most 68 tokens' of a block, one after another), then at most 64 threads' sums; 64 bits behind that
        dw, bound = (t * hat).sum((0, 1)), (size * hat.abs()).sum((0, 1)) * (R.ROT + (dim / 2 + 68 * heads + 64 + 32) * 2.0 ** -24)
        within(grads[2 + i], dw, bound + out_tol(dw, torch.float32))


def test_gradient_of_no_tokens_is_zero(K):
    e, w = torch.empty((0, 2, 64), device="cuda"), torch.ones(64, device="cuda")
    freq = torch.ones(32, dtype=torch.float64, device="cuda")
    out = K.qk_norm_rope_backward(e, e, e, e, w, w, torch.empty(0, dtype=torch.int64, device="cuda"), freq)
    assert float(out[2].abs().sum()) == 0.0 and float(out[3].abs().sum()) == 0.0


# -------------------------------------------------------------------------------------------------------------- cache

def stored(cache, slots, name):
    page, off = slots // cache.page_size, slots % cache.page_size
    return getattr(cache, name + "_codes")[page, :, off], getattr(cache, name + "_params")[page, :, off]


def plain_quantize(x, group):
    """The row format's formulas with fp32 tensor operations (each separately rounded, as the kernel's are)."""
    g = x.float().unflatten(-1, (-1, group))
    lo = g.amin(-1).half()
    span = g.amax(-1) - lo.float()
    step = (span / torch.full_like(span, 15.0)).clamp_min(0.0).half()       # by a number torch would multiply with its inverse
    inv = torch.where(step > 0, 1.0 / step.float(), 0.0)
    codes = ((g - lo.float()[..., None]) * inv[..., None]).round().clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack([lo, step], -1)


CACHES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dim, group", CACHES)
def test_append_and_gather(K, kv4, dim, group, token_major, dtype):
    heads, page, t = 3, 20, 45
    cache = kv4.Kv4Cache.allocate(7, page, heads, dim, group, token_major=token_major)
    marks = [c.fill_(v) for c, v in ((cache.k_codes, 0x5A), (cache.v_codes, 0x5A), (cache.k_params, 0.25), (cache.v_params, 0.25))]
    k, v = randn(1, t, heads, dim, dtype=dtype) * 2, randn(2, t, heads, dim, dtype=dtype) + 0.5
    v[3] = 1.75                                                # a constant group: step 0
    slots = torch.randperm(7 * page, generator=torch.Generator().manual_seed(3))[:t].cuda()
    skip = slots.clone()
    skip[[0, 17, 44]] = -1
    before = [m.clone() for m in marks]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(k, v, skip, status=status)
    keep = skip >= 0
    for name, x in (("k", k), ("v", v)):
        codes, params = stored(cache, slots, name)
        want_c, want_p = plain_quantize(x, group)
        assert torch.equal(params[keep], want_p[keep]) and torch.equal(codes[keep], want_c[keep])
        # half a step, and what rounding lo and step to halves moves
        lo, step = want_p[..., 0].double(), want_p[..., 1].double()
        back = R.dequantize(codes, params).double().unflatten(-1, (-1, group))
        off = (back - x.double().unflatten(-1, (-1, group))).abs().amax(-1)
        assert (off <= step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -20) + lo.abs() * 2.0 ** -11 + 2.0 ** -24)[keep].all()
    # nothing else was touched
    mine = torch.zeros(7 * page, dtype=torch.bool, device="cuda")
    mine[skip[keep]] = True
    mine = mine.view(7, page)
    for now, was in zip(marks, before):
        assert torch.equal(now.transpose(1, 2)[~mine], was.transpose(1, 2)[~mine])
    for odt in (torch.float32, torch.float16, torch.bfloat16):
        gk, gv = cache.gather(skip.int(), odt, status=status)
        for name, y in (("k", gk), ("v", gv)):
            want = torch.where(keep[:, None, None], R.dequantize(*stored(cache, slots, name)), 0.0).to(odt)
            assert torch.equal(y, want)
    assert int(status) == 0


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim, rot, offset", [(64, 64, 0), (128, 64, 0), (128, 20, 0), (256, 256, 0), (128, 128, 3), (64, 2, 1)])
def test_append_rotates_keys(K, kv4, dim, rot, offset, interleaved):
    heads, page, t, group = 2, 16, 33, 32
    cache = kv4.Kv4Cache.allocate(4, page, heads, dim, group)
    buf = randn(1, t * 3 * heads * dim + 8)
    kv = buf[offset:offset + t * 3 * heads * dim].view(t, 3 * heads * dim)
    k, v = kv[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim)), kv[:, 2 * heads * dim:].unflatten(1, (heads, dim))
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
    pos = torch.arange(t, device="cuda") * 30011
    slots = torch.randperm(4 * page, generator=torch.Generator().manual_seed(3))[:t].cuda()
    cache.append(k, v, slots, positions=pos, inv_freq=freq, interleaved=interleaved, mscale=1.25)
    want, size = R.rotate(k.double(), pos, freq, interleaved, 1.25)
    want_v = plain_quantize(v, group)
    assert all(torch.equal(a, b) for a, b in zip(stored(cache, slots, "v"), want_v))
    g, lo, step = R.quantize(want, group)
    codes, params = stored(cache, slots, "k")
    # the minimum and the range are off by the fp32 rotation (three roundings of products of fp32 cosines: 2^-22 of the pair)
    big = size.unflatten(-1, (-1, group)).amax(-1)
    assert ((params[..., 0].double() - lo.double()).abs() <= 2.0 ** -10 * lo.double().abs() + big * 2.0 ** -21).all()
    assert ((params[..., 1].double() - step.double()).abs() <= 2.0 ** -10 * step.double() + 2.0 ** -9 * lo.double().abs() / 15 + big * 2.0 ** -21).all()
    lo, step = params[..., 0].double(), params[..., 1].double()
    off = (R.dequantize(codes, params).double().unflatten(-1, (-1, group)) - g).abs().amax(-1)
    assert (off <= step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -20) + lo.abs() * 2.0 ** -11 + big * 2.0 ** -21).all()


def test_append_marks_groups_it_cannot_hold(kv4):
    cache = kv4.Kv4Cache.allocate(2, 16, 1, 128, 32)
    k = randn(1, 5, 1, 128)
    k[0, 0, 5], k[1, 0, 40], k[2, 0, 70], k[3, 0, 100] = math.nan, math.inf, -math.inf, -70000.0
    k[4, 0, 0] = 65504.0
    v = torch.zeros_like(k)
    slots = torch.arange(5, device="cuda")
    cache.append(k, v, slots)
    got, zero = cache.gather(slots, torch.float32)
    nan = torch.isnan(got.view(5, 4, 32))
    want = torch.zeros((5, 4), dtype=torch.bool, device="cuda")
    for r, g in ((0, 0), (1, 1), (2, 2), (3, 3)):
        want[r, g] = True
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)
    assert float(zero.abs().max()) == 0.0


def test_bad_slots_are_reported_and_skipped(kv4):
    cache = kv4.Kv4Cache.allocate(2, 16, 2, 64, 32)
    k, v = randn(1, 4, 2, 64), randn(2, 4, 2, 64)
    for bad in (32, -2, 1 << 40):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        before = [t.clone() for t in (cache.k_codes, cache.v_params)]
        slots = torch.tensor([bad, -1, -1, -1], device="cuda")
        cache.append(k, v, slots, status=status)
        assert int(status) == kv4.STATUS_BAD_INDEX
        assert torch.equal(cache.k_codes, before[0]) and torch.equal(cache.v_params, before[1])
        status.zero_()
        gk, gv = cache.gather(slots, status=status)
        assert int(status) == kv4.STATUS_BAD_INDEX and float(gk.abs().max()) == 0.0 and float(gv.abs().max()) == 0.0
        cache.append(k, v, slots)                               # without a status word: skipped in silence


# ---------------------------------------------------------------------------------------------------------- attention

def filled(kv4, pages, page, heads, dim, group, seed=1, token_major=False):
    """A cache full of quantized normal values, a few key channels loud."""
    cache = kv4.Kv4Cache.allocate(pages, page, heads, dim, group, token_major=token_major)
    n = pages * page
    loud = 1 + 2 * (torch.arange(dim, device="cuda") % 23 == 5)
    cache.append(randn(seed, n, heads, dim) * loud, randn(seed + 1, n, heads, dim), torch.arange(n, device="cuda"))
    return cache


def tables(kept, page, pages, seed=5):
    """Pages of all sequences in a random order; -1 behind each sequence's last."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    need = [-(-n // page) for n in kept]
    table = torch.full((len(kept), max(1, max(need)) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table.cuda()


def attend(kv4, cache, new, kept, heads, dtype, seed=9, behind=0, **kw):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = randn(seed, starts[-1] + behind, heads, cache.head_dim, dtype=dtype)
    table = tables(kept, cache.page_size, cache.num_pages)
    out = torch.full_like(q, 7.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = cache.attention(q, table, torch.tensor(kept, dtype=torch.int32, device="cuda"), q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                          max_new=max(new), max_kept=max(kept), out=out, status=status, **kw)
    assert got is out and int(status) == 0
    assert (out[starts[-1]:] == 7.0).all()
    want, size, dots = R.attention(cache, q, table, kept, starts, kw.get("causal", True), kw.get("window", 0), kw.get("scale"))
    R.check_attention(out, want, size, dots, starts[-1], (new, kept, heads, kw))
    return out, want


NEW_KEPT = [
    ([1], [1]), ([1], [0]), ([1, 1, 1], [5, 0, 70]), ([1] * 4, [16, 17, 15, 64]), ([1, 1], [700, 1333]), ([1], [5000]), ([2, 1, 4], [2, 300, 129]),
    ([5, 3], [5, 1025]), ([9, 0, 2], [40, 33, 2]), ([17, 40], [200, 40]), ([130], [130]), ([200, 1, 65], [513, 90, 65]), ([3], [1])]


@pytest.mark.parametrize("dim, group", CACHES)
@pytest.mark.parametrize("new, kept", NEW_KEPT)
def test_attention(kv4, new, kept, dim, group):
    dtype = torch.bfloat16 if (dim // group) % 2 else torch.float16
    cache = filled(kv4, sum(-(-n // 16) for n in kept) + 2, 16, 2, dim, group)
    attend(kv4, cache, new, kept, 8, dtype, behind=3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("share", [1, 2, 3, 5, 7, 8, 12, 16, 33])
@pytest.mark.parametrize("new, kept", [([1, 1], [77, 300]), ([3, 2], [129, 10]), ([50, 7], [50, 400])])
def test_attention_shared_heads(kv4, share, new, kept, dtype):
    cache = filled(kv4, 40, 20, 2, 128, 64)
    attend(kv4, cache, new, kept, 2 * share, dtype)


@pytest.mark.parametrize("page", [1, 3, 16, 20, 64, 256])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("new, kept", [([1, 1, 1], [3, 250, 129]), ([6, 40], [6, 300])])
def test_attention_pages_and_layouts(kv4, page, token_major, new, kept):
    cache = filled(kv4, sum(-(-n // page) for n in kept) + 1, page, 2, 128, 64, token_major=token_major)
    attend(kv4, cache, new, kept, 8, torch.bfloat16)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [0, 1, 2, 63, 64, 65, 1000])
@pytest.mark.parametrize("new, kept", [([1, 1], [300, 64]), ([5, 4], [300, 4]), ([70, 129], [333, 129])])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_masks(kv4, causal, window, new, kept, dim):
    cache = filled(kv4, 40, 16, 1, dim, 32)
    attend(kv4, cache, new, kept, 4, torch.float16, causal=causal, window=window, scale=0.2)


@pytest.mark.parametrize("new, kept", [([4], [2]), ([40, 2], [7, 0]), ([200], [30])])
def test_attention_rows_that_see_nothing_are_zero(kv4, new, kept):
    cache = filled(kv4, 8, 16, 2, 128, 128)
    out, _ = attend(kv4, cache, new, kept, 4, torch.bfloat16)
    at = 0
    for n, k in zip(new, kept):
        assert (out[at:at + max(0, n - k)] == 0).all()
        at += n


@pytest.mark.parametrize("heads", [4, 40])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_attention_ignores_what_no_query_sees(kv4, heads, new):
    """NaN and infinities in rows behind the last, before the window, and in pages of nobody change no bit."""
    page, kept, window = 16, 203, 100
    cache = filled(kv4, 20, page, 2, 128, 32)
    table = tables([kept], page, 20)
    q = randn(3, new, heads, 128, dtype=torch.float16)
    lens = torch.tensor([kept], dtype=torch.int32, device="cuda")

    def go():
        return cache.attention(q, table, lens, max_new=new, max_kept=kept, window=window)

    clean = go()
    j = torch.arange(20 * page, device="cuda")
    used = torch.zeros(20 * page, dtype=torch.bool, device="cuda")
    at = torch.arange(max(0, kept - new - window + 1), kept, device="cuda")
    used[table[0].long()[at // page] * page + at % page] = True
    bad = (~used).view(20, page)
    for t in (cache.k_params, cache.v_params):
        view = t.transpose(1, 2)
        view[bad] = torch.tensor([math.nan, math.inf], dtype=torch.float16, device="cuda")
    for t in (cache.k_codes, cache.v_codes):
        t.transpose(1, 2)[bad] = 255
    assert torch.equal(go(), clean) and torch.isfinite(clean).all()


@pytest.mark.parametrize("new", [1, 2, 80])
def test_attention_passes_visible_nan_on(kv4, new):
    """A key row stored as NaN makes the rows that see it NaN, a value group stored as NaN that group of them."""
    cache = filled(kv4, 8, 16, 2, 128, 64)
    table = tables([100], 16, 8)
    q = randn(3, new, 4, 128, dtype=torch.bfloat16)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    page = int(table[0, 99 // 16])
    cache.v_params[page, 0, 99 % 16, 1] = math.nan
    out = cache.attention(q, table, lens, max_new=new)
    assert torch.isnan(out[-1, :2, 64:]).all() and torch.isfinite(out[-1, :2, :64]).all() and torch.isfinite(out[-1, 2:]).all()
    assert torch.isfinite(out[:-1]).all()
    cache.k_params[page, 1, 99 % 16, 0] = math.nan
    out = cache.attention(q, table, lens, max_new=new)
    assert torch.isnan(out[-1, 2:]).all() and torch.isfinite(out[:-1]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("gain", [1e-3, 30.0, 1000.0])
def test_attention_of_small_and_large_values(kv4, dtype, new, gain):
    """Scores from flat to one-hot and values far from one; the shares stay finite and in bounds."""
    cache = kv4.Kv4Cache.allocate(20, 16, 2, 64, 64)
    n = 320
    cache.append(randn(1, n, 2, 64), randn(2, n, 2, 64) * gain, torch.arange(n, device="cuda"))
    q = (randn(3, new, 8, 64) * 2 if gain < 100 else randn(3, new, 8, 64) * 50).to(dtype)
    table = tables([317], 16, 20)
    got = cache.attention(q, table, torch.tensor([317], dtype=torch.int32, device="cuda"), max_new=new)
    want, size, dots = R.attention(cache, q, table, [317], [0, new])
    g, d = got.double(), dots
    # as in decoder_ref.check_attention, with the score's error where the scores are large
    e = 2.0 * d * (2.0 ** -11 + 2.0 ** -16)
    tol = R.U[dtype] * want.abs() + R.TINY[dtype] + size * (2.0 ** -8 + 2.0 ** -11 + torch.expm1(e.clamp_max(5.0)))
    assert torch.isfinite(g).all() and ((g - want).abs() <= tol).all()


def test_attention_bad_pages_and_lengths_are_reported(kv4):
    """A page outside the cache is not read and its rows do not count; lengths beyond the bounds are cut."""
    for new in (1, 4, 80):
        cache = filled(kv4, 12, 16, 2, 128, 64)
        table = tables([150], 16, 12)
        q = randn(3, new, 8, 128, dtype=torch.bfloat16)
        starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        for bad in (-5, 12, 1 << 30):
            broken = table.clone()
            broken[0, 2] = bad
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            got = cache.attention(q, broken, torch.tensor([150], dtype=torch.int32, device="cuda"), max_new=new, max_kept=150, status=status)
            assert int(status) == kv4.STATUS_BAD_INDEX
            hidden = torch.zeros((1, 150), dtype=torch.bool, device="cuda")
            hidden[0, 32:48] = True
            R.check_attention(got, *R.attention(cache, q, table, [150], [0, new], hidden=hidden), new, bad)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = cache.attention(q, table, torch.tensor([151], dtype=torch.int32, device="cuda"), q_starts=starts, max_new=new, max_kept=150, status=status)
        assert int(status) == kv4.STATUS_BAD_INDEX
        R.check_attention(got, *R.attention(cache, q, table, [150], [0, new]), new, "cut")
        for wrong in ([0, new + 1], [-3, new], [new + 1, new + 2], [2, 1], [-(1 << 31), (1 << 31) - 1]):
            status.zero_()
            out = torch.full_like(q, 7.0)
            cache.attention(q, table, torch.tensor([150], dtype=torch.int32, device="cuda"), q_starts=torch.tensor(wrong, dtype=torch.int32, device="cuda"),
                            max_new=new, max_kept=150, status=status, out=out)
            torch.cuda.synchronize()
            assert int(status) == kv4.STATUS_BAD_INDEX


def test_attention_beyond_32_bit_offsets(kv4):
    """A pool whose codes pass 2^32 bytes, its pages at both ends of it."""
    page, dim = 64, 256
    pages = (1 << 32) // (page * dim // 2) + 40
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    cache = kv4.Kv4Cache.allocate(pages, page, 1, dim, 128)
    table = torch.tensor([[pages - 1, 0, pages - 30, 5, pages - 2]], dtype=torch.int32, device="cuda")
    n = 5 * page - 7
    j = torch.arange(n, device="cuda")
    slots = table[0].long()[j // page] * page + j % page
    cache.append(randn(1, n, 1, dim), randn(2, n, 1, dim), slots)
    back = cache.gather(slots, torch.float32)[1]
    assert float((back - randn(2, n, 1, dim)).abs().max()) < 1.0
    for new in (1, 40):
        q = randn(3, new, 4, dim, dtype=torch.bfloat16)
        got = cache.attention(q, table, torch.tensor([n], dtype=torch.int32, device="cuda"), max_new=new)
        R.check_attention(got, *R.attention(cache, q, table, [n], [0, new]), new, "far pages")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("most", [1, 8, 23])
def test_attention_of_many_sequences(kv4, most, dtype):
    """More sequences than a block has threads, most of them short or idle."""
    new = [(7 * b) % (most + 1) for b in range(330)]
    new[5] = most
    kept = [n + (37 * b) % 90 if n else 0 for b, n in enumerate(new)]
    cache = filled(kv4, sum(-(-n // 16) for n in kept) + 1, 16, 1, 64, 64)
    attend(kv4, cache, new, kept, 4, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 256])
def test_attention_prompts_of_all_lengths(kv4, dim, dtype):
    """Odd and even numbers of tiles follow each other in a block's part, with one half of rows and with two."""
    new = [1, 63, 64, 65, 127, 129, 190, 0, 257, 33, 320, 5]
    kept = [n + (0, 64, 130, 3)[b % 4] if n else 0 for b, n in enumerate(new)]
    cache = filled(kv4, sum(-(-n // 16) for n in kept) + 1, 16, 3, dim, 64)
    attend(kv4, cache, new, kept, 6, dtype)
    attend(kv4, cache, new, kept, 6, dtype, window=50)


@pytest.mark.parametrize("share, new", [(4, 8), (3, 11), (32, 1), (33, 1)])
def test_attention_on_both_sides_of_the_choice_of_kernel(kv4, share, new):
    cache = filled(kv4, 40, 16, 2, 128, 128)
    attend(kv4, cache, [new, 1], [300, 200], 2 * share, torch.float16)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-4])
@pytest.mark.parametrize("new", [2, 70])
def test_attention_of_any_scale(kv4, scale, new):
    cache = filled(kv4, 30, 16, 2, 64, 32)
    for dtype in (torch.float16, torch.bfloat16):
        attend(kv4, cache, [new, 1], [300, 100], 8, dtype, scale=scale)


def test_a_captured_prompt_replays(kv4):
    """Lengths, tables and rows are read at each replay; max_new and max_kept only bound them."""
    cache = filled(kv4, 120, 16, 2, 128, 64)
    q, kept, starts = randn(1, 300, 8, 128, dtype=torch.float16), ints([0, 0]), ints([0, 0, 0])
    table = tables([900, 900], 16, 120)
    out = torch.empty_like(q)
    cache.attention(q, table, kept, q_starts=starts, max_new=200, max_kept=900, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attention(q, table, kept, q_starts=starts, max_new=200, max_kept=900, out=out)
    for new, have in (([200, 100], [900, 100]), ([1, 0], [1, 0]), ([70, 130], [500, 130]), ([0, 1], [30, 30])):
        kept.copy_(ints(have))
        starts.copy_(ints([0, new[0], sum(new)]))
        g.replay()
        want, size, dots = R.attention(cache, q, table, have, [0, new[0], sum(new)])
        R.check_attention(out, want, size, dots, sum(new), (new, have))


def test_attention_strided_queries_and_outputs(kv4):
    cache = filled(kv4, 30, 16, 2, 128, 64)
    table = tables([100, 200], 16, 30)
    lens = torch.tensor([100, 200], dtype=torch.int32, device="cuda")
    for new in (1, 3, 60):
        for offset, pad in ((0, 0), (3, 1)):
            width = 12 * 128 + pad
            buf = randn(1, 2 * new * width + offset, dtype=torch.bfloat16)
            q = buf[offset:].view(2 * new, width)[:, 128:9 * 128].unflatten(1, (8, 128))
            plain = cache.attention(q.contiguous(), table, lens, max_new=new)
            hold = torch.full((2 * new * width + offset,), 3.0, dtype=torch.bfloat16, device="cuda")
            out = hold[offset:].view(2 * new, width)[:, :8 * 128].unflatten(1, (8, 128))
            cache.attention(q, table, lens, max_new=new, out=out)
            assert torch.equal(out, plain)
            assert (hold[offset:].view(2 * new, width)[:, 8 * 128:] == 3.0).all()


# --------------------------------------------------------------------------------------- a layer's run, streams, graphs

class Layer:
    """What a decoder layer does between its QKV linear and its output linear, and the same in 64 bits."""

    def __init__(self, kv4, K, seqs, heads=8, kv_heads=2, dim=128, page=16, pages=64):
        self.K, self.heads, self.kv_heads, self.dim, self.page = K, heads, kv_heads, dim, page
        self.cache = kv4.Kv4Cache.allocate(pages, page, kv_heads, dim, 64)
        self.freq, self.m = kv4.rope_frequencies(dim, scaling="by_parts", factor=4.0, trained=256)
        self.wq, self.wk = 1 + 0.1 * randn(50, dim).to(torch.bfloat16), 1 + 0.1 * randn(51, dim).to(torch.bfloat16)
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)[:seqs * (pages // seqs)].view(seqs, -1).cuda()

    def __call__(self, qkv, positions, slots, kept, starts, max_new, max_kept):
        nq, nk = self.heads * self.dim, self.kv_heads * self.dim
        q = qkv[:, :nq].unflatten(1, (self.heads, self.dim))
        k = qkv[:, nq:nq + nk].unflatten(1, (self.kv_heads, self.dim))
        v = qkv[:, nq + nk:].unflatten(1, (self.kv_heads, self.dim))
        q, k = self.K.qk_norm_rope(q, k, self.wq, self.wk, positions, self.freq, mscale=self.m)
        self.cache.append(k, v, slots)
        return self.cache.attention(q, self.table, kept, q_starts=starts, max_new=max_new, max_kept=max_kept), q

    def slots(self, seq, pos):
        return self.table[seq].long()[pos // self.page] * self.page + pos % self.page


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def test_a_layer_prefills_and_decodes(K, kv4):
    """Ragged prompts, then steps of one token each (the second sequence idle in one of them), padded rows in the batch."""
    layer = Layer(kv4, K, 3)
    kept = [0, 0, 0]
    for step, new in enumerate([[70, 33, 1], [1, 1, 1], [1, 0, 1], [2, 1, 40]]):
        starts, pos, slots = [0], [], []
        for b, n in enumerate(new):
            p = torch.arange(kept[b], kept[b] + n, device="cuda")
            pos.append(p)
            slots.append(layer.slots(b, p))
            kept[b] += n
            starts.append(starts[-1] + n)
        pad = 2
        pos.append(torch.zeros(pad, dtype=torch.int64, device="cuda"))
        slots.append(torch.full((pad,), -1, dtype=torch.int64, device="cuda"))
        qkv = randn(100 + step, starts[-1] + pad, (layer.heads + 2 * layer.kv_heads) * layer.dim, dtype=torch.bfloat16)
        out, q = layer(qkv, torch.cat(pos), torch.cat(slots), ints(kept), ints(starts), max(new), max(kept))
        R.check_attention(out, *R.attention(layer.cache, q, layer.table, kept, starts), starts[-1], (step, new))
        # what the cache now holds is what went in, to half a step
        at = torch.cat(slots)[:starts[-1]]
        back = layer.cache.gather(at, torch.float32)[1]
        v = qkv[:starts[-1], -layer.kv_heads * layer.dim:].unflatten(1, (layer.kv_heads, layer.dim)).float()
        step_size = stored(layer.cache, at, "v")[1][..., 1].float().repeat_interleave(64, -1)
        assert ((back - v).abs() <= step_size * 0.52 + v.abs().amax() * 2.0 ** -11).all()


def test_a_captured_step_replays(K, kv4):
    """One decoding step as a CUDA graph, lengths, slots and rows read from device memory at each replay; two graphs on one pool."""
    layer = Layer(kv4, K, 2, pages=40)
    heads_all = (layer.heads + 2 * layer.kv_heads) * layer.dim
    first = randn(1, 60, heads_all, dtype=torch.bfloat16)
    pos = torch.cat([torch.arange(30), torch.arange(30)]).cuda()
    seq_slots = torch.cat([layer.slots(b, torch.arange(30, device="cuda")) for b in range(2)])
    layer(first, pos, seq_slots, ints([30, 30]), ints([0, 30, 60]), 30, 30)
    qkv, pos, slots, kept, starts = torch.zeros((2, heads_all), dtype=torch.bfloat16, device="cuda"), ints([0, 0], torch.int64), ints([-1, -1], torch.int64), \
        ints([0, 0]), ints([0, 1, 2])
    layer(qkv, pos, slots, kept, starts, 1, 300)
    graphs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out, q = layer(qkv, pos, slots, kept, starts, 1, 300)
        graphs.append((g, out, q))
    n = [30, 30]
    for step in range(6):
        g, out, q = graphs[step % 2]
        qkv.copy_(randn(200 + step, 2, heads_all, dtype=torch.bfloat16))
        pos.copy_(ints(n, torch.int64))
        slots.copy_(torch.stack([layer.slots(b, pos[b]) for b in range(2)]))
        n = [v + 1 for v in n]
        kept.copy_(ints(n))
        g.replay()
        R.check_attention(out, *R.attention(layer.cache, q, layer.table, n, [0, 1, 2]), 2, step)
        want = layer.cache.attention(q, layer.table, kept, q_starts=starts, max_new=1, max_kept=300)
        assert torch.equal(out, want)


def test_calls_on_other_streams_at_once(K, kv4):
    """Calls on two streams at the same time give what each gives alone."""
    cache = filled(kv4, 140, 16, 2, 128, 64)
    table = tables([1000, 1100], 16, 140)
    lens = ints([1000, 1100])
    cases = [(randn(s, 2 * new, 8, 128, dtype=torch.bfloat16), new) for s, new in ((1, 1), (2, 3), (3, 70), (4, 1))]
    alone = [cache.attention(q, table, lens, max_new=n, max_kept=1100) for q, n in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, (q, n) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(cache.attention(q, table, lens, max_new=n, max_kept=1100))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))


def test_python_face_refuses_on_gpu(K, kv4):
    cache = kv4.Kv4Cache.allocate(4, 16, 2, 64, 32)
    q, lens, table = randn(1, 2, 4, 64, dtype=torch.bfloat16), ints([3, 4]), torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    k = randn(1, 2, 2, 64)
    bad = [lambda: cache.attention(q.float(), table, lens), lambda: cache.attention(q, table.long(), lens), lambda: cache.attention(q, table[:1], lens),
           lambda: cache.attention(q, table, lens.long()), lambda: cache.attention(q[:, :3], table, lens), lambda: cache.attention(q, table, lens, max_new=2),
           lambda: cache.attention(q, table, lens, q_starts=ints([0, 1])), lambda: cache.attention(q, table, lens, out=q.half()),
           lambda: cache.attention(q, table.cpu(), lens), lambda: cache.append(k, k, torch.zeros(3, dtype=torch.int64, device="cuda")),
           lambda: cache.append(k, k[:, :1], ints([0, 1])), lambda: cache.append(k, k, ints([0, 1]), positions=ints([0, 1])),
           lambda: cache.append(k, k, ints([0, 1]), positions=ints([0, 1]), inv_freq=torch.ones(33, dtype=torch.float64, device="cuda")),
           lambda: cache.append(k, k, ints([0, 1]), status=ints([0, 0])), lambda: cache.gather(ints([0]), torch.int8), lambda: cache.gather(ints([0]), out_k=k),
           lambda: kv4.Kv4Cache(cache.k_codes, cache.k_params, cache.v_codes[:2], cache.v_params), lambda: kv4.Kv4Cache.allocate(4, 16, 2, 96, 32).append(randn(1, 1, 2, 96), randn(1, 1, 2, 96), ints([0])),
           lambda: K.rope(k, ints([0, 1]), torch.ones(32, device="cuda")), lambda: K.rope(k, ints([0, 1]), torch.ones(33, dtype=torch.float64, device="cuda")),
           lambda: K.qk_norm_rope(k, k, torch.ones(64, device="cuda"), torch.ones(64, device="cuda").half(), ints([0, 1]), torch.ones(32, dtype=torch.float64, device="cuda"))]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError, KeyError)):
            call()
            pytest.fail("call %d was taken" % i)
