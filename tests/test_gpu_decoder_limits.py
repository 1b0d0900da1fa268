"""The decoder operators at the edges of what they take, on the GPU: scores, values and steps of any size, bounds that tell the
roundings of one type from another's."""
import importlib
import math

import pytest
import torch

import decoder_bounds as B

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


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def table_of(pages, seed=5):
    return torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)[None].cuda()


# ------------------------------------------------------------------------------------------------------ scores of any size

def far_scores(kv4, dim, kept, sign, seed=3):
    """A cache whose keys are the same whole number in every channel, so that products with queries of ones are exact; the largest is
    there three times (at the first, a middle and the last token), one less than it once."""
    pages = -(-kept // 16)
    cache = kv4.Kv4Cache.allocate(pages, 16, 1, dim, 32)
    a = torch.randint(-1000, 1000, (kept,), generator=torch.Generator().manual_seed(seed)).double()
    a[[0, kept // 2, kept - 1]] = 1001.0
    a[kept // 3] = 1000.0
    if sign < 0:      # all scores far below zero
        a = a - 1024.0
    table = table_of(pages)
    j = torch.arange(kept, device="cuda")
    slots = table[0].long()[j // 16] * 16 + j % 16
    k = a.cuda().float()[:, None, None].expand(kept, 1, dim).contiguous()
    cache.append(k, randn(seed, kept, 1, dim), slots)
    assert torch.equal(cache.gather(slots, torch.float32)[0], k)
    return cache, table


def check_far_scores(kv4, dtype, dim, power, sign, new, kept=700):
    cache, table = far_scores(kv4, dim, kept, sign)
    q = torch.ones((new, 1, dim), device="cuda", dtype=dtype)
    scale = 2.0 ** power / (1024.0 * dim)         # scores up to 2^power
    out = cache.attention(q, table, ints([kept]), max_new=new, max_kept=kept, scale=scale)
    r = B.attention(cache, q, table, [kept], [0, new], scale=scale)
    # products are exact; scale * log2(e) is off by 2^-23 of itself, which enters through differences of scores that count (below 32);
    # up to scores of 2^10 7 - maximum is rounded to 2^-14, twice
    B.check(out, r, score=torch.full_like(r["dots"], 2.0 ** -13), context=(power, sign))


POWERS = [3, 9, 10, 11, 16, 24, 27, 28, 29, 30, 34, 40, 60, 120]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("dim", [64, 256])
def test_many_rows_with_scores_of_any_size(kv4, dtype, dim, power, sign):
    """Scores far beyond what an fp32 exponent resolves: equal largest ones share the output, all others are nothing."""
    check_far_scores(kv4, dtype, dim, power, sign, new=70)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_many_rows_with_queries_of_any_finite_value(kv4, dtype):
    """Rows of a padded batch may hold anything: the largest numbers of the type, both signs, mixed with ordinary rows and with keys that
    answer them with both signs.  Finite queries give finite shares, and the ordinary rows are right beside them."""
    cache = kv4.Kv4Cache.allocate(12, 16, 2, 128, 64)
    n, new = 190, 64
    loud = 1.0 + 999.0 * (torch.arange(128, device="cuda") % 23 == 5)
    cache.append(randn(1, n, 2, 128) * loud, randn(2, n, 2, 128), torch.arange(n, device="cuda"))
    table = torch.arange(12, dtype=torch.int32, device="cuda")[None]
    q = randn(3, new, 4, 128, dtype=dtype)
    plain = cache.attention(q, table, ints([n]), max_new=new)
    wild = q.clone()
    size = torch.finfo(dtype).max * 2.0 ** -torch.arange(32, dtype=torch.float64, device="cuda")
    wild[1::2] = torch.where(wild[1::2] > 0, size[:, None, None], -size[:, None, None]).to(dtype)
    out = cache.attention(wild, table, ints([n]), max_new=new)
    assert torch.isfinite(out).all()
    v = cache.gather(torch.arange(n, device="cuda"), torch.float32)[1].abs().amax()
    assert float(out.float().abs().max()) <= float(v) * (1 + 2.0 ** -7)
    # a warp takes its maxima off either way for all its rows: ordinary rows agree to the roundings of both
    r = B.attention(cache, q, table, [n], [0, new])
    tol = B.tolerance(r, dtype)
    for x in (plain, out):
        assert ((x.double() - r["out"]).abs() <= tol)[0::2].all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", POWERS)
@pytest.mark.parametrize("dim, new", [(64, 1), (128, 3), (256, 12)])
def test_few_rows_with_scores_of_any_size(kv4, dtype, dim, new, power, sign):
    check_far_scores(kv4, dtype, dim, power, sign, new)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_few_rows_with_queries_of_any_finite_value(kv4, dtype):
    """As for many rows; each query row here is alone in its sequence."""
    cache = kv4.Kv4Cache.allocate(12, 16, 2, 128, 64)
    n, seqs = 190, 32
    loud = 1.0 + 999.0 * (torch.arange(128, device="cuda") % 23 == 5)
    cache.append(randn(1, n, 2, 128) * loud, randn(2, n, 2, 128), torch.arange(n, device="cuda"))
    table = torch.arange(12, dtype=torch.int32, device="cuda")[None].expand(seqs, 12)
    size = torch.finfo(dtype).max * 2.0 ** -torch.arange(seqs, dtype=torch.float64, device="cuda")
    wild = torch.where(randn(3, seqs, 4, 128) > 0, size[:, None, None], -size[:, None, None]).to(dtype)
    out = cache.attention(wild, table, ints([n] * seqs), max_new=1)
    v = cache.gather(torch.arange(n, device="cuda"), torch.float32)[1].abs().amax()
    assert torch.isfinite(out).all() and float(out.float().abs().max()) <= float(v) * (1 + 2.0 ** -7)


# ------------------------------------------------------------------------------------------------------ values of any size

def check_values(kv4, dtype, dim, group, gains, new, seed=1, heads=4, keys=1.0, norm=None, **kw):
    """Attention over values of standard deviation gains[token, channel]."""
    n = gains.shape[0]
    pages = -(-n // 16)
    cache = kv4.Kv4Cache.allocate(pages, 16, 2, dim, group)
    table = table_of(pages)
    j = torch.arange(n, device="cuda")
    slots = table[0].long()[j // 16] * 16 + j % 16
    v = randn(seed + 1, n, 2, dim) * gains.cuda().float()[:, None, :]
    cache.append(randn(seed, n, 2, dim) * keys, v.clamp(-60000.0, 60000.0), slots)
    q = randn(seed + 2, new, heads, dim, dtype=dtype)
    out = cache.attention(q, table, ints([n]), max_new=new, max_kept=n, **kw)
    B.check(out, B.attention(cache, q, table, [n], [0, new], **kw), norm=norm, context=(dim, group, new))


SHAPES = [(64, 64), (128, 32), (128, 128), (256, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gain", [1.0, 1e-3, 3e-4, 1e-4, 1e-5, 300.0, 15000.0])
@pytest.mark.parametrize("dim, group", SHAPES)
@pytest.mark.parametrize("new", [1, 6])
def test_few_rows_with_values_of_any_size(kv4, dtype, gain, dim, group, new):
    """The product of a weight and a step keeps its digits whatever the steps are.  Below 0.1 a half's output has fewer digits of its own."""
    norm = 2.1e-3 if dtype == torch.bfloat16 else (3.3e-4 if gain >= 1.0 else None)
    check_values(kv4, dtype, dim, group, torch.full((417, dim), gain), new, norm=norm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group", SHAPES)
@pytest.mark.parametrize("kind", ["rising", "falling", "groups", "one"])
def test_few_rows_with_values_of_all_sizes_at_once(kv4, dtype, dim, group, kind):
    n = 600
    if kind == "groups":            # neighbouring groups of channels far apart
        gains = (1e-5 * 10.0 ** (9.0 * torch.arange(dim, dtype=torch.float64).div(group, rounding_mode="floor") * group / dim)).expand(n, dim)
    elif kind == "one":             # a single loud token late in the context
        gains = torch.full((n, dim), 1e-3, dtype=torch.float64)
        gains[500] = 5000.0
    else:
        gains = (10.0 ** torch.linspace(-5.0, 4.0, n, dtype=torch.float64))[:, None].expand(n, dim)
        gains = gains.flip(0) if kind == "falling" else gains
    for new in (1, 5):
        check_values(kv4, dtype, dim, group, gains, new)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tail, power", [(3000, 20), (3000, 23), (50000, 17), (50000, 21)])
def test_few_rows_with_one_token_above_a_long_tail(kv4, dtype, tail, power):
    """One token's weight is 2^power times that of each other; their values are alike, so what is lost of each is lost of the sum."""
    dim, n = 128, tail + 1
    pages = -(-n // 16)
    cache = kv4.Kv4Cache.allocate(pages, 16, 1, dim, 64)
    slots = torch.arange(n, device="cuda")
    k = torch.zeros((n, 1, dim), device="cuda")
    k[7] = 1.0
    v = 0.9 + 0.1 * torch.rand((n, 1, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    v[..., 0::64], v[7] = -1.0, 0.0                       # ranges of 2 around values near their upper end; the one token's is zero
    cache.append(k, v, slots)
    q = torch.ones((1, 2, dim), dtype=dtype, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    scale = power * math.log(2.0) / dim
    out = cache.attention(q, table, ints([n]), max_new=1, max_kept=n, scale=scale)
    r = B.attention(cache, q, table, [n], [0, 1], scale=scale)
    B.check(out, r, score=torch.full_like(r["dots"], power * 2.0 ** -21), context=(tail, power))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gain", [1.0, 1e-3, 3e-4, 1e-4, 1e-5, 300.0, 15000.0])
@pytest.mark.parametrize("dim, group", SHAPES)
def test_many_rows_with_values_of_any_size(kv4, dtype, gain, dim, group):
    """Groups whose range is wider than the largest half are right too: each of their values is one."""
    norm = 2.1e-3 if dtype == torch.bfloat16 else (3.3e-4 if 1.0 <= gain <= 300.0 else None)
    check_values(kv4, dtype, dim, group, torch.full((417, dim), gain), 60, norm=norm)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group", SHAPES)
@pytest.mark.parametrize("new", [1, 60])
def test_keys_of_wide_range(kv4, dtype, dim, group, new):
    check_values(kv4, dtype, dim, group, torch.ones(300, dim), new, keys=12000.0, scale=1e-5)
    gains = torch.where(torch.arange(dim) < group, 1e-3, 14000.0).double().expand(300, dim)
    check_values(kv4, dtype, dim, group, gains, new)


def test_append_of_ranges_at_the_end_of_halves(kv4):
    """Any group of finite halves is stored as halves; what passes them by more than a lower step makes up for is stored as NaN."""
    ends = [(-65504.0, 65504.0, True), (0.0, 65504.0, True), (-65504.0, 65519.0, True), (-65519.0, -65500.0, True), (65504.0, 65504.0, True), (60000.0, 65519.9, True),
            (-40000.0, 40000.0, True),
            (0.0, 65521.0, True),      # 65521 / 15 rounds to 4368, 15 times that to infinity; 15 * 4364 = 65460 does not
            (-3.0, 70000.0, False), (0.0, 900000.0, False), (-65504.0, 900000.0, False), (-65521.0, 0.0, False),
            (0.0, math.inf, False), (-math.inf, 0.0, False), (0.0, 3e38, False), (-3e38, 3e38, False)]
    n, group = len(ends), 64
    x = torch.rand((n, 1, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    for i, (low, high, _) in enumerate(ends):
        if math.isfinite(low) and math.isfinite(high):
            x[i, 0, :group] = low + (high - low) * x[i, 0, :group].double()
        x[i, 0, 11], x[i, 0, 42] = low, high
    cache = kv4.Kv4Cache.allocate(2, 16, 1, 128, group)
    slots = torch.arange(n, device="cuda")
    cache.append(x, x, slots)
    k, v = cache.gather(slots, torch.float32)
    half = cache.gather(slots, torch.float16)[0]
    assert torch.equal(k.view(torch.int32), v.view(torch.int32)) and torch.isfinite(k[..., group:]).all()
    for i, (low, high, fits) in enumerate(ends):
        got = k[i, 0, :group].double()
        if not fits:
            assert torch.isnan(got).all()
            continue
        assert torch.isfinite(half[i]).all()
        lo, step = (float(cache.k_params[0, 0, i, 0, e]) for e in (0, 1))
        assert lo + 15 * step < 65520
        # half a step, and what the roundings of lo and step move: step down by up to one unit, 2^-10 of it, 15 times
        off = (got - x[i, 0, :group].double()).abs().amax()
        assert off <= step * (0.5 + 15 * 2.0 ** -10 + 2.0 ** -20) + abs(lo) * 2.0 ** -11


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [3, 60])
@pytest.mark.parametrize("pair", [(60000.0, 3000.0), (65504.0, 65504.0), (-60000.0, 65504.0), (math.inf, 0.0), (0.0, math.inf), (math.nan, math.nan)])
def test_pairs_past_halves_touch_no_other_row(kv4, dtype, new, pair):
    n = 150
    cache = kv4.Kv4Cache.allocate(10, 16, 2, 128, 64)
    cache.append(randn(1, n, 2, 128), randn(2, n, 2, 128), torch.arange(n, device="cuda"))
    q, table = randn(3, new, 4, 128, dtype=dtype), torch.arange(10, dtype=torch.int32, device="cuda")[None]
    clean = cache.attention(q, table, ints([n]), max_new=new)
    tol = B.tolerance(B.attention(cache, q, table, [n], [0, new]), dtype)
    page, off = (n - 1) // 16, (n - 1) % 16
    for side in (cache.v_params, cache.k_params):
        side[page, 0, off, 1] = torch.tensor(pair, dtype=torch.float16, device="cuda")
        out = cache.attention(q, table, ints([n]), max_new=new)
        assert torch.equal(out[-1, 2:], clean[-1, 2:])
        if new > 3:
            assert torch.equal(out[:-1], clean[:-1])
        else:
            # The few-row kernel scales a group's steps by one power of two for all rows of a warp, so that the largest is at least 2^9: a
            # product of a weight and a small step is then off by up to 2^-25 of its unit, 2^-34 of the largest step in the weights'
            # unit, where a row's weights add up to 2^-2 at least.  At 8 steps' distance, over n tokens: n * step * 2^-29.  All rows of a
            # warp move their maxima together, so that the weights' roundings differ too: each result is within `tolerance`.
            s = pair[1] if math.isfinite(pair[1]) else 0.0
            assert ((out.double() - clean.double()).abs() <= n * s * 2.0 ** -29 + 2.0 * tol)[:-1].all()
        if math.isnan(pair[0]):
            assert torch.isnan(out[-1, :2]).any(-1).all()


# ----------------------------------------------------------------------------------------------------- queries of any size

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 2e-5, 1000.0])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 4, 60])
def test_queries_of_any_size(kv4, dtype, size, dim, new):
    """Small queries with a large scale: no channel loses digits."""
    n = 260
    cache = kv4.Kv4Cache.allocate(17, 16, 2, dim, 64)
    slots = torch.arange(n, device="cuda")
    cache.append(randn(1, n, 2, dim), randn(2, n, 2, dim), slots)
    q = randn(3, new, 6, dim) * size
    q[:, 1, :dim // 2] *= 64.0                   # rows with a loud and a quiet half
    q[:, 3] *= 1.0 + 500.0 * (torch.arange(dim, device="cuda") % 16 == 0)
    q[:, 1], q[:, 3] = q[:, 1] * 0.02, q[:, 3] * 0.004
    q = q.to(dtype)
    scale = 2.0 / (size * dim ** 0.5)
    table = torch.arange(17, dtype=torch.int32, device="cuda")[None]
    out = cache.attention(q, table, ints([n]), max_new=new, scale=scale)
    r = B.attention(cache, q, table, [n], [0, new], scale=scale)
    # fp32 sums of up to 256 products, 16 at a time, in two roundings each: 2^-19 of the sum of magnitudes
    score = None if r["many"] else r["dots"] * 2.0 ** -18
    B.check(out, r, score=score, norm=2.1e-3 if dtype == torch.bfloat16 and new < 60 else None, context=(size, dim, new))


# ------------------------------------------------------------------------------------------------------------- the boundary

@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_a_workspace_aligned_to_sixteen_bytes_and_no_more(kv4, dim, new):
    """One sequence that many blocks share, so that their results go through the workspace; nothing before or behind it is written."""
    n = 5000
    cache = kv4.Kv4Cache.allocate(320, 16, 2, dim, 32)
    cache.append(randn(1, n, 2, dim), randn(2, n, 2, dim), torch.arange(n, device="cuda"))
    q, table = randn(3, new, 4, dim, dtype=torch.bfloat16), torch.arange(320, dtype=torch.int32, device="cuda")[None]
    want = cache.attention(q, table, ints([n]), max_new=new)
    with pytest.raises(RuntimeError, match="workspace of") as refusal:
        cache.attention(q, table, ints([n]), max_new=new, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    need = int(str(refusal.value).split("workspace of ")[1].split()[0])
    hold = torch.full((need + 128,), 0x5A, dtype=torch.uint8, device="cuda")
    at = (16 - hold.data_ptr()) % 32                 # 16 bytes past a multiple of 32
    got = cache.attention(q, table, ints([n]), max_new=new, workspace=hold[at:at + need])
    assert torch.equal(got, want) and (hold[:at] == 0x5A).all() and (hold[at + need:] == 0x5A).all()
    with pytest.raises(RuntimeError, match="16-byte aligned workspace"):
        cache.attention(q, table, ints([n]), max_new=new, workspace=hold[at + 8:at + 8 + need])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim, group", [(64, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("window", [0, 70])
def test_value_groups_stored_as_nan_reach_the_rows_that_see_them_and_no_other(kv4, dtype, dim, group, window):
    """Many rows, several sequences and heads, units that blocks share: NaN exactly where a visible token's group is NaN."""
    new, kept, share, kvh, page = [300, 5, 129], [900, 40, 129], 2, 2, 16
    need = [-(-n // page) for n in kept]
    cache = kv4.Kv4Cache.allocate(sum(need), page, kvh, dim, group)
    rows = sum(need) * page
    cache.append(randn(1, rows, kvh, dim), randn(2, rows, kvh, dim), torch.arange(rows, device="cuda"))
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    for b in range(3):
        table[b, :need[b]] = torch.arange(sum(need[:b]), sum(need[:b + 1]), dtype=torch.int32)
    starts = [0, 300, 305, 434]
    q = randn(3, starts[-1], kvh * share, dim, dtype=dtype)

    def go():
        return cache.attention(q, table.cuda(), ints(kept), q_starts=ints(starts), max_new=300, max_kept=900, window=window)

    clean = go()
    assert torch.isfinite(clean).all()
    expect = torch.zeros(clean.shape, dtype=torch.bool, device="cuda")
    for b, tok, h, g in [(0, 0, 0, 0), (0, 613, 1, 1), (0, 613, 1, 0), (0, 899, 0, 1), (1, 38, 0, 1), (2, 64, 1, 0), (2, 127, 1, 1)]:
        cache.v_params[int(table[b, tok // page]), h, tok % page, g] = math.nan
        place = torch.arange(new[b], device="cuda") + kept[b] - new[b]
        sees = (place >= tok) & ((place - window < tok) if window else True)
        expect[starts[b]:starts[b + 1], h * share:(h + 1) * share, g * group:(g + 1) * group] |= sees[:, None, None]
    out = go()
    assert torch.equal(torch.isnan(out), expect) and torch.equal(out[~expect], clean[~expect])


def test_a_value_group_stored_as_nan_costs_little(kv4):
    """One NaN group at the start of a long list of sequences: the other segments of a block do not look for it."""
    seqs, new, kept = 64, 64, 2048
    cache = kv4.Kv4Cache.allocate(seqs * kept // 64, 64, 8, 128, 64)
    rows = seqs * kept
    for at in range(0, rows, 1 << 14):
        cache.append(randn(1, 1 << 14, 8, 128, dtype=torch.bfloat16), randn(2, 1 << 14, 8, 128, dtype=torch.bfloat16), torch.arange(at, at + (1 << 14), device="cuda"))
    table = torch.arange(rows // 64, dtype=torch.int32, device="cuda").view(seqs, -1)
    q = randn(3, seqs * new, 32, 128, dtype=torch.bfloat16)

    def time():
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = math.inf
        for _ in range(6):
            a.record()
            cache.attention(q, table, ints([kept] * seqs), max_new=new, max_kept=kept)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    clean = time()
    for b in range(seqs):                # a head's first segment in each block or so
        cache.v_params[int(table[b, 3]), 0, 5, 0] = math.nan
    assert time() <= 2.0 * clean


@pytest.mark.parametrize("tokens", [0, 7])
def test_the_gradient_of_no_key_heads_is_zero(K, tokens):
    """Every output of the call is written, the weights' gradients of heads that are not there too."""
    q, g = randn(1, tokens, 2, 64), randn(2, tokens, 2, 64)
    none = torch.empty((tokens, 0, 64), device="cuda")
    w = torch.ones(64, device="cuda")
    pos, freq = torch.arange(tokens, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    marks = [torch.full((64,), 7.0, device="cuda") for _ in range(64)]      # what the allocator hands out again
    torch.cuda.synchronize()
    del marks
    dq, dk, dwq, dwk = K.qk_norm_rope_backward(g, none, q, none, w, w, pos, freq)
    assert dk.shape == none.shape and torch.equal(dwk, torch.zeros_like(w))
    both = K.qk_norm_rope_backward(g, g, q, q, w, w, pos, freq)
    assert torch.equal(dq, both[0]) and torch.equal(dwq, both[2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [256, 20])
@pytest.mark.parametrize("new", [1, 40])
def test_contexts_up_to_the_last_length(kv4, dtype, page, new):
    """Places of tokens near 2^31, through a table that repeats its pages; longer contexts are cut to the longest and reported."""
    cache = kv4.Kv4Cache.allocate(8, page, 2, 128, 64)
    n = 8 * page
    cache.append(randn(1, n, 2, 128), randn(2, n, 2, 128), torch.arange(n, device="cuda"))
    longest = 2 ** 31 - 4097
    table = (torch.arange(-(-2 ** 31 // page), dtype=torch.int32, device="cuda") % 8)[None]
    q = randn(3, new, 4, 128, dtype=dtype)
    for kept, told in ((longest, False), (longest - 9, False), (longest + 1, True), (2 ** 31 - 1, True)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = cache.attention(q, table, ints([kept]), max_new=new, window=100, status=status)
        assert int(status) == (kv4.STATUS_BAD_INDEX if told else 0)
        # the same rows in a context of as many periods as a window needs
        short = min(kept, longest) % (16 * n) + 16 * n
        r = B.attention(cache, q, table, [short], [0, new], window=100)
        B.check(out, r, context=kept)


def test_a_cache_follows_its_tensors(kv4):
    """A tensor's storage may move; its old place is not written any more."""
    cache = kv4.Kv4Cache.allocate(2, 16, 2, 64, 32)
    assert (cache.num_pages, cache.page_size, cache.kv_heads, cache.head_dim, cache.group) == (2, 16, 2, 64, 32)
    k, v, slots = randn(1, 5, 2, 64), randn(2, 5, 2, 64), torch.arange(5, device="cuda")
    old = [t.data.clone() for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)]
    held = []
    for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params):
        held.append(t.detach())
        t.data = t.data.clone()
    cache.append(k, v, slots)
    assert all(torch.equal(a, b) for a, b in zip(held, old))
    fresh = kv4.Kv4Cache.allocate(2, 16, 2, 64, 32)
    fresh.append(k, v, slots)
    assert torch.equal(cache.k_codes, fresh.k_codes) and torch.equal(cache.v_params, fresh.v_params)
    assert all(torch.equal(a, b) for a, b in zip(cache.gather(slots), fresh.gather(slots)))


def test_a_cache_tells_what_its_calls_skipped(kv4):
    """Without a status word of the call, reports go to the cache's own; with one, to that alone; a captured call reports at replay."""
    cache = kv4.Kv4Cache.allocate(4, 16, 2, 64, 32)
    k, v = randn(1, 2, 2, 64), randn(2, 2, 2, 64)
    q, table = randn(3, 2, 4, 64, dtype=torch.bfloat16), ints([[0, 1]])
    good, bad = ints([0, 1]), ints([0, 64])
    cache.append(k, v, good)
    cache.gather(good)
    cache.attention(q, table, ints([2]))
    cache.check()
    for call in (lambda **kw: cache.append(k, v, bad, **kw), lambda **kw: cache.gather(bad, **kw), lambda **kw: cache.attention(q, table, ints([33]), **kw),
                 lambda **kw: cache.attention(q, ints([[4, 1]]), ints([2]), **kw)):
        own = ints([0])
        call(status=own)
        cache.check()
        assert int(own) == kv4.STATUS_BAD_INDEX
        call()
        with pytest.raises(RuntimeError, match="outside its tensor"):
            cache.check()
        cache.check()
    slots = good.clone()
    cache.append(k, v, slots)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.append(k, v, slots)
    slots.copy_(bad)
    g.replay()
    with pytest.raises(RuntimeError, match="outside its tensor"):
        cache.check()
    plain = kv4.Kv4Cache(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)
    plain.append(k, v, bad)
    with pytest.raises(ValueError, match="without a status word"):
        plain.check()
    with pytest.raises(ValueError, match="one int32"):
        kv4.Kv4Cache(cache.k_codes, cache.k_params, cache.v_codes, cache.v_params, status=ints([0, 0]))


# ------------------------------------------------------------------------------------------- bounds that tell types apart

@pytest.mark.parametrize("dtype, norm", [(torch.float16, 3.3e-4), (torch.bfloat16, 2.1e-3)])
@pytest.mark.parametrize("dim, group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("new, kept, window", [([1, 1], [1500, 77], 0), ([5, 2], [700, 33], 0), ([60, 200], [900, 200], 0), ([70, 130], [333, 600], 64)])
def test_errors_are_those_of_the_type(kv4, dtype, norm, dim, group, new, kept, window):
    """The 2-norm of the error against 64 bits.  An output's own rounding is uniform within half a step, whose size relative to the value
    varies over a binade: 2^-11 (2^-8) / 3^1/2 times 0.74 is 2.1e-4 (1.7e-3).  Weights rounded to halves (and, for bf16 in the many-row
    kernel, keys and values) add 1.2e-4 to 2.1e-4 each before averaging over tokens; one half per operand for half inputs would make the sum
    3.8e-4."""
    pages = [-(-n // 16) for n in kept]
    cache = kv4.Kv4Cache.allocate(sum(pages), 16, 2, dim, group)
    loud = 1.0 + 2.0 * (torch.arange(dim, device="cuda") % 23 == 5)
    rows = sum(pages) * 16
    cache.append(randn(1, rows, 2, dim) * loud, randn(2, rows, 2, dim), torch.arange(rows, device="cuda"))
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(4)).to(torch.int32)
    table = torch.full((2, max(pages)), -1, dtype=torch.int32)
    table[0, :pages[0]], table[1, :pages[1]] = order[:pages[0]], order[pages[0]:]
    table, starts = table.cuda(), [0, new[0], sum(new)]
    q = randn(3, starts[-1], 8, dim, dtype=dtype)
    out = cache.attention(q, table, ints(kept), q_starts=ints(starts), max_new=max(new), max_kept=max(kept), window=window)
    B.check(out, B.attention(cache, q, table, kept, starts, window=window), norm=norm, context=(dim, group, new))


@pytest.mark.parametrize("dim, group", [(64, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("new", [1, 6, 60])
def test_small_steps_on_a_large_common_value(kv4, dim, group, new):
    """Half inputs: what is left of a value beside its first half is as large as the differences between tokens, for keys as for values."""
    n = 300
    cache = kv4.Kv4Cache.allocate(19, 16, 2, dim, group)
    # lo near 1, 15 steps of 2^-12 each: a half near 1 resolves 2^-10
    base = 1.0 + torch.randint(0, 16, (n, 2, dim), generator=torch.Generator().manual_seed(1)).cuda() * 2.0 ** -12
    base[..., 0::group], base[..., 1::group] = 1.0, 1.0 + 15 * 2.0 ** -12
    cache.append(base.float(), base.flip(0).float(), torch.arange(n, device="cuda"))
    q = randn(3, new, 4, dim, dtype=torch.float16)
    q -= q.float().mean(-1, keepdim=True).half()          # scores of the common value are small, their differences count
    scale = 300.0 / dim ** 0.5
    table = torch.arange(19, dtype=torch.int32, device="cuda")[None]
    out = cache.attention(q, table, ints([n]), max_new=new, scale=scale)
    r = B.attention(cache, q, table, [n], [0, new], scale=scale)
    # keys off by 2^-21 where they are two halves, fp32 sums of 16 products at a time: 2^-19 of the sum of magnitudes in all
    B.check(out, r, score=r["dots"] * 2.0 ** -19, context=(dim, group, new))


@pytest.mark.parametrize("value", [-math.inf, math.inf, math.nan, -70000.0, 70000.0, -65520.0, 65520.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_group_of_one_value_that_is_no_half_is_stored_as_nan(kv4, dtype, value):
    cache = kv4.Kv4Cache.allocate(1, 16, 1, 128, 64)
    x = randn(1, 3, 1, 128, dtype=dtype)
    x[1, 0, 64:] = value
    cache.append(x, x, ints([0, 1, 2]))
    for y in cache.gather(ints([0, 1, 2]), torch.float32):
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[1, 0, 64:] = True
        assert torch.equal(torch.isnan(y), bad) and torch.isfinite(y[~bad]).all()
