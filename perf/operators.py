"""Measured cases of the decoder operators: rotary positions, per-head norms with the rotation, the 4-bit paged
key/value cache (append and read back) and attention over it.

`run` computes a case with plain torch operations (own = False) or with the calls a user makes of this library
(own = True, `kernels.py` and `kv4.py`).  Cache format, shared by every function here: a page holds `page` tokens of every
key/value head; a row is one token of one head, head_dim 4-bit codes (element 2i in the low, 2i + 1 in the high nibble of
byte i) and, for each `group` of consecutive elements, a half-precision pair (lo, step); the element is lo + step * code."""
import importlib
import importlib.util
import math
import os
import sys

import torch

own = False

_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    """The package directory has hyphens in its name: it is imported by path as `itex_b200`."""
    if "itex_b200" not in sys.modules:
        at = os.path.join(_ROOT, "intel-extension-for-tensorflow_b200")
        spec = importlib.util.spec_from_file_location("itex_b200", os.path.join(at, "__init__.py"), submodule_search_locations=[at])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["itex_b200"] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module("itex_b200.kernels"), importlib.import_module("itex_b200.kv4")


# ---------------------------------------------------------------------------------------------------------- cases

def _rope(name, tokens, q_heads, kv_heads, dim, rot, kind, interleaved=False, inverse=False, far=0, scaling="none"):
    return {"name": name, "op": "rope", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "type": kind,
            "interleaved": interleaved, "inverse": inverse, "far": far, "scaling": scaling}


def _norm(name, op, tokens, q_heads, kv_heads, dim, rot, kind, interleaved=False, far=0):
    return {"name": name, "op": op, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "type": kind,
            "interleaved": interleaved, "far": far}


def _store(name, tokens, kv_heads, dim, group, page, kind, interleaved=False, far=0, padded=0):
    return {"name": name, "op": "store", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "group": group, "page": page, "type": kind,
            "interleaved": interleaved, "far": far, "padded": padded}


def _attend(name, seqs, queries, context, q_heads, kv_heads, dim, group, page, kind, ragged=0.0, window=0, causal=True, idle=False):
    return {"name": name, "op": "attend", "seqs": seqs, "queries": queries, "context": context, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "group": group, "page": page, "type": kind, "ragged": ragged, "window": window, "causal": causal, "idle": idle}


def listed():
    return [
        # one decoding step of a batch of 64: the call is all latency
        _rope("rope-step", 64, 32, 8, 128, 128, "bf16", far=6000),
        # a long prompt far into a stretched context, interleaved pairs, half of the head rotated
        _rope("rope-stretched", 16384, 32, 8, 128, 64, "fp16", interleaved=True, far=1000000, scaling="by_parts"),
        # a prompt through the norms of its queries and keys and the rotation
        _norm("norm-rope-prompt", "norm_rope", 8192, 32, 8, 128, 128, "bf16", far=32000),
        # the gradient of the same in a training step over odd token counts, 16 heads of 64 on each side
        _norm("norm-rope-grad", "norm_rope_grad", 6143, 16, 16, 64, 64, "bf16"),
        # a decoding step's new keys and values into the cache, and back out
        _store("store-step", 96, 8, 128, 64, 16, "bf16", far=6000, padded=3),
        # a long prompt's keys and values into the cache, and back out (a prefix that is shared is read like this)
        _store("store-prompt", 16384, 8, 128, 64, 64, "bf16", far=32000),
        # a small interactive batch: short contexts, one of the batch's places idle
        _attend("attend-few", 5, 1, 700, 32, 8, 128, 64, 16, "bf16", ragged=0.8, idle=True),
        # a full serving batch, contexts of all lengths: the cache's bytes bound it
        _attend("attend-batch", 64, 1, 8192, 32, 8, 128, 64, 64, "bf16", ragged=0.6, idle=True),
        # one document of 128 Ki tokens: the work of one row is split over the whole GPU
        _attend("attend-long", 1, 1, 131072, 32, 8, 128, 128, 64, "bf16"),
        # five drafted tokens each to be verified, 16 heads of 64 that share nothing
        _attend("attend-verify", 24, 5, 3000, 16, 16, 64, 32, 16, "fp16", ragged=0.5),
        # the last chunk of a long prompt
        _attend("attend-chunk", 1, 2048, 10240, 32, 8, 128, 64, 64, "bf16"),
        # ragged prompts from their first token on, with a sliding window
        _attend("attend-prompts", 6, 1900, 1900, 32, 8, 128, 128, 32, "fp16", ragged=0.7, window=1024),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "norm_rope", "norm_rope_grad", "store", "attend", "attend", "attend"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op in ("rope", "norm_rope", "norm_rope_grad"):
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        kv = rng.choice([1, 2, 4, 8])
        q_heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        tokens = _log(rng, 1, max(2, min(16384, 16384 * 40 * 128 // ((q_heads + kv) * dim * (2 if op == "norm_rope_grad" else 1)))))
        far = rng.choice([0, 1000, 100000, 1000000])
        if op == "rope":
            c = _rope("", tokens, q_heads, kv, dim, rot, kind, rng.random() < 0.5, rng.random() < 0.3, far, rng.choice(["none", "linear", "by_parts"]))
        else:
            c = _norm("", op, tokens, q_heads, kv, dim, rot, kind, rng.random() < 0.5, far)
    elif op == "store":
        dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 3, 8, 16])
        tokens = _log(rng, 1, min(16384, 16384 * 8 * 128 // (kv * dim)))
        c = _store("", tokens, kv, dim, rng.choice([g for g in (32, 64, 128) if g <= dim]), rng.choice([16, 20, 32, 64, 128]),
                   rng.choice(["bf16", "fp16"]), rng.random() < 0.5, rng.choice([0, 10000, 300000]), rng.choice([0, 0, 5]))
    else:
        dim = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        q_heads = kv * rng.choice([1, 2, 3, 4, 5, 8, 16])
        queries = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 16, 2048)])
        seqs = _log(rng, 1, 64)
        most = min(131072, 64 * 8192 * 8 * 128 // (seqs * kv * dim), 2048 * 10240 * 32 * 128 // (seqs * queries * q_heads * dim))
        queries = min(queries, most)
        context = _log(rng, queries, max(queries + 1, most))
        window = rng.choice([0, 0, 0, _log(rng, 1, 2 * context)])
        c = _attend("", seqs, queries, context, q_heads, kv, dim, rng.choice([g for g in (32, 64, 128) if g <= dim]),
                    rng.choice([16, 20, 32, 64, 128]), rng.choice(["bf16", "fp16"]), rng.choice([0.0, 0.5, 0.9]), window, rng.random() < 0.85,
                    seqs > 1 and rng.random() < 0.3)
    del c["name"]
    return c


def _lengths(c):
    """(new tokens, tokens in the cache) of each sequence: the case alone says them."""
    new, kept = [], []
    for b in range(c["seqs"]):
        less = 1.0 - c["ragged"] * math.modf((b + 1) * 0.7548776662466927)[0]
        n = max(1, int(round(c["queries"] * less)))
        kept.append(max(n, int(round(c["context"] * less))))
        new.append(n)
    if c["idle"]:
        new[-1], kept[-1] = 1, 0
    return new, kept


def _visible(c):
    """(query, key) pairs that the masks leave, and cache rows that some query sees, over all sequences."""
    pairs = rows = 0
    for n, kept in zip(*_lengths(c)):
        first = None
        for i in range(n):
            last = kept - n + i if c["causal"] else kept - 1
            low = max(0, kept - n + i - c["window"] + 1) if c["window"] else 0
            if last >= low:
                pairs += last - low + 1
                first = low if first is None else min(first, low)
        rows += 0 if first is None else kept - first
    return pairs, rows


def work(c):
    if c["op"] == "attend":
        pairs, rows = _visible(c)
        q = 2 * sum(_lengths(c)[0]) * c["q_heads"] * c["dim"] * 2
        row = 2 * (c["dim"] // 2 + 4 * (c["dim"] // c["group"]))
        return {"bytes": q + rows * c["kv_heads"] * row, "flops": 4.0 * pairs * c["q_heads"] * c["dim"]}
    size = torch.empty(0, dtype=_T[c["type"]]).element_size()
    if c["op"] == "store":
        n = c["tokens"] * c["kv_heads"]
        row = c["dim"] // 2 + 4 * (c["dim"] // c["group"])
        # in: keys and values; the cache's rows written and read; out: keys and values
        return {"bytes": 2 * n * (c["dim"] * size * 2 + 2 * row) + 16 * c["tokens"], "flops": 16.0 * n * c["dim"]}
    n = c["tokens"] * (c["q_heads"] + c["kv_heads"]) * c["dim"]
    if c["op"] == "norm_rope_grad":
        return {"bytes": 3 * n * size + 8 * c["tokens"], "flops": 16.0 * n}
    return {"bytes": 2 * n * size + 8 * c["tokens"], "flops": (3.0 if c["op"] == "rope" else 7.0) * n}


# --------------------------------------------------------------------------------------------------------- inputs

def _frequencies(rot, scaling):
    """Radians a position, in 64 bits on the host (what kv4.rope_frequencies returns), and the factor on cos and sin."""
    pairs = torch.arange(rot // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * pairs / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "by_parts":
        # slow pairs (less than one turn over the trained length) are stretched 32 times, fast ones (over 32 turns) kept
        at = [rot * math.log(8192.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(10000.0)) for turns in (32.0, 1.0)]
        low, high = max(0.0, math.floor(at[0])), min(rot / 2.0 - 1.0, math.ceil(at[1]))
        stretch = ((pairs - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return f * (1.0 - stretch) + f / 32.0 * stretch, 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def _quantised(x, group):
    """fp32 rows [..., dim] -> (codes uint8 [..., dim / 2], params fp16 [..., dim / group, 2])."""
    g = x.unflatten(-1, (-1, group))
    lo = g.amin(-1).half()
    span = g.amax(-1) - lo.float()
    step = (span / torch.full_like(span, 15.0)).clamp_min(0.0).half()     # a tensor: by a number torch multiplies with its inverse
    inv = torch.where(step > 0, 1.0 / step.float(), torch.zeros((), device=x.device))
    codes = ((g - lo.float()[..., None]) * inv[..., None]).round().clamp(0.0, 15.0).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack([lo, step], -1)


def _values(codes, params):
    """The fp32 values that rows of the cache stand for."""
    v = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = params.float()
    return (v.unflatten(-1, (p.shape[-2], -1)) * p[..., 1:] + p[..., :1]).flatten(-2)


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, kind=_T[c["type"]]):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(kind)

    s = {"case": c}
    if c["op"] == "attend":
        new, kept = _lengths(c)
        page, heads, dim = c["page"], c["kv_heads"], c["dim"]
        pages = [-(-n // page) for n in kept]
        total, most = sum(pages) + 3, max(max(pages), 1)
        order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((c["seqs"], most), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
            at += n
        table = table.cuda()
        s["table"] = torch.where(table >= 0, order[table.clamp_min(0).long()], table)
        # keys have a few channels that stand out, values have none
        loud = 1.0 + 2.0 * (torch.arange(dim, device="cuda") % 23 == 5)
        for name, gain in (("k", loud), ("v", torch.ones(dim, device="cuda"))):
            codes = torch.empty((total, heads, page, dim // 2), dtype=torch.uint8, device="cuda")
            params = torch.empty((total, heads, page, dim // c["group"], 2), dtype=torch.float16, device="cuda")
            step = max(1, (1 << 27) // (heads * page * dim))
            for i in range(0, total, step):
                n = min(step, total - i)
                codes[i:i + n], params[i:i + n] = _quantised(normal(n, heads, page, dim, kind=torch.float32) * gain, c["group"])
            s[name + "_codes"], s[name + "_params"] = codes, params
        s["q"] = normal(sum(new), c["q_heads"], dim)
        s["kept"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
        s["starts"] = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        s["most_new"], s["most_kept"] = max(new), max(kept)
        return s
    tokens = c["tokens"]
    s["positions"] = (torch.arange(tokens, device="cuda") + int(torch.randint(0, c["far"] + 1, (1,), generator=gen, device="cuda"))).to(torch.int64)
    if c["op"] == "store":
        page, heads, dim = c["page"], c["kv_heads"], c["dim"]
        total = -(-tokens // page) + 4
        s["k_codes"] = torch.zeros((total, heads, page, dim // 2), dtype=torch.uint8, device="cuda")
        s["k_params"] = torch.zeros((total, heads, page, dim // c["group"], 2), dtype=torch.float16, device="cuda")
        s["v_codes"], s["v_params"] = torch.zeros_like(s["k_codes"]), torch.zeros_like(s["k_params"])
        order = torch.randperm(total, generator=gen, device="cuda")
        t = torch.arange(tokens, device="cuda") + page // 2
        s["slots"] = order[t // page] * page + t % page
        if c["padded"]:
            s["slots"][max(1, tokens - c["padded"]):] = -1       # rows behind the last sequence of a padded batch
        # keys and values are columns of one projection's output
        qkv = normal(tokens, 4 * heads * dim)
        s["k"] = qkv[:, 2 * heads * dim:3 * heads * dim].unflatten(1, (heads, dim))
        s["v"] = qkv[:, 3 * heads * dim:].unflatten(1, (heads, dim))
        s["freq"] = _frequencies(dim, "none")[0].cuda()
        return s
    qkv = normal(tokens, (c["q_heads"] + 2 * c["kv_heads"]) * c["dim"])
    nq, nk = c["q_heads"] * c["dim"], c["kv_heads"] * c["dim"]
    s["q"] = qkv[:, :nq].unflatten(1, (c["q_heads"], c["dim"]))
    s["k"] = qkv[:, nq:nq + nk].unflatten(1, (c["kv_heads"], c["dim"]))
    freq, s["mscale"] = _frequencies(c["rot"], c.get("scaling", "none"))
    s["freq"] = freq.cuda()
    if c["op"] != "rope":
        s["wq"], s["wk"] = ((1.0 + 0.1 * normal(c["dim"], kind=torch.float32)).to(_T[c["type"]]) for _ in range(2))
    if c["op"] == "norm_rope_grad":
        s["gq"], s["gk"] = normal(tokens, c["q_heads"], c["dim"]), normal(tokens, c["kv_heads"], c["dim"])
    return s


# ----------------------------------------------------------------------------------------------------- plain forms

def _turned(x, cos, sin, interleaved):
    """fp32 rows [tokens, heads, dim] with their first 2 * cos.shape[-1] elements rotated."""
    h = cos.shape[-1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., 2 * h:]], -1)
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _cos_sin(s):
    angle = s["positions"].double()[:, None] * s["freq"][None, :]
    m = s.get("mscale", 1.0)
    return (angle.cos() * m).float(), (angle.sin() * m).float()


_EPS = 1e-6


def _plain_rope(s):
    c = s["case"]
    cos, sin = _cos_sin(s)
    if c["inverse"]:
        sin = -sin
    return [_turned(x.float(), cos, sin, c["interleaved"]).to(x.dtype) for x in (s["q"], s["k"])]


def _plain_norm_rope(s):
    cos, sin = _cos_sin(s)
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        f = x.float()
        f = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + _EPS) * w.float()
        out.append(_turned(f, cos, sin, s["case"]["interleaved"]).to(x.dtype))
    return out


def _plain_norm_rope_grad(s):
    cos, sin = _cos_sin(s)
    dx, dw = [], []
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        f = x.float()
        r = torch.rsqrt(f.square().mean(-1, keepdim=True) + _EPS)
        hat = f * r
        t = _turned(g.float(), cos, -sin, s["case"]["interleaved"])       # the rotation's transpose
        dw.append((t * hat).sum((0, 1), dtype=torch.float64).to(w.dtype))
        u = t * w.float()
        dx.append((r * (u - hat * (u * hat).mean(-1, keepdim=True))).to(x.dtype))
    return dx + dw


def _plain_store(s):
    c = s["case"]
    cos, sin = _cos_sin(s)
    page = c["page"]
    here = s["slots"] >= 0
    slots = torch.where(here, s["slots"], 0)
    at, off = slots // page, slots % page
    out = []
    for name, x in (("k", _turned(s["k"].float(), cos, sin, c["interleaved"])), ("v", s["v"].float())):
        codes, params = _quantised(x, c["group"])
        pool_c, pool_p = s[name + "_codes"], s[name + "_params"]
        pool_c[at[here], :, off[here]] = codes[here]
        pool_p[at[here], :, off[here]] = params[here]
        back = _values(pool_c[at, :, off], pool_p[at, :, off])
        out.append(torch.where(here[:, None, None], back, 0.0).to(s[name].dtype))
    return out


def _plain_attend(s):
    c = s["case"]
    group, dim, kv = c["q_heads"] // c["kv_heads"], c["dim"], c["kv_heads"]
    starts, kept = s["starts"].long(), s["kept"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["most_new"], device="cuda")
    at = (starts[:-1, None] + i).clamp_max(s["q"].shape[0] - 1)                     # [seqs, most_new]
    q = s["q"].float()[at].unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4)          # [seqs, kv, group, most_new, dim]
    j = torch.arange(max(1, s["most_kept"]), device="cuda")
    pages = s["table"].long().clamp_min(0)[:, j // c["page"]]                        # [seqs, most_kept]
    k = _values(s["k_codes"][pages, :, j % c["page"]], s["k_params"][pages, :, j % c["page"]])    # [seqs, most_kept, kv, dim]
    score = torch.matmul(q.flatten(2, 3), k.permute(0, 2, 3, 1)).unflatten(2, (group, -1)) * dim ** -0.5
    del k
    place = (kept - new)[:, None] + i                                                # of each query in its sequence
    seen = (j < kept[:, None])[:, None, :].expand(-1, i.numel(), -1)
    if c["causal"]:
        seen = seen & (j <= place[:, :, None])
    if c["window"]:
        seen = seen & (j > place[:, :, None] - c["window"])
    seen = seen[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    del score
    total = p.sum(-1, keepdim=True)
    v = _values(s["v_codes"][pages, :, j % c["page"]], s["v_params"][pages, :, j % c["page"]])
    out = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (group, -1))
    out = torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)                                   # [seqs, most_new, q_heads, dim]
    return out[i < new[:, None]].to(s["q"].dtype)


def run(s):
    c = s["case"]
    if not own:
        return {"rope": _plain_rope, "norm_rope": _plain_norm_rope, "norm_rope_grad": _plain_norm_rope_grad, "store": _plain_store,
                "attend": _plain_attend}[c["op"]](s)
    K, kv4 = _package()
    if c["op"] == "rope":
        return list(K.rope(s["q"], s["positions"], s["freq"], k=s["k"], interleaved=c["interleaved"], mscale=s["mscale"], inverse=c["inverse"]))
    if c["op"] == "norm_rope":
        return list(K.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["freq"], eps=_EPS, interleaved=c["interleaved"]))
    if c["op"] == "norm_rope_grad":
        return list(K.qk_norm_rope_backward(s["gq"], s["gk"], s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["freq"], eps=_EPS,
                                            interleaved=c["interleaved"]))
    cache = kv4.Kv4Cache(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"])
    if c["op"] == "store":
        cache.append(s["k"], s["v"], s["slots"], positions=s["positions"], inv_freq=s["freq"], interleaved=c["interleaved"])
        return list(cache.gather(s["slots"], s["k"].dtype))
    return cache.attention(s["q"], s["table"], s["kept"], q_starts=s["starts"], max_new=s["most_new"], max_kept=s["most_kept"],
                           causal=c["causal"], window=c["window"])


# ----------------------------------------------------------------------------------------------- 64 bits, on their own

def _exact_turn(x, s, sign=1.0):
    """Rows as complex numbers times mscale * exp(i * angle)."""
    c = s["case"]
    rot = 2 * s["freq"].numel()
    turn = torch.polar(torch.full_like(s["freq"], s.get("mscale", 1.0)).expand(s["positions"].numel(), -1),
                       sign * torch.outer(s["positions"].double(), s["freq"]))[:, None, :]
    y = x.clone()
    if c["interleaved"]:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * turn
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def _exact_rows(codes, params):
    n = codes.shape[-1]
    v = torch.empty(codes.shape[:-1] + (2 * n,), dtype=torch.float64, device=codes.device)
    v[..., 0::2], v[..., 1::2] = torch.remainder(codes, 16), torch.div(codes, 16, rounding_mode="floor")
    each = 2 * n // params.shape[-2]
    return v * params[..., 1].double().repeat_interleave(each, -1) + params[..., 0].double().repeat_interleave(each, -1)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        return [_exact_turn(s[n].double(), s, -1.0 if c["inverse"] else 1.0) for n in ("q", "k")]
    if c["op"] == "norm_rope":
        out = []
        for n in ("q", "k"):
            x = s[n].double()
            out.append(_exact_turn(x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + _EPS).sqrt() * s["w" + n].double(), s))
        return out
    if c["op"] == "norm_rope_grad":
        out = []
        for n in ("q", "k"):
            x, w = s[n].double().requires_grad_(), s["w" + n].double().requires_grad_()
            y = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + _EPS).sqrt() * w
            out.append(torch.autograd.grad(y, (x, w), _exact_turn(s["g" + n].double(), s, -1.0)))
        return [out[0][0], out[1][0], out[0][1], out[1][1]]
    if c["op"] == "store":
        out = []
        for n, x in (("k", _exact_turn(s["k"].double(), s)), ("v", s["v"].double())):
            x = x.unflatten(-1, (c["dim"] // c["group"], c["group"]))
            lo = x.min(-1, keepdim=True).values.half().double()
            step = torch.clamp((x.max(-1, keepdim=True).values - lo) / 15.0, min=0.0).half().double()
            code = torch.where(step > 0, torch.clamp(torch.round((x - lo) / torch.where(step > 0, step, 1.0)), 0.0, 15.0), 0.0)
            out.append(((lo + step * code).flatten(-2)) * (s["slots"] >= 0)[:, None, None])
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    share = c["q_heads"] // c["kv_heads"]
    at = 0
    for b, (n, kept) in enumerate(zip(*_lengths(c))):
        if kept:
            ids = s["table"][b, :-(-kept // c["page"])].long()
            seen = torch.ones((n, kept), dtype=torch.bool, device="cuda")
            if c["causal"]:
                seen = seen.tril(kept - n)
            if c["window"]:
                seen = seen.triu(kept - n - c["window"] + 1)
            some = seen.any(-1, keepdim=True)
            for h in range(c["kv_heads"]):
                k, v = (_exact_rows(s[m + "_codes"][ids, h].flatten(0, 1)[:kept], s[m + "_params"][ids, h].flatten(0, 1)[:kept]) for m in "kv")
                for g in range(h * share, (h + 1) * share):
                    a = (s["q"][at:at + n, g].double() @ k.T / math.sqrt(c["dim"])).masked_fill(~seen & some, -math.inf)
                    out[at:at + n, g] = (torch.softmax(a, -1) @ v) * some
        at += n
    return out
