"""A paged key/value cache held in 4 bits, attention over it, and the rotary frequencies of a decoder.

A decoder layer's step between its QKV linear and its output linear, on columns of the QKV linear's output:

    inv_freq, mscale = kv4.rope_frequencies(128, device="cuda")
    cache = kv4.Kv4Cache.allocate(num_pages, 64, kv_heads, 128)
    q = kernels.rope(q, positions, inv_freq, mscale=mscale)        # or kernels.qk_norm_rope
    cache.append(k, v, slots, positions=positions, inv_freq=inv_freq, mscale=mscale)
    out = cache.attention(q, block_table, kept, max_new=1, max_kept=8192)

Every method is one call into the C-ABI (layer 2 of include/itexb200.h, where the row format is defined) on torch's current
stream; none of them synchronises (but check), and all may be captured into a CUDA graph.  Kernels report indexes outside the
cache, and waits that expired, through a device int32 `status` instead of following them: the call's, else the cache's own, which
Kv4Cache.check reads.
"""
import math

import torch

from . import _lib as L
from . import kernels as K

STATUS_BAD_INDEX = L.STATUS_BAD_INDEX
STATUS_WAIT_EXPIRED = L.STATUS_WAIT_EXPIRED


def rope_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, trained=8192, fast=32.0, slow=1.0, device="cuda"):
    """-> (inv_freq, mscale): radians per position for each of the rotary_dim / 2 pairs (float64 on `device`) and the factor on
    cos and sin, for kernels.rope, kernels.qk_norm_rope and Kv4Cache.append.  scaling stretches a model trained on `trained`
    positions to `factor` times as many:
      None        base ** (-2 i / rotary_dim)
      "linear"    all frequencies divided by factor
      "base"      base raised so that the slowest pair is divided by factor, the fastest kept
      "by_parts"  pairs that turn fewer than `slow` times over `trained` positions divided by factor, those that turn more
                  than `fast` times kept, a linear ramp over the pair's index between (its ends on whole indexes, the upper one
                  behind the last pair where that turns more than `slow` times); mscale = 0.1 ln(factor) + 1
      "by_length" the same two ends with the ramp linear in the number of turns; mscale = 1"""
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError("rotary_dim must be even and positive, got %r" % (rotary_dim,))
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1, got %r and %r" % (base, factor))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rotary_dim)
    mscale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "base":
        if rotary_dim < 4:
            raise ValueError("scaling='base' needs more than one pair")
        f = (base * factor ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim)
    elif scaling in ("by_parts", "by_length"):
        if not fast > slow > 0.0 or trained <= 0:
            raise ValueError("fast > slow > 0 and trained > 0 are needed, got %r, %r, %r" % (fast, slow, trained))
        if scaling == "by_parts":
            at = [rotary_dim * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base)) for turns in (fast, slow)]
            low, high = max(0.0, math.floor(at[0])), min(rotary_dim - 1.0, math.ceil(at[1]))
            stretch = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
            mscale = 0.1 * math.log(factor) + 1.0
        else:
            stretch = ((fast - trained * f / (2.0 * math.pi)) / (fast - slow)).clamp(0.0, 1.0)
        f = f * (1.0 - stretch) + f / factor * stretch
    elif scaling is not None:
        raise ValueError("unknown scaling %r" % (scaling,))
    return f.to(device), mscale


class Kv4Cache:
    """The cache's four tensors: codes uint8 [pages, kv_heads, page_size, head_dim / 2] and params float16
    [pages, kv_heads, page_size, head_dim / group, 2], for keys and for values.  The first three dimensions may have any
    strides (a token-major cache is passed as its transpose(1, 2)); keys and values share them.  The object holds no state
    besides the tensors, which are its own for good (k_codes, k_params, v_codes, v_params; read-only attributes, as are the sizes and status):
    which page belongs to which sequence is the caller's block table.  status: one int32 (zero) on the same device for what calls
    without a status word of their own report; without it (a cache that allocate did not make) such calls skip in silence."""

    def __init__(self, k_codes, k_params, v_codes, v_params, status=None):
        self.dev = K.device_of(k_codes, k_params, v_codes, v_params, status)
        if status is not None:
            _status(status)
        self._own = status
        cs, ps, ct, pt = k_codes.shape, k_params.shape, k_codes.stride(), k_params.stride()
        if len(cs) != 4 or len(ps) != 5 or k_codes.dtype != torch.uint8 or k_params.dtype != torch.float16:
            raise ValueError("codes must be uint8 [pages, kv_heads, page_size, head_dim / 2] and params float16 [.., head_dim / group, 2]")
        if v_codes.shape != cs or v_codes.stride() != ct or v_codes.dtype != torch.uint8 or v_params.shape != ps or v_params.stride() != pt \
                or v_params.dtype != torch.float16:
            raise ValueError("keys and values must agree in shapes, strides and types")
        pages, heads, page_size, row = cs
        groups = ps[3]
        if ps[:3] != cs[:3] or ps[4] != 2 or groups < 1 or ct[3] != 1 or pt[4] != 1 or (groups > 1 and pt[3] != 2) or (pt[0] | pt[1] | pt[2]) & 1 \
                or 2 * row % groups != 0:
            raise ValueError("codes %s and params %s do not describe one cache with dense rows" % (tuple(cs), tuple(ps)))
        self._tensors = (k_codes, k_params, v_codes, v_params)
        self._sizes = (pages, page_size, heads, 2 * row, 2 * row // groups, 0)
        self._strides = (ct[0], ct[1], ct[2], pt[0] // 2, pt[1] // 2, pt[2] // 2)

    k_codes, k_params, v_codes, v_params = (property(lambda self, i=i: self._tensors[i]) for i in range(4))
    status = property(lambda self: self._own)
    num_pages, page_size, kv_heads, head_dim, group = (property(lambda self, i=i: self._sizes[i]) for i in range(5))

    def _cache(self):
        """The C struct's fields.  Addresses are those of now: a tensor's storage may be replaced, its sizes and strides may not."""
        kc, kp, vc, vp = self._tensors
        return (*self._sizes, kc.data_ptr(), kp.data_ptr(), vc.data_ptr(), vp.data_ptr(), *self._strides)

    @classmethod
    def allocate(cls, num_pages, page_size, kv_heads, head_dim, group=64, device="cuda", token_major=False):
        """An empty cache; token_major lays a page out token by token instead of head by head."""
        dims = (num_pages, page_size, kv_heads) if token_major else (num_pages, kv_heads, page_size)
        made = []
        for _ in range(2):
            made.append(torch.zeros(dims + (head_dim // 2,), dtype=torch.uint8, device=device))
            made.append(torch.zeros(dims + (head_dim // group, 2), dtype=torch.float16, device=device))
        return cls(*[t.transpose(1, 2) if token_major else t for t in made], status=torch.zeros(1, dtype=torch.int32, device=device))

    def check(self):
        """Waits for the calls of torch's current stream and raises RuntimeError if one without a status word of its own has reported
        something since the last check; the first report is kept, and cleared here."""
        if self.status is None:
            raise ValueError("this cache was made without a status word")
        code = int(self.status)
        if code != 0:
            self.status.zero_()
            raise RuntimeError({STATUS_BAD_INDEX: "a slot, page, length or row offset outside its tensor was skipped",
                                STATUS_WAIT_EXPIRED: "a bounded wait ran out; the output is incomplete"}.get(code, "status %d" % code))

    def _kv(self, k, v, what):
        kp, vp = K._rows(k, "k"), K._rows(v, "v", k)
        n, heads, dim = k.shape
        if heads != self.kv_heads or dim != self.head_dim:
            raise ValueError("%s: rows %s for a cache of %d heads of %d" % (what, tuple(k.shape), self.kv_heads, self.head_dim))
        return n, kp, vp

    def append(self, k, v, slots, *, positions=None, inv_freq=None, interleaved=False, mscale=1.0, status=None):
        """Writes k, v [tokens, kv_heads, head_dim] (strided views are fine) into rows slots[t] = page * page_size + offset; -1
        skips a token; the other slots of a call must differ.  With positions and inv_freq the keys are rotated on the way."""
        K.device_of(self._tensors[0], k, v, slots, positions, inv_freq, status)
        if (positions is None) != (inv_freq is None):
            raise ValueError("positions and inv_freq go together")
        n, kp, vp = self._kv(k, v, "append")
        sp = K._vector(slots, "slots", K._INDEX_DT, n)
        pos = freq = pdt = rot = 0
        if positions is not None:
            pos, pdt = K._vector(positions, "positions", K._INDEX_DT, n), K._INDEX_DT[positions.dtype]
            freq, rot = K._vector(inv_freq, "inv_freq", K._FLOAT64), 2 * inv_freq.shape[0]
        K.launch(L.load().itexb_kv4_append, L.pack_kv4_append(*self._cache(), n, K._REAL_DT[k.dtype], K._INDEX_DT[slots.dtype], *kp, *vp, sp, pos, freq, pdt, rot,
                                                              int(interleaved), mscale, _status(status, self._own)), self.dev)

    def gather(self, slots, dtype=torch.bfloat16, *, out_k=None, out_v=None, status=None):
        """-> (k, v) [len(slots), kv_heads, head_dim]: the values that rows `slots` stand for, zeros for slot -1."""
        K.device_of(self._tensors[0], slots, out_k, out_v, status)
        sp = K._vector(slots, "slots", K._INDEX_DT)
        tokens = slots.shape[0]
        k = torch.empty((tokens, self.kv_heads, self.head_dim), dtype=dtype, device=slots.device) if out_k is None else out_k
        v = torch.empty_like(k) if out_v is None else out_v
        n, kp, vp = self._kv(k, v, "gather")
        if n != tokens:
            raise ValueError("gather: %d rows for %d slots" % (n, tokens))
        K.launch(L.load().itexb_kv4_gather, L.pack_kv4_gather(*self._cache(), n, K._REAL_DT[k.dtype], K._INDEX_DT[slots.dtype], *kp, *vp, sp, _status(status, self._own)),
                 self.dev)
        return k, v

    def attention(self, q, block_table, kept, *, q_starts=None, max_new=None, max_kept=None, causal=True, window=0, scale=None, out=None,
                  status=None, workspace=None):
        """Attention of the new tokens q [rows, q_heads, head_dim] over the cache (itexb_kv4_attention): block_table int32
        [sequences, pages each], kept int32 [sequences] = rows of each sequence in the cache, the new tokens' included.
        q_starts int32 [sequences + 1] gives each sequence's rows of q; without it every sequence has max_new rows.  max_new and
        max_kept are upper bounds of a sequence's new and kept tokens (by default as many as q and the table can hold); a tight
        bound saves work.  -> out, whose rows behind the last sequence stay as they were (uninitialised without `out`).
        workspace: a dense uint8 tensor to use instead of a fresh one, at least as large as a refusal asks for; calls that may
        run at the same time need different ones."""
        K.device_of(self._tensors[0], q, block_table, kept, q_starts, out, status, workspace)
        qp = K._rows(q, "q")
        kp = K._vector(kept, "kept", _INT32)
        seqs = kept.shape[0]
        rows, heads, dim = q.shape
        if dim != self.head_dim or heads % self.kv_heads != 0:
            raise ValueError("q %s for a cache of %d heads of %d" % (tuple(q.shape), self.kv_heads, self.head_dim))
        ts, tst = block_table.shape, block_table.stride()
        if len(ts) != 2 or block_table.dtype != torch.int32 or ts[0] != seqs or (tst[1] != 1 and ts[1] > 1):
            raise ValueError("block_table must be int32 [sequences, pages] with dense rows, got %s %s" % (block_table.dtype, tuple(ts)))
        cols = ts[1]
        sp = 0
        if q_starts is not None:
            sp = K._vector(q_starts, "q_starts", _INT32, seqs + 1)
            max_new = rows if max_new is None else max_new
        else:
            max_new = rows // max(1, seqs) if max_new is None else max_new
            if max_new * seqs > rows:
                raise ValueError("%d sequences of %d new tokens, but q has %d rows" % (seqs, max_new, rows))
        max_kept = min(cols * self.page_size, (1 << 31) - 1) if max_kept is None else max_kept
        if out is None:
            out = torch.empty_like(q)
            op = K._rows(out, "out")
        else:
            op = K._rows(out, "out", q)
        args = (*self._cache(), K._REAL_DT[q.dtype], seqs, heads, int(causal), window, max_new, max_kept, dim ** -0.5 if scale is None else scale,
                rows, *qp, *op, block_table.data_ptr(), tst[0], cols, kp, sp, _status(status, self._own))
        lib = L.load()
        if workspace is None:
            need = lib.itexb_kv4_attention_workspace_bytes(L.pack_kv4_attention(*args, 0, 0))
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be a dense uint8 tensor")
        K.launch(lib.itexb_kv4_attention, L.pack_kv4_attention(*args, workspace.data_ptr(), workspace.numel()), self.dev)
        return out


_INT32 = {torch.int32: 0}


def _status(t, own=None):
    t = own if t is None else t
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.numel() != 1:
        raise ValueError("status must be one int32")
    return t.data_ptr()
