"""CPU checks of the decoder operators' boundary: what the C-ABI and its Python face refuse, and the rotary frequencies."""
import ctypes as C
import importlib
import math

import pytest
import torch


@pytest.fixture(scope="module")
def mods(itex):
    return itex.load(), itex._lib, importlib.import_module("itex_b200.kernels"), importlib.import_module("itex_b200.kv4")


PTR = 1 << 20      # never followed: every case below is refused before a launch


def refused(lib, L, name, params, text, code=None):
    assert getattr(lib, "itexb_" + name)(C.byref(params) if params is not None else None, None) == (L.INVALID_ARGUMENT if code is None else code)
    assert text in lib.itexb_last_error().decode(), lib.itexb_last_error()


def rope_params(L, **kw):
    p = L.RopeParams(tokens=4, q_heads=2, k_heads=1, head_dim=64, rotary_dim=64, dtype=L.DT_BFLOAT16, positions_dtype=L.DT_INT64, mscale=1.0,
                     positions=PTR, inv_freq=PTR, q=PTR, q_token_stride=128, q_head_stride=64, k=PTR, k_token_stride=64, k_head_stride=64,
                     q_out=PTR, q_out_token_stride=128, q_out_head_stride=64, k_out=PTR, k_out_token_stride=64, k_out_head_stride=64)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change, text", [
    (dict(dtype=11), "unsupported type qint8"), (dict(positions_dtype=1), "positions must be int32 or int64"), (dict(tokens=-1), "bad shape"),
    (dict(q_heads=0), "bad shape"), (dict(k_heads=-1), "bad shape"), (dict(head_dim=63), "head_dim must be even"), (dict(head_dim=514), "head_dim must be even"),
    (dict(rotary_dim=66), "rotary_dim must be even"), (dict(rotary_dim=3), "rotary_dim must be even"), (dict(rotary_dim=-2), "rotary_dim must be even"),
    (dict(tokens=1 << 31), "2^31 rows"), (dict(q=0), "NULL tensor"), (dict(q_out=0), "NULL tensor"), (dict(k=0), "NULL tensor"),
    (dict(positions=0), "NULL positions"), (dict(inv_freq=0), "NULL positions")])
def test_rope_refuses(mods, change, text):
    lib, L, _, _ = mods
    refused(lib, L, "rope", rope_params(L, **change), text)
    n = L.QkNormRopeParams(rope_params(L, **change), PTR, PTR, L.DT_FLOAT, 1e-6)
    refused(lib, L, "qk_norm_rope", n, text)
    refused(lib, L, "qk_norm_rope_grad", L.QkNormRopeGradParams(n, PTR, 128, 64, PTR, 64, 64, PTR, PTR, PTR), text)


def test_norm_rope_refuses(mods):
    lib, L, _, _ = mods
    for name in ("rope", "qk_norm_rope", "qk_norm_rope_grad"):
        refused(lib, L, name, None, "NULL params")
    refused(lib, L, "qk_norm_rope", L.QkNormRopeParams(rope_params(L), PTR, PTR, L.DT_INT32, 1e-6), "unsupported weight type int32")
    refused(lib, L, "qk_norm_rope", L.QkNormRopeParams(rope_params(L, inverse=1), PTR, PTR, L.DT_HALF, 1e-6), "inverse does not apply")
    refused(lib, L, "qk_norm_rope", L.QkNormRopeParams(rope_params(L), PTR, PTR, L.DT_HALF, -1.0), "epsilon")
    refused(lib, L, "qk_norm_rope", L.QkNormRopeParams(rope_params(L), PTR, PTR, L.DT_HALF, math.nan), "epsilon")
    refused(lib, L, "qk_norm_rope", L.QkNormRopeParams(rope_params(L), PTR, 0, L.DT_HALF, 1e-6), "NULL weight")
    n = L.QkNormRopeParams(rope_params(L), PTR, PTR, L.DT_HALF, 1e-6)
    refused(lib, L, "qk_norm_rope_grad", L.QkNormRopeGradParams(n, PTR, 128, 64, PTR, 64, 64, PTR, 0, PTR), "NULL weight gradient")
    refused(lib, L, "qk_norm_rope_grad", L.QkNormRopeGradParams(n, PTR, 128, 64, 0, 64, 64, PTR, PTR, PTR), "NULL gradient or workspace")
    refused(lib, L, "qk_norm_rope_grad", L.QkNormRopeGradParams(n, PTR, 128, 64, PTR, 64, 64, PTR, PTR, 0), "NULL gradient or workspace")
    assert lib.itexb_rope(C.byref(rope_params(L, tokens=0, q=0, q_out=0)), None) == L.OK         # nothing to do, nothing launched
    assert lib.itexb_qk_norm_rope_grad_workspace_bytes(0, 8, 8, 64) == 0
    assert lib.itexb_qk_norm_rope_grad_workspace_bytes(3, 2, 1, 64) == 2 * 3 * 64 * 4


def cache_params(L, **kw):
    c = L.Kv4CacheParams(10, 16, 2, 128, 64, 0, PTR, PTR, PTR, PTR, 2 * 16 * 64, 16 * 64, 64, 2 * 16 * 2, 16 * 2, 2)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


CACHE = [
    (dict(num_pages=0), "bad cache shape"), (dict(page_size=0), "bad cache shape"), (dict(kv_heads=-1), "bad cache shape"),
    (dict(num_pages=1 << 20, page_size=1 << 11), "2^31 cache rows"), (dict(head_dim=96), "head_dim must be 64, 128 or 256, got 96"),
    (dict(group=48), "group must be"), (dict(group=128, head_dim=64), "group must be"), (dict(k_codes=0), "NULL cache tensor"), (dict(v_params=0), "NULL cache tensor"),
    (dict(k_codes=PTR + 8), "16-byte aligned"), (dict(codes_token_stride=72), "16-byte aligned"), (dict(v_params=PTR + 4), "aligned to 8 bytes"),
    (dict(params_head_stride=33), "aligned to 8 bytes"), (dict(group=32, params_token_stride=6), "aligned to 16 bytes")]


def append_params(L, cache=None, **kw):
    p = L.Kv4AppendParams(cache or cache_params(L), 4, L.DT_HALF, L.DT_INT64, PTR, 256, 128, PTR, 256, 128, PTR, PTR, PTR, L.DT_INT64, 128, 0, 1.0, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def gather_params(L, cache=None, **kw):
    p = L.Kv4GatherParams(cache or cache_params(L), 4, L.DT_HALF, L.DT_INT64, PTR, 256, 128, PTR, 256, 128, PTR, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def attention_params(L, cache=None, **kw):
    p = L.Kv4AttentionParams(cache or cache_params(L), L.DT_HALF, 3, 8, 1, 0, 1, 160, 0.1, 3, PTR, 1024, 128, PTR, 1024, 128, PTR, 10, 10, PTR, 0, 0, PTR, 1 << 30)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change, text", CACHE)
def test_cache_refuses(mods, change, text):
    lib, L, _, _ = mods
    c = cache_params(L, **change)
    refused(lib, L, "kv4_append", append_params(L, c), text)
    refused(lib, L, "kv4_gather", gather_params(L, c), text)
    refused(lib, L, "kv4_attention", attention_params(L, c), text)


def test_append_and_gather_refuse(mods):
    lib, L, _, _ = mods
    for name in ("kv4_append", "kv4_gather", "kv4_attention"):
        refused(lib, L, name, None, "NULL params")
    for name, make in (("kv4_append", append_params), ("kv4_gather", gather_params)):
        refused(lib, L, name, make(L, dtype=L.DT_QINT8), "unsupported type qint8")
        refused(lib, L, name, make(L, slots_dtype=L.DT_FLOAT), "slots must be int32 or int64")
        refused(lib, L, name, make(L, tokens=-1), "bad number of tokens")
        refused(lib, L, name, make(L, tokens=1 << 31), "bad number of tokens")
        refused(lib, L, name, make(L, slots=0), "NULL tensor")
        refused(lib, L, name, make(L, v=0), "NULL tensor")
        assert getattr(lib, "itexb_" + name)(C.byref(make(L, tokens=0, slots=0)), None) == L.OK
    refused(lib, L, "kv4_append", append_params(L, positions_dtype=L.DT_HALF), "positions must be int32 or int64")
    refused(lib, L, "kv4_append", append_params(L, rotary_dim=130), "rotary_dim must be even")
    refused(lib, L, "kv4_append", append_params(L, rotary_dim=5), "rotary_dim must be even")
    refused(lib, L, "kv4_append", append_params(L, inv_freq=0), "NULL frequencies")


@pytest.mark.parametrize("change, text", [
    (dict(dtype=1), "unsupported type float"), (dict(q_heads=7), "multiple of kv_heads"), (dict(q_heads=0), "multiple of kv_heads"), (dict(num_seqs=-1), "multiple of kv_heads"),
    (dict(max_new=-1), "negative bound"), (dict(max_kept=-1), "negative bound"), (dict(window=-1), "negative bound"), (dict(total_rows=-1), "negative bound"),
    (dict(table_cols=-1), "negative bound"), (dict(num_seqs=65536), "65535"), (dict(max_new=1 << 29), "2^31 query rows"), (dict(q=0), "NULL tensor"),
    (dict(kept=0), "NULL tensor"), (dict(block_table=0), "NULL tensor")])
def test_attention_refuses(mods, change, text):
    lib, L, _, _ = mods
    refused(lib, L, "kv4_attention", attention_params(L, **change), text)


def test_attention_of_nothing_is_nothing(mods):
    lib, L, _, _ = mods
    for change in (dict(num_seqs=0), dict(max_new=0), dict(total_rows=0)):
        assert lib.itexb_kv4_attention(C.byref(attention_params(L, q=0, **change)), None) == L.OK


def test_python_face_refuses(mods):
    _, _, K, kv4 = mods
    q, pos, freq = torch.zeros(4, 2, 64), torch.arange(4), torch.ones(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        K.rope(q, pos, freq)
    with pytest.raises(ValueError, match="CUDA tensors"):
        kv4.Kv4Cache.allocate(4, 16, 2, 64, device="cpu")
    for bad in (torch.zeros(4, 64), torch.zeros(4, 2, 64).transpose(1, 2)):
        with pytest.raises(ValueError, match="dense last dimension"):
            K._rows(bad, "q")
    with pytest.raises(ValueError, match="unsupported type"):
        K._rows(q.double(), "q")
    with pytest.raises(ValueError, match="expected"):
        K._rows(q.half(), "out", q)
    with pytest.raises(ValueError, match="dense vector of 5"):
        K._vector(pos, "positions", K._INDEX_DT, 5)
    with pytest.raises(ValueError, match="dense vector"):
        K._vector(pos.float(), "positions", K._INDEX_DT)


def test_rope_frequencies(mods):
    _, _, _, kv4 = mods
    plain, m = kv4.rope_frequencies(64, base=500.0, device="cpu")
    assert plain.dtype == torch.float64 and m == 1.0
    for i in (0, 1, 31):
        assert math.isclose(plain[i].item(), 500.0 ** (-2 * i / 64), rel_tol=1e-14)
    assert torch.equal(kv4.rope_frequencies(64, base=500.0, scaling="linear", factor=4.0, device="cpu")[0], plain / 4.0)
    f, _ = kv4.rope_frequencies(64, base=500.0, scaling="base", factor=4.0, device="cpu")
    assert f[0] == 1.0 and math.isclose(f[-1].item(), plain[-1].item() / 4.0, rel_tol=1e-12)
    for kind in ("by_parts", "by_length"):
        f, m = kv4.rope_frequencies(128, scaling=kind, factor=8.0, trained=4096, fast=32.0, slow=1.0, device="cpu")
        base = kv4.rope_frequencies(128, device="cpu")[0]
        turns = 4096 * base / (2 * math.pi)
        ratio = base / f
        # 1 + 2^-40: one rounding of a 64-bit blend
        assert torch.all(ratio >= 1.0 - 2.0 ** -40) and torch.all(ratio <= 8.0 * (1.0 + 2.0 ** -40))
        assert torch.all(ratio[1:] >= ratio[:-1] * (1.0 - 2.0 ** -40))           # never less stretched than a faster pair
        assert ratio[0] == 1.0 and math.isclose(ratio[-1].item(), 8.0, rel_tol=1e-12)
        assert m == (0.1 * math.log(8.0) + 1.0 if kind == "by_parts" else 1.0)
        if kind == "by_length":
            assert torch.all(ratio[turns >= 32.0] == 1.0)
            assert torch.allclose(ratio[turns <= 1.0], torch.full_like(ratio[turns <= 1.0], 8.0), rtol=1e-12)
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="stretch"),
                dict(rotary_dim=2, scaling="base", factor=2.0), dict(rotary_dim=8, scaling="by_parts", fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            kv4.rope_frequencies(device="cpu", **bad)
