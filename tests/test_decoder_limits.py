"""CPU checks of the decoder operators' boundary, beside test_decoder_ops.py."""
import ctypes as C
import importlib
import math

import pytest
import torch

from test_decoder_ops import attention_params, refused


@pytest.fixture(scope="module")
def mods(itex):
    return itex.load(), itex._lib, importlib.import_module("itex_b200.kernels"), importlib.import_module("itex_b200.kv4")


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38])
def test_attention_refuses_scales_that_are_not_finite(mods, scale):
    """3e38 is none either once the base of its exponential is changed to 2."""
    lib, L, _, _ = mods
    refused(lib, L, "kv4_attention", attention_params(L, scale=scale), "scale must be finite")
    assert lib.itexb_kv4_attention_workspace_bytes(C.byref(attention_params(L, scale=scale))) == 0


@pytest.mark.parametrize("trained, base", [(4096, 10000.0), (62000, 10000.0), (70000, 10000.0), (300000, 10000.0), (131072, 1000.0)])
def test_by_parts_stretches_pairs_by_their_turns(mods, trained, base):
    """The ramp's upper end is where a pair would turn `slow` times, also where that lies behind the last pair: the slowest pairs are
    then between the two ends, not fully stretched."""
    kv4 = mods[3]
    dim, factor, fast, slow = 128, 16.0, 32.0, 1.0
    f, _ = kv4.rope_frequencies(dim, base=base, scaling="by_parts", factor=factor, trained=trained, fast=fast, slow=slow, device="cpu")

    def index(turns):            # of the pair that turns so often: trained * base ** (-2 i / dim) / (2 pi) = turns
        return dim / 2 * math.log(trained / (2 * math.pi * turns), base)

    low, high = math.floor(index(fast)), math.ceil(index(slow))
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        stretch = min(1.0, max(0.0, (i - low) / (min(high, dim - 1) - low)))
        assert math.isclose(f[i].item(), plain * (1 - stretch) + plain / factor * stretch, rel_tol=1e-12)
        turns = trained * plain / (2 * math.pi)
        if i <= low:
            assert f[i].item() == plain
        if i >= high:            # turns <= slow
            assert math.isclose(f[i].item(), plain / factor, rel_tol=1e-12)
        if turns > slow and low < i < high:
            assert plain / factor < f[i].item() < plain


@pytest.mark.parametrize("name", ["k_codes", "k_params", "v_codes", "v_params", "num_pages", "page_size", "kv_heads", "head_dim", "group", "status"])
def test_a_cache_keeps_its_tensors_and_sizes(mods, name):
    cache = object.__new__(mods[3].Kv4Cache)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(4))
