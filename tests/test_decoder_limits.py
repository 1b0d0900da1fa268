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
