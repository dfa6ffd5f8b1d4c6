"""What the prompt-side operators (append with rotation, chunk attention) refuse before they touch a device."""
import ctypes as C

import pytest
import torch

import rmlx_kv
from rmlx_kv import _lib


def test_null_pool_and_rope():
    rope = _lib.RopeStruct(None, None, 32, 0, 1)
    lib = _lib.lib
    assert lib.rmlx_kv_append_rope(None, 0, C.byref(rope), None, 0, None, 0, 0, 0, None, 0, 0, None, None, 0, 0, None, 0,
                                   None) == _lib.E_BAD_ARG
    assert lib.rmlx_kv_chunk_attention(None, 0, None, 0, 0, 1, None, 1, None, None, 0, 0, 1.0, 0, None, None, 0,
                                       None) == _lib.E_BAD_ARG
    n = C.c_size_t()
    assert lib.rmlx_kv_chunk_attention_workspace_size(None, 1, C.byref(n)) == _lib.E_BAD_ARG


def test_rope_arrays():
    inv = torch.ones(16)
    rmlx_kv.Rope(inv, 32)
    rmlx_kv.Rope(inv, 32, pair_axis=torch.zeros(16, dtype=torch.int32), num_axes=3)
    for args in ((inv.double(), 32), (inv, 64), (torch.ones(32)[::2], 32), (inv, 32, False, torch.zeros(16)),
                 (inv, 32, False, torch.zeros(15, dtype=torch.int32))):
        with pytest.raises(ValueError):
            rmlx_kv.Rope(*args)
