"""Rotation of heads: numbers of heads next to 2^31 are refused before they overflow, without a GPU."""
import ctypes as C

import pytest

from native_sparse_attention_pytorch_b200 import _lib as L

MOST = (1 << 31) - 1


@pytest.mark.parametrize('hq, hk, code', [(MOST, 0, -2), (MOST, MOST, -2), (0, MOST - 63, -2), (1 << 30, 1 << 30, -2), (MOST - 64, 0, -1), (1 << 29, 1 << 29, -1)])
def test_heads_next_to_2_to_the_31(hq, hk, code):
    lib = L.load()
    a = L.HeadsArgs(batch=1, seq=1, dim_head=2, rotary_dim=2, dtype=L.NSA_BF16)
    a.part[0].heads, a.part[1].heads = hq, hk
    for call in (lib.nsa_heads_fwd, lib.nsa_heads_bwd):
        assert call(C.byref(a), None) == code          # -1: sizes pass, the frequencies are NULL
