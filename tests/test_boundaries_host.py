"""Pointers that do not lie on a boundary of their type are refused by the entry points for heads and drafted tokens, without a GPU."""
import ctypes as C

import pytest

from native_sparse_attention_pytorch_b200 import _lib as L


def heads(**kw):
    a = L.HeadsArgs(batch=1, seq=4, dim_head=64, rotary_dim=64, dtype=L.NSA_BF16, norm=1, steps=0x1000, pos_i64=1, positions=0x2000)
    a.part[0].heads = 2
    for name in ('x', 'dy', 'out'):
        getattr(a.part[0], name).ptr = 0x1000
    a.part[0].weight = a.part[0].dweight = 0x1000
    for name, value in kw.items():
        setattr(a.part[0] if name in ('weight', 'dweight') else a, name, value)
    return a


@pytest.mark.parametrize('change, forward', [(dict(steps=0x1004), -4), (dict(positions=0x2004), -4), (dict(positions=0x2002, pos_i64=0), -4),
                                             (dict(weight=0x1001), -4), (dict(weight=0x1002, weight_f32=1), -4), (dict(dweight=0x1001), None),
                                             (dict(dweight=0x1002, weight_f32=1), None)])
def test_heads(change, forward):
    lib = L.load()
    if forward is not None:
        assert lib.nsa_heads_fwd(C.byref(heads(**change)), None) == forward
    assert lib.nsa_heads_bwd(C.byref(heads(**change)), None) == -4


@pytest.mark.parametrize('change', [dict(), dict(positions=0x2004, pos_i64=0), dict(weight=0x1002), dict(weight=0x1004, dweight=0x1004, weight_f32=1)])
def test_heads_on_their_boundaries(change):
    assert L.load().nsa_heads_bwd(C.byref(heads(**change)), None) == -5       # as far as the missing work buffer


@pytest.mark.parametrize('field', ['lengths', 'lse', 'status'])
def test_drafted_tokens(field):
    lib = L.load()
    a = L.TreeArgs(batch=1, q_heads=4, kv_heads=2, tokens=3, dim_head=64, capacity=4096, length=4096, dtype=L.NSA_F32, scale=0.125)
    for name in ('q', 'k', 'v', 'out', 'k_cache', 'v_cache'):
        getattr(a, name).ptr = 0x1000
    setattr(a, field, 0x1004)
    assert lib.nsa_tree_attend(C.byref(a), None) == -5
    setattr(a, field, 0x1002)
    assert lib.nsa_tree_attend(C.byref(a), None) == -4
