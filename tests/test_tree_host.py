"""Attention of drafted tokens over a cache, host side: what is refused, and how the key blocks are shared out, without a GPU."""
import ctypes as C

import pytest
import torch

from native_sparse_attention_pytorch_b200 import _lib as L
from native_sparse_attention_pytorch_b200 import tree_attend


def test_no_cpu_path():
    q, c = torch.randn(1, 2, 3, 64), torch.randn(1, 2, 8, 64)
    with pytest.raises(L.NsaError, match='CUDA tensors only'):
        tree_attend(q, c, c, None, q, q)
    with pytest.raises(L.NsaError, match='capacity'):
        tree_attend(q, c, c, 9, q, q)


def args(**kw):
    a = L.TreeArgs(batch=1, q_heads=4, kv_heads=2, tokens=3, dim_head=64, capacity=8, length=8, dtype=L.NSA_F32, scale=0.125)
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize('change, code', [(dict(q_heads=3), -2), (dict(dim_head=60), -2), (dict(dim_head=136), -2), (dict(dtype=5), -3),
                                          (dict(capacity=-1), -2), (dict(tokens=-1), -2), (dict(impl=3), -2), (dict(tokens=1 << 24), -2),
                                          (dict(), -1)])
def test_entry_point_checks_its_arguments(change, code):
    lib = L.load()
    assert lib.nsa_tree_attend(None, None) == -1 and lib.nsa_tree_workspace_bytes(None) == -1
    assert lib.nsa_tree_attend(C.byref(args(**change)), None) == code


def test_pointers_and_work_buffer_are_checked():
    lib = L.load()
    a = args(capacity=4096, length=4096)
    for name in ('q', 'k', 'v', 'out', 'k_cache', 'v_cache'):
        getattr(a, name).ptr = 0x1000
    need = lib.nsa_tree_workspace_bytes(C.byref(a))
    assert need > 0 and lib.nsa_tree_attend(C.byref(a), None) == -5
    a.workspace, a.workspace_bytes = 0x1000, need - 1
    assert lib.nsa_tree_attend(C.byref(a), None) == -5
    a.workspace, a.workspace_bytes = 0x1080, need
    assert lib.nsa_tree_attend(C.byref(a), None) == -5
    a.k.ptr = 0x1002
    assert lib.nsa_tree_attend(C.byref(a), None) == -4
    a.tokens = 0
    assert lib.nsa_tree_attend(C.byref(a), None) == 0 and lib.nsa_tree_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize('blocks, groups', [([1], 1), ([1], 148), ([3, 1, 9], 5), ([7] * 12, 148), ([100, 1, 1, 57], 74), ([2, 2, 2], 3)])
def test_pieces_cover_every_unit_once(blocks, groups):
    """The arithmetic by which kernels and merge share key blocks: `begin` of a group, and the group that has a block."""
    total = sum(blocks)

    def begin(g):
        return total * g // groups

    def group_of(x):
        return ((x + 1) * groups - 1) // total
    start = 0
    for n in blocks:
        g0, g1 = group_of(start), group_of(start + n - 1)
        covered = [x for g in range(g0, g1 + 1) for x in range(max(begin(g), start), min(begin(g + 1), start + n))]
        assert covered == list(range(start, start + n))
        writers = [g for g in range(groups) if begin(g) < start + n and begin(g + 1) > start and begin(g) < begin(g + 1)]
        assert writers[0] == g0 and writers[-1] == g1
        # a group's partial of a unit that it begins with lies in slot 1, else in slot 0; it has at most one of each
        for g in writers:
            assert (begin(g) <= start) == (g == g0)
        start += n
