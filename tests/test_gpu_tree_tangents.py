"""Attention of drafted tokens in forward mode: tensors with a tangent are refused, tensors without one are not."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from native_sparse_attention_pytorch_b200 import _lib as L
from native_sparse_attention_pytorch_b200 import tree_attend
from test_gpu_tree import problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_tangents_are_refused_not_dropped(dtype):
    args = problem(1, 3, 4, 2, 64, 10, dtype)
    expected = tree_attend(*args[:3], None, *args[3:])
    for i in range(5):
        with fw.dual_level():
            given = [fw.make_dual(x, torch.ones_like(x)) if j == i else x for j, x in enumerate(args)]
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(L.NsaError, match='no forward-mode derivative'):
                    tree_attend(*given[:3], None, *given[3:])
            plain = [fw.unpack_dual(x).primal for x in given]
            assert torch.equal(tree_attend(*plain[:3], None, *plain[3:]), expected)
    assert torch.equal(tree_attend(*args[:3], None, *args[3:]), expected)
