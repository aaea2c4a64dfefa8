"""Views that PyTorch negates when they are read, as the imaginary part of a conjugate is: rotation of heads, its gradients, drafted
tokens over a cache."""
import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads, rotate_heads, tree_attend
from native_sparse_attention_pytorch_b200 import _lib as L
from test_gpu_heads import DEV, randn
from test_gpu_tree import problem

pytestmark = pytest.mark.gpu


def negated(x):
    """-x as a view of its memory"""
    view = torch._neg_view(x)
    assert view.is_neg() and view.data_ptr() == x.data_ptr()
    return view


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_rotation_and_gradients(dtype):
    rotary = RotaryFrequencies(64, layout='half')
    q, k = randn((2, 4, 5, 64), 1, dtype).requires_grad_(), randn((2, 2, 5, 64), 2, dtype).requires_grad_()
    w = [(1 + randn((64,), i, dtype, 0.2)).requires_grad_() for i in (3, 4)]
    dy, dz = randn(q.shape, 5, dtype), randn(k.shape, 6, dtype)
    for call in (lambda a, b, *w: rotate_heads(a, b, rotary), lambda a, b, *w: norm_rotate_heads(a, b, *w, rotary)):
        leaves = (q, k, *w)
        plain, views = call(-q, -k, -w[0], w[1]), call(negated(q), negated(k), negated(w[0]), w[1])
        assert all(torch.equal(a, b) for a, b in zip(plain, views))
        expected = torch.autograd.grad(plain, leaves, (-dy, dz), allow_unused=True)
        for a, b in zip(torch.autograd.grad(views, leaves, (negated(dy), dz), allow_unused=True), expected):
            assert (a is None and b is None) or torch.equal(a, b)
    with pytest.raises(L.NsaError, match='negated'):
        rotate_heads(q.detach(), None, rotary, out=(negated(torch.empty_like(q)).detach(), None))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_drafted_tokens(dtype):
    q, kc, vc, k, v = problem(2, 3, 4, 2, 64, 30, dtype)
    expected = tree_attend(-q, kc, vc, 20, -k, -v, return_lse=True)
    for a, b in zip(tree_attend(negated(q), kc, vc, 20, negated(k), negated(v), return_lse=True), expected):
        assert torch.equal(a, b)
    for caches in ((negated(kc), vc), (kc, negated(vc))):
        with pytest.raises(L.NsaError, match='negated'):
            tree_attend(q, *caches, 20, k, v)
