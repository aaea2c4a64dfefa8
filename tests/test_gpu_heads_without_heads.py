"""Norm and rotation of tensors without a head: their shared weight gets a gradient of zeros, beside one that gets its own."""
import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads, rotate_heads
from test_gpu_heads import DEV, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('hq, hk', [(0, 2), (3, 0), (0, 0), (0, None)])
def test_weights_of_no_heads(dtype, hq, hk):
    rotary = RotaryFrequencies(64)
    q = randn((2, hq, 5, 64), 1, dtype).requires_grad_()
    k = None if hk is None else randn((2, hk, 5, 64), 2, dtype).requires_grad_()
    weights = [(1 + randn((64,), 3 + i, dtype, 0.2)).requires_grad_() if x is not None else None for i, x in enumerate((q, k))]
    spoiled = [torch.full((64,), 7., device=DEV, dtype=dtype) for _ in range(64)]     # what the allocator hands out next
    del spoiled
    outs = [(y, x, w) for y, x, w in zip(norm_rotate_heads(q, k, *weights, rotary), (q, k), weights) if x is not None]
    ys, xs, ws = zip(*outs)
    dys = [torch.ones_like(y) for y in ys]
    grads = torch.autograd.grad(ys, (*xs, *ws), dys)
    for x, w, dx, dw in zip(xs, ws, grads, grads[len(xs):]):
        assert dx.shape == x.shape
        if x.shape[1] == 0:
            assert (dw == 0).all()
        else:
            alone = norm_rotate_heads(x, None, w, None, rotary)[0]
            assert torch.equal(dx, torch.autograd.grad(alone, x, torch.ones_like(alone))[0]) and (dw != 0).any()
    rotated = rotate_heads(q, k, rotary)
    assert rotated[0].shape == q.shape and (k is None or rotated[1].shape == k.shape)
