"""Norm and rotation of rows and weights that start on narrow boundaries, gradients of all of them.

Bounds as in test_gpu_heads, whose 4 * 2^-24 for a sine or cosine is made up so: the phase cut to 2^-32 turns (7e-10), as fp32 and times
2 pi / 2^32 (pi / 4 of 2^-25 and of 2^-24: 1.2 units of 2^-24), the first term left out of the series (2.5e-8, 0.4 units), the
roundings of the last steps (at most 2 units)."""
import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads
from test_gpu_heads import DEV, angles, check_backward, check_forward, randn

pytestmark = pytest.mark.gpu
EPS = torch.finfo(torch.float32).eps


def check_both(x, w, rotary, dy, what):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = norm_rotate_heads(x, None, w, None, rotary)[0]
    angle = angles(rotary, torch.arange(x.shape[2], device=DEV))
    check_forward(x.detach(), w.detach(), y.detach(), rotary, angle, EPS, what)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dw.dtype == w.dtype and dw.shape == w.shape
    check_backward(x.detach(), w.detach(), dy, dx, dw, rotary, angle, EPS, what)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout, r', [('half', 32), ('half', 20), ('interleaved', 64), ('interleaved', 6)])
@pytest.mark.parametrize('weights', ['shared', 'heads'])
@pytest.mark.parametrize('pad, shift', [(1, 0), (2, 2), (4, 4), (0, 1), (3, 5), (8, 0)])
def test_rows_on_narrow_boundaries(dtype, layout, r, weights, pad, shift):
    """A slice of rows of d + pad elements, `shift` into the buffer; the gradient that arrives in another order, on its own boundaries."""
    b, h, n, d = 2, 3, 11, 64
    rotary = RotaryFrequencies(d, r, layout=layout)
    x = randn((shift + b * h * n * (d + pad),), 3, dtype)[shift:].view(b, h, n, d + pad)[..., :d]
    w = 1 + randn((h, d) if weights == 'heads' else (d,), 4, dtype, 0.3)
    for dy in (randn((b, n, h, d + pad), 5, dtype)[..., :d].transpose(1, 2), randn((b, h, n, d), 6, dtype)):
        check_both(x, w, rotary, dy, f'{pad} {shift}')
    last = randn((b, h, d, n), 6, dtype).transpose(2, 3)          # the last axis is not contiguous, neither x's nor the gradient's
    check_both(last, w, rotary, randn((b, h, d, n), 7, dtype).transpose(2, 3), 'transposed')


@pytest.mark.parametrize('layout', ['interleaved', 'half'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_weights_on_narrow_boundaries(layout, dtype):
    """Weights of the rows' type and fp32 ones, views into a flat buffer of parameters."""
    rotary, x = RotaryFrequencies(64, layout=layout), randn((1, 3, 6, 64), 1, dtype)
    dy = randn((1, 3, 6, 64), 2, dtype)
    for wdtype in {dtype, torch.float32}:
        flat = 1 + randn((64 * 3 + 8,), 3, wdtype, 0.3)
        for shift in (0, 1, 2, 3, 4):
            check_both(x, flat[shift:shift + 64], rotary, dy, f'{wdtype} {shift}')
            check_both(x, flat[shift:shift + 192].view(3, 64), rotary, dy, f'{wdtype} {shift} by heads')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('weights', ['shared', 'heads'])
def test_many_tokens_on_narrow_boundaries(dtype, weights):
    """More tokens than the blocks of the weights' partial sums take in one go."""
    b, h, n, d = 2, 4, 9001, 32
    x = randn((b, n, h, d + 2), 1, dtype)[..., :d].transpose(1, 2)
    w = (1 + randn((h, d) if weights == 'heads' else (d,), 2, dtype, 0.3)).requires_grad_()
    dy, rotary = randn((b, h, n, d), 3, dtype), RotaryFrequencies(d)
    leaf = x.detach().requires_grad_()
    y = norm_rotate_heads(leaf, None, w, None, rotary)[0]
    dx, dw = torch.autograd.grad(y, (leaf, w), dy)
    angle = angles(rotary, torch.arange(n, device=DEV))
    check_forward(x, w.detach(), y.detach(), rotary, angle, EPS, 'y')
    check_backward(x, w.detach(), dy, dx, dw, rotary, angle, EPS, 'many')     # at most 256 additions in a row here as well
