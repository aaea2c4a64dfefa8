"""Outputs of the rotation of heads that overlap what is read, as views that are not dense: heads of one projection, rows of one cache."""
import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads, rotate_heads
from native_sparse_attention_pytorch_b200 import _lib as L
from test_gpu_heads import DEV, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_views_that_overlap_are_refused(dtype):
    rotary, w = RotaryFrequencies(64), torch.ones(64, device=DEV, dtype=dtype)
    qkv, cache = randn((2, 5, 9, 64), 1, dtype).transpose(1, 2), randn((2, 2, 40, 64), 2, dtype)
    q, k = qkv[:, :6], qkv[:, 6:8]
    flat = randn((2 * 6 * 5 * 64,), 3, dtype)
    cases = [
        (lambda: rotate_heads(q, None, rotary, out=(qkv[:, 1:7], None)), 'must not overlap it'),                 # a head further
        (lambda: rotate_heads(cache[:, :, 6:11], None, rotary, out=(cache[:, :, 7:12], None)), 'must not overlap it'),     # a row further
        (lambda: rotate_heads(cache[:, :, 6:11], None, rotary, out=(cache[:, :, 2:7], None)), 'must not overlap it'),
        (lambda: rotate_heads(cache[:, :, :5], None, rotary, out=(cache[:, :, 0:10:2], None)), 'must not overlap it'),
        (lambda: rotate_heads(q, k, rotary, out=(qkv[:, 2:8], None)), 'must not overlap'),
        (lambda: rotate_heads(q.clone(), k, rotary, out=(qkv[:, 2:8], None)), "overlap the other"),
        (lambda: rotate_heads(q.clone(), k.clone(), rotary, out=(qkv[:, :6], qkv[:, 5:7])), "overlap the other"),
        (lambda: norm_rotate_heads(q, k, w, w, rotary, out=(None, q[:, 4:])), "overlap the other"),
        (lambda: rotate_heads(q, None, rotary, out=(flat.as_strided((2, 6, 5, 64), (1920, 320, 32, 1)), None)), 'overlap itself'),
        (lambda: norm_rotate_heads(q.clone(), None, qkv[0, 3, 2], None, rotary, out=(q, None)), 'weights'),
        (lambda: rotate_heads(q.clone(), None, rotary, flat.view(torch.int64)[8:13], out=(flat.view_as(q), None)), 'positions'),
    ]
    before = qkv.clone(), cache.clone(), flat.clone()
    for call, match in cases:
        with pytest.raises(L.NsaError, match=match):
            call()
    assert all(torch.equal(a, b) for a, b in zip(before, (qkv, cache, flat)))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_views_beside_one_another_are_served(dtype):
    rotary = RotaryFrequencies(64, 32, layout='half')
    qkv, cache = randn((2, 5, 17, 64), 1, dtype).transpose(1, 2), randn((2, 2, 40, 64), 2, dtype)
    q, k = qkv[:, :6], qkv[:, 6:8]
    y, z = rotate_heads(q, k, rotary, offset=3)
    rest = qkv[:, 14:].clone(), cache[:, :, :6].clone(), cache[:, :, 11:].clone()
    rotate_heads(q, k, rotary, offset=3, out=(qkv[:, 8:14], cache[:, :, 6:11]))        # other heads of the same buffer, rows of a cache
    assert torch.equal(qkv[:, 8:14], y) and torch.equal(cache[:, :, 6:11], z)
    assert torch.equal(q, qkv[:, :6]) and all(torch.equal(a, b) for a, b in zip(rest, (qkv[:, 14:], cache[:, :, :6], cache[:, :, 11:])))
    rotate_heads(cache[:, :, 6:11], None, rotary, out=(cache[:, :, 20:25], None))      # rows that have been used, further back
    assert torch.equal(cache[:, :, 20:25], rotate_heads(z, None, rotary)[0])
    rotate_heads(q, k, rotary, offset=3, out=(q, k))
    assert torch.equal(q, y) and torch.equal(k, z)
    one = randn((3, 1, 8, 64), 4, dtype).transpose(1, 2)                               # one token: an axis of one entry has any stride
    y, z = rotate_heads(one[:, :6], one[:, 6:], rotary, offset=9)
    rotate_heads(one[:, :6], one[:, 6:], rotary, offset=9, out=(one[:, :6], one[:, 6:]))
    assert torch.equal(one[:, :6], y) and torch.equal(one[:, 6:], z)
