"""Which outputs of the rotation of heads meet which tensors in memory: against sets of addresses, for views as callers make them and
for any strides, without a GPU."""
import random
import time

import pytest
import torch

from native_sparse_attention_pytorch_b200 import _lib as L


def elements(t):
    at = torch.tensor([t.storage_offset()])
    for size, stride in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(size) * stride).flatten()
    return at.tolist()


def expect(a, b, what=''):
    ours = set(elements(a)) & set(elements(b))
    assert L.host().tensors_meet(a, b) == bool(ours), (what, a.shape, a.stride(), b.shape, b.stride())
    assert L.host().tensors_meet(b, a) == bool(ours), what


def test_heads_of_a_projection_and_rows_of_a_cache():
    qkv = torch.zeros(2, 5, 9, 16).transpose(1, 2)
    for a0 in range(0, 9):
        for a1 in range(a0 + 1, 10):
            for b0, b1 in ((0, 6), (6, 8), (8, 9), (3, 4)):
                expect(qkv[:, a0:a1], qkv[:, b0:b1])
    cache = torch.zeros(2, 3, 40, 16)
    for n in (1, 10):
        for shift in range(-12, 13):
            expect(cache[:, :, 14:14 + n], cache[:, :, 14 + shift:14 + shift + 10])
    expect(cache[:, :, :10, :8], cache[:, :, :10, 8:])              # halves of the features
    expect(cache[:1], cache[1:])
    expect(cache[:, ::2], cache[:, 1::2])
    expect(cache, cache.transpose(1, 2))
    assert not L.host().tensors_meet(cache, torch.zeros(2, 3, 40, 16)) and not L.host().tensors_meet(cache, cache[:0])


@pytest.mark.parametrize('seed', range(40))
def test_any_strides(seed):
    rng = random.Random(seed)
    flat = torch.zeros(4000)

    def view():
        sizes = [rng.choice((1, 1, 2, 3, 4, 5)) for _ in range(4)]
        strides = [rng.choice((0, 1, 2, 3, 4, 7, 12, 16, 30, 48, 60, 64, 128)) for _ in range(4)]
        return flat.as_strided(sizes, strides, rng.randrange(300))
    for _ in range(50):
        a, b = view(), view()
        expect(a, b)
        at = elements(a)
        assert L.host().tensor_meets_itself(a) == (len(set(at)) < len(at)), (a.shape, a.stride())


def test_other_types_and_large_tensors():
    flat = torch.zeros(64, dtype=torch.int64)
    as_bf16 = flat.view(torch.bfloat16)
    assert L.host().tensors_meet(as_bf16[6:7], flat[1:2]) and not L.host().tensors_meet(as_bf16[8:9], flat[1:2])
    # sizes as they are used (no page of these is touched)
    cache = torch.empty_strided((2, 4, 70000, 128), (4 * 70000 * 128, 70000 * 128, 128, 1), dtype=torch.bfloat16)
    qkv = torch.empty_strided((2, 80, 4000, 128), (4000 * 80 * 128, 128, 80 * 128, 1), dtype=torch.bfloat16)
    begin = time.perf_counter()
    for _ in range(100):
        assert not L.host().tensors_meet(cache[:, :, 100:200], cache[:, :, 200:300]) and L.host().tensors_meet(cache[:, :, 100:201], cache[:, :, 200:300])
        assert not L.host().tensors_meet(qkv[:, :64], qkv[:, 64:72]) and not L.host().tensor_meets_itself(qkv[:, :64])
        assert not L.host().tensors_meet(cache, qkv)
    assert time.perf_counter() - begin < 1          # some microseconds each
