"""Caches of as many rows as an int holds: lengths less than a block below 2^31.  Rows overlap in memory (a stride of zero, or of
sixteen bytes, which is what the tensor-core kernels want at least); all logits are zero and all values one, so that sums are whole
numbers below 2^24 in every thread and tile, and the joined ones are off by a rounding for each of a few hundred parts."""
import math

import pytest
import torch

from native_sparse_attention_pytorch_b200 import ops, tree_attend

pytestmark = pytest.mark.gpu
DEV = 'cuda'
MOST = (1 << 31) - 1


def check(q, cache, t, length, impl):
    k = torch.ones(1, 1, t, q.shape[-1], device=DEV, dtype=q.dtype)
    out, lse = tree_attend(q, cache, cache, length, k, k, return_lse=True, impl=impl)
    ops.check_device_status()
    n = min(length, MOST) if isinstance(length, int) else int(length)
    expect = torch.log(n + torch.arange(1, t + 1, device=DEV).double())
    assert ((lse[0].double() - expect).abs() <= 512 * 2.0 ** -24 + 2.0 ** -23 * math.log(2.0 ** 31)).all()
    assert ((out.double() - 1).abs() <= 512 * 2.0 ** -24 + torch.finfo(q.dtype).eps / 2).all()


@pytest.mark.parametrize('t', [1, 12])
def test_on_the_cuda_cores(t):
    row = torch.ones(1, 1, 1, 8, device=DEV).expand(1, 1, MOST, 8)
    check(torch.zeros(1, 1, t, 8, device=DEV), row, t, MOST, 'auto')


def test_on_the_tensor_cores():
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip('34 GB of rows')
    flat = torch.ones(8 * MOST + 64, device=DEV, dtype=torch.bfloat16)
    cache = flat.as_strided((1, 1, MOST, 64), (8, 8, 8, 1))
    for t in (1, 20, 60, 100, 200):
        check(torch.zeros(1, 1, t, 64, device=DEV, dtype=torch.bfloat16), cache, t, MOST, 'sm100')
    check(torch.zeros(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16), cache, 1, torch.tensor([MOST - 60], device=DEV), 'sm100')
    del flat, cache
    torch.cuda.empty_cache()
