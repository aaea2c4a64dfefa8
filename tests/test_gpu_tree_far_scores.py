"""Attention of drafted tokens where logits are as low as the type holds or far apart: a bias of the keys carried in a feature (queries 1
there) that pads the front of a cache, and queries and keys of large numbers.

References.  A key whose logit lies 10^37 below another visible one has weight zero in any precision, so padded rows may be left out of
the 64-bit formula, and the bounds are those of test_gpu_tree.  Where all logits are alike the weights are 1 / n, exact in bf16 before
the division: sums of n terms are off by n 2^-24, quotient and type by a rounding each; lse by 2^-24 for each of the two factors, the
product by scale and the sum."""
import pytest
import torch

from test_gpu_tree import DEV, U, check, problem, reference, rounded, run, tree_mask
from test_gpu_tree_scores import FAMILIES, ROWS, check_by_sequence

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', ROWS)
def test_padded_rows_at_the_front_of_a_cache(dtype, impl, t, hq, hkv):
    """Padding of a part of a block, whole blocks, whole pieces of the cache and all of it."""
    b, d, capacity = 7, 64, 2600
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, capacity, dtype, seed=t)
    q, k = q.clone(), k.clone()
    pads, lengths = [0, 1, 128, 129, 700, 2599, 2600], [2600, 2600, 2500, 300, 2600, 2600, 2600]
    q[..., -1], kc[..., -1], k[..., -1] = 1, 0, 0
    for s, p in enumerate(pads):
        kc[s, :, :p, -1] = torch.finfo(dtype).min
    mask = tree_mask(b, t, t)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    for m in (mask, None):
        check_by_sequence(run(q, kc, vc, n, k, v, m, impl), q, kc, vc, lengths, k, v, m, pads, rounded(dtype, impl))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', ROWS)
def test_padded_rows_between_others(dtype, impl, t, hq, hkv):
    """Blocks of padding in the middle and at the end of a cache, and drafted tokens whose own keys are padded."""
    b, d, capacity = 3, 128, 1500
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, capacity, dtype, seed=t + 1)
    q, k = q.clone(), k.clone()
    q[..., -1], kc[..., -1], k[..., -1] = 1, 0, 0
    low = torch.finfo(dtype).min
    kc[:, :, 100:700, -1], kc[:, :, 900:, -1] = low, low
    k[:, :, 1::2, -1] = low
    keep = torch.cat((torch.arange(100), torch.arange(700, 900))).to(DEV)
    mask = torch.ones(b, t, t, dtype=torch.bool, device=DEV).tril()
    seen = mask.clone()
    seen[:, :, 1::2] = False
    got = run(q, kc, vc, None, k, v, mask, impl)
    check(got, reference(q, kc[:, :, keep], vc[:, :, keep], [300] * b, k, v, seen, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', ROWS)
@pytest.mark.parametrize('length', [0, 130, 2000])
def test_all_logits_the_lowest_value(dtype, impl, t, hq, hkv, length):
    """The bias outweighs everything: all visible keys alike."""
    d = 64
    q, kc, vc, k, v = problem(1, t, hq, hkv, d, 2000, dtype, seed=4)
    q = q.clone()
    low = torch.finfo(dtype).min
    kc, k = torch.zeros_like(kc), torch.zeros_like(k)
    q[..., -1], kc[..., -1], k[..., -1] = 1, low, low
    got = run(q, kc, vc, length, k, v, None, impl)
    n = length + torch.arange(1, t + 1, device=DEV).double()[:, None]
    values = torch.cat((vc[0, :, :length], v[0]), 1).double()
    mean, size = values.cumsum(1)[:, length:] / n, values.abs().cumsum(1)[:, length:] / n
    mean, size = (x.repeat_interleave(hq // hkv, 0)[None] for x in (mean, size))
    half = torch.finfo(dtype).eps / 2
    assert ((got[0].double() - mean).abs() <= (length + t + 4) * U * size + half * mean.abs() * (1 + U)).all()
    lse = low * d ** -0.5
    assert ((got[1].double() - lse).abs() <= 4 * 2 * U * abs(lse)).all()


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', ROWS)
@pytest.mark.parametrize('sign', [1, -1])
@pytest.mark.parametrize('power', [15, 40])
def test_logits_far_apart(dtype, impl, t, hq, hkv, sign, power):
    """Logits of a few exact numbers above 2^32: the keys of the largest share the weight evenly, wherever they lie."""
    b, d, capacity = 3, 64, 1800
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, capacity, dtype, seed=5)
    gen = torch.Generator().manual_seed(7)
    steps = torch.randint(1, 5, (b, hkv, capacity), generator=gen).to(DEV)
    steps[1] = torch.arange(capacity, device=DEV) // 300 + 1                 # grows from block to block
    steps[2] = steps[1].flip(-1)                                             # falls
    q, kc, k = torch.zeros_like(q), torch.zeros_like(kc), torch.zeros_like(k)
    q[..., 0], kc[..., 0], k[..., 0] = 2. ** power, steps.to(dtype) * sign * 2. ** 20, (-100. if sign < 0 else -1.) * 2. ** 20
    out, lse = run(q, kc, vc, None, k, v, None, impl)
    top = (steps * sign).amax(-1, keepdim=True)
    where = (steps * sign == top).double()
    count = where.sum(-1)
    mean = torch.einsum('bkn,bknd->bkd', where, vc.double()) / count[..., None]
    size = torch.einsum('bkn,bknd->bkd', where, vc.double().abs()) / count[..., None]
    mean, size = (x.repeat_interleave(hq // hkv, 1)[:, :, None] for x in (mean, size))
    half = torch.finfo(dtype).eps / 2
    assert ((out.double() - mean).abs() <= (capacity + 4) * U * size + half * mean.abs() * (1 + U)).all()
    expect = (top.double() * 2. ** (power + 20) * d ** -0.5).repeat_interleave(hq // hkv, 1)
    assert ((lse.double() - expect).abs() <= 4 * 2 * U * expect.abs()).all()


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', ROWS)
def test_scaled_far_apart_between_ordinary_ones(dtype, impl, t, hq, hkv):
    """One sequence of large numbers leaves the others' bits as they are."""
    b, d = 4, 64
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, 1200, dtype, seed=6)
    n = torch.tensor([1200, 1100, 5, 1200], dtype=torch.int32, device=DEV)
    clean = run(q, kc, vc, n, k, v, None, impl)
    q, kc = q.clone(), kc.clone()
    q[1] *= 2. ** 30
    kc[1] *= 2. ** 10
    got = run(q, kc, vc, n, k, v, None, impl)
    for s in (0, 2, 3):
        assert torch.equal(got[0][s], clean[0][s]) and torch.equal(got[1][s], clean[1][s])
    assert got[0][1].isfinite().all() and got[1][1].isfinite().all()
    # the largest logit's value alone, as far as fp32 tells them apart: no value beyond those of the sequence
    most = torch.cat((vc[1, :, :1100], v[1]), 1).abs().amax((1, 2)).repeat_interleave(hq // hkv)[:, None, None]
    assert (got[0][1].abs() <= most * (1 + 2. ** -7)).all()
