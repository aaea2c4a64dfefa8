"""Attention of drafted tokens where logits are -inf although everything is visible: a bias of the keys carried in a feature (queries 1
there), as it pads the front of a cache.

Such keys have weight zero, so they are left out of the 64-bit formula, and the bounds are those of test_gpu_tree."""
import math

import pytest
import torch

from test_gpu_tree import DEV, check, problem, reference, rounded, run, tree_mask

pytestmark = pytest.mark.gpu

FAMILIES = [(torch.float32, 'auto'), (torch.bfloat16, 'simt'), (torch.bfloat16, 'sm100')]
# rows of a KV head: every tile of either kernel
ROWS = [(1, 8, 2), (6, 8, 2), (16, 8, 2), (25, 8, 2), (64, 8, 2)]


def check_by_sequence(got, q, kc, vc, lengths, k, v, mask, pads, weights_rounded):
    """Every sequence by itself, its first rows left out"""
    for s, (n, p) in enumerate(zip(lengths, pads)):
        at = slice(s, s + 1)
        p = min(p, n)
        ref = reference(q[at], kc[at, :, p:], vc[at, :, p:], [n - p], k[at], v[at], None if mask is None else mask[at], weights_rounded=weights_rounded)
        check((got[0][at], got[1][at]), ref, f'sequence {s}')


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
        kc[s, :, :p, -1] = -math.inf
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
    low = -math.inf
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
def test_nothing_but_logits_of_minus_infinity(dtype, impl, t, hq, hkv):
    """A token that sees keys of -inf alone is one that sees nothing."""
    q, kc, vc, k, v = problem(2, t, hq, hkv, 64, 900, dtype, seed=3)
    q, k = q.clone(), k.clone()
    q[..., -1], kc[..., -1], k[..., -1] = 1, -math.inf, -math.inf
    out, lse = run(q, kc, vc, torch.tensor([900, 0], dtype=torch.int32, device=DEV), k, v, None, impl)
    assert (out == 0).all() and (lse == -math.inf).all()
