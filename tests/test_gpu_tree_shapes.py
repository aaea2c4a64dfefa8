"""Attention of drafted tokens over a cache, further shapes and uses: every number of rows at which another tile is chosen, more
tokens than a tile, long chains, calls side by side on two streams, recorded calls whose masks and caches change, drafts of padded
batches."""
import pytest
import torch

from native_sparse_attention_pytorch_b200 import ops, tree_attend
from test_gpu_tree import DEV, FAMILIES, check, problem, reference, rounded, run, tree_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('t, g', [(1, 8), (2, 4), (1, 9), (1, 16), (16, 1), (1, 17), (4, 8), (8, 4), (11, 3), (1, 40), (16, 4), (13, 5), (32, 4), (43, 3), (64, 4), (65, 4), (97, 4)])
def test_rows_around_the_tiles(dtype, impl, d, t, g):
    q, kc, vc, k, v = problem(2, t, 2 * g, 2, d, 700, dtype, seed=t * 10 + g)
    lengths = torch.tensor([690, 257], dtype=torch.int32, device=DEV)
    mask = tree_mask(2, t, t)
    check(run(q, kc, vc, lengths, k, v, mask, impl), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('t, hq, hkv', [(300, 4, 1), (513, 2, 2)])
def test_long_chains(dtype, impl, t, hq, hkv):
    """A chunk of a prompt against a cache: several tiles, and drafted blocks that a tile's early rows do not see at all."""
    q, kc, vc, k, v = problem(1, t, hq, hkv, 64, 900, dtype, seed=t)
    for length in (0, 777):
        check(run(q, kc, vc, length, k, v, None, impl), reference(q, kc, vc, [length], k, v, None, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
def test_drafts_of_a_padded_batch(dtype, impl):
    """Sequences with fewer drafted tokens than the batch has room for: what lies in the other rows, NaN included, changes nothing."""
    b, t = 3, 20
    q, kc, vc, k, v = problem(b, t, 8, 2, 64, 300, dtype, seed=3)
    lengths = torch.tensor([299, 5, 128], dtype=torch.int32, device=DEV)
    drafted = [20, 7, 1]
    mask = tree_mask(b, t, 4)
    for s, n in enumerate(drafted):
        mask[s, n:], mask[s, :, n:] = False, False
    q, k, v = q.clone(), k.clone(), v.clone()
    clean = run(q, kc, vc, lengths, k, v, mask, impl)
    check(clean, reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))
    for s, n in enumerate(drafted):
        q[s, :, n:], k[s, :, n:], v[s, :, n:] = float('nan'), float('nan'), float('inf')
    got = run(q, kc, vc, lengths, k, v, mask, impl)
    for s, n in enumerate(drafted):
        assert torch.equal(got[0][s, :, :n], clean[0][s, :, :n]) and torch.equal(got[1][s, :, :n], clean[1][s, :, :n])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_streams_at_once(dtype):
    problems = [problem(2, t, 8, 2, 64, 3000, dtype, seed=t) for t in (3, 40)]
    lengths = torch.tensor([3000, 1234], dtype=torch.int32, device=DEV)
    expected = [run(q, kc, vc, lengths, k, v) for q, kc, vc, k, v in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (q, kc, vc, k, v) in enumerate(problems):
            with torch.cuda.stream(streams[i]):
                got[i].append(tree_attend(q, kc, vc, lengths, k, v, return_lse=True))
    torch.cuda.synchronize()
    ops.check_device_status()
    for g, e in zip(got, expected):
        for out, lse in g:
            assert torch.equal(out, e[0]) and torch.equal(lse, e[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_recorded_step_with_another_tree_and_cache(dtype):
    b, t = 2, 12
    q, kc, vc, k, v = problem(b, t, 8, 2, 64, 500, dtype, seed=1)
    held = [x.clone() for x in (q, kc, vc, k, v)] + [tree_mask(b, t, 1), torch.tensor([10, 20], dtype=torch.int32, device=DEV)]
    tree_attend(*held[:3], held[6], held[3], held[4], held[5])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = tree_attend(*held[:3], held[6], held[3], held[4], held[5], return_lse=True)
    for seed, lengths in ((5, [500, 0]), (6, [77, 128])):
        new = [*problem(b, t, 8, 2, 64, 500, dtype, seed=seed), tree_mask(b, t, seed), torch.tensor(lengths, dtype=torch.int32, device=DEV)]
        for h, n in zip(held, new):
            h.copy_(n)
        g.replay()
        q, kc, vc, k, v, mask, n = new
        check((out, lse), reference(q, kc, vc, n, k, v, mask, weights_rounded=dtype == torch.bfloat16))


def test_merging_with_attention_over_other_keys():
    """Two halves of a cache by themselves, joined by their log sums, against the whole: what the sums are returned for."""
    q, kc, vc, k, v = problem(2, 6, 8, 2, 64, 600, torch.float32, seed=9)
    whole, total = run(q, kc, vc, 600, k, v)
    near, a = run(q, kc[:, :, 200:], vc[:, :, 200:], 400, k, v)
    none = torch.zeros(6, 6, dtype=torch.bool, device=DEV)
    far, b = run(q, kc[:, :, :200], vc[:, :, :200], 200, k, v, none)
    lse = torch.logaddexp(a, b)
    joined = near * (a - lse).exp()[..., None] + far * (b - lse).exp()[..., None]
    ref = reference(q, kc, vc, [600, 600], k, v, None)
    # both sides are within the bounds of the same value; the join adds a few roundings of numbers no larger than the values'
    assert ((joined.double() - whole.double()).abs() <= 3 * ref[2] + 1e-6).all()
    assert ((lse.double() - total.double()).abs() <= 3 * ref[3]).all()
