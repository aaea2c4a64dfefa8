"""Attention of drafted tokens over a cache against the formula in 64 bits: trees, chains and single tokens, ragged lengths
(zero among them), head groupings, strides, masks that leave a row empty, values that are not finite where nobody looks.

Bounds, element by element.  A logit is a sum of d products: off by (d + 4) 2^-24 of scale * sum |q k| (the tensor cores add
fp32 products of bf16 values, the CUDA cores the same in fp32) -- `slip`; weights are then off by 2 slip relative to their
sum, by the sums' roundings (at most a row's keys, n 2^-24, twice), exponentials (2^-22) and, on the tensor cores, by the
rounding of the weights to bf16, 2^-8 of each.  All of it times sum p |v|; behind it one rounding to the type, eps / 2."""
import math

import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads, ops, tree_attend
from native_sparse_attention_pytorch_b200 import _lib as L

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def tree_mask(b, t, seed):
    gen = torch.Generator().manual_seed(seed)
    mask = torch.zeros(b, t, t, dtype=torch.bool)
    for i in range(t):
        parent = torch.randint(-1, i, (b,), generator=gen) if i else torch.full((b,), -1)
        for s in range(b):
            if parent[s] >= 0:
                mask[s, i] = mask[s, parent[s]]
        mask[:, i, i] = True
    return mask.to(DEV)


def reference(q, kc, vc, lengths, k, v, mask, scale=None, weights_rounded=False):
    """-> out, lse, bound of out, bound of lse; in 64 bits, sequence by sequence"""
    b, hq, t, d = q.shape
    hkv = k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    outs = [[], [], [], []]
    for s in range(b):
        n = min(max(int(lengths[s]), 0), kc.shape[2])
        keys, vals = (torch.cat((c[s, :, :n], x[s]), 1).double() for c, x in ((kc, k), (vc, v)))
        m = torch.ones(t, t, dtype=torch.bool, device=DEV).tril() if mask is None else (mask if mask.dim() == 2 else mask[s if mask.shape[0] > 1 else 0])
        seen = torch.cat((torch.ones(t, n, dtype=torch.bool, device=DEV), m.bool()), 1)
        qs = q[s].double().view(hkv, hq // hkv, t, d)
        logits = torch.einsum('kgtd,knd->kgtn', qs, keys) * scale
        slip = (d + 4) * U * scale * torch.einsum('kgtd,knd->kgtn', qs.abs(), keys.abs()).masked_fill(~seen, 0).amax(-1)
        logits = logits.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(logits, -1)
        p = torch.exp(logits - lse[..., None]).masked_fill(~seen, 0)
        vals = vals[:, None, None].expand(-1, hq // hkv, t, -1, -1).masked_fill(~seen[None, None, :, :, None], 0)
        out, size = (p[..., None] * vals).sum(-2), (p[..., None] * vals.abs()).sum(-2)
        off = 2 * slip + 2 * (n + t) * U + 2.0 ** -21 + (2.0 ** -8 if weights_rounded else 0)
        for o, x in zip(outs, (out, lse, size * off[..., None], slip + (n + t) * U + 2.0 ** -21 * (1 + lse.abs()))):
            o.append(x.reshape(hq, t, *x.shape[3:]))
    return [torch.stack(o) for o in outs]


def check(got, ref, what=''):
    (out, lse), (r, rl, bound, lbound) = got, ref
    half = torch.finfo(out.dtype).eps / 2
    assert out.shape == r.shape and lse.shape == rl.shape
    empty = rl == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all(), what
    excess = ((out.double() - r).abs() - bound - half * (r.abs() + bound))[~empty]
    assert excess.numel() == 0 or excess.max() <= 0, f'{what} out: {excess.max().item():.3e} beyond the bound'
    excess = ((lse.double() - rl).abs() - lbound)[~empty]
    assert excess.numel() == 0 or excess.max() <= 0, f'{what} lse: {excess.max().item():.3e} beyond the bound'


def problem(b, t, hq, hkv, d, capacity, dtype, seed=0, scale=1.0):
    qkv = randn((b, t, hq + 2 * hkv, d), seed, dtype, scale).transpose(1, 2)
    return qkv[:, :hq], randn((b, hkv, capacity, d), seed + 1, dtype), randn((b, hkv, capacity, d), seed + 2, dtype), qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def run(q, kc, vc, lengths, k, v, mask=None, impl='auto', **kw):
    got = tree_attend(q, kc, vc, lengths, k, v, mask, return_lse=True, impl=impl, **kw)
    ops.check_device_status()
    return got


FAMILIES = [(torch.float32, 'auto'), (torch.bfloat16, 'simt'), (torch.bfloat16, 'auto')]


def rounded(dtype, impl):
    return dtype == torch.bfloat16 and impl != 'simt'


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('b, t, hq, hkv, d', [(1, 1, 1, 1, 64), (2, 1, 32, 4, 64), (3, 7, 8, 2, 64), (2, 16, 16, 4, 128), (1, 33, 12, 4, 32), (2, 5, 8, 8, 80),
                                              (1, 64, 8, 1, 128), (2, 9, 14, 2, 96), (1, 130, 4, 2, 64), (1, 3, 5, 1, 8)])
def test_shapes(dtype, impl, b, t, hq, hkv, d):
    capacity = 700
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, capacity, dtype, seed=b * 100 + t)
    lengths = torch.tensor([650, 1, 300][:b], dtype=torch.int32, device=DEV)
    for mask in (None, tree_mask(b, t, t), tree_mask(1, t, t + 1)[0]):
        check(run(q, kc, vc, lengths, k, v, mask, impl), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('length', [0, 1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500])
def test_lengths_around_the_blocks(dtype, impl, length):
    q, kc, vc, k, v = problem(1, 6, 8, 2, 64, 500, dtype, seed=length)
    ref = reference(q, kc, vc, [length], k, v, None, weights_rounded=rounded(dtype, impl))
    check(run(q, kc, vc, length, k, v, None, impl), ref)
    lengths = torch.tensor([length], device=DEV)          # int64 on the device
    check(run(q, kc, vc, lengths, k, v, None, impl), ref)


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('b', [1, 5, 37, 70])
def test_ragged_batches(dtype, impl, b):
    """One long sequence among short and empty ones, lengths below zero and above the capacity held to it."""
    gen = torch.Generator().manual_seed(b)
    lengths = torch.randint(0, 90, (b,), generator=gen)
    lengths[b // 2] = 1900
    lengths[0] = 5000 if b > 1 else 1900
    if b > 2:
        lengths[1], lengths[2] = -5, 0
    q, kc, vc, k, v = problem(b, 4, 4, 2, 64, 2000, dtype, seed=b)
    mask = tree_mask(b, 4, b)
    check(run(q, kc, vc, lengths.int().to(DEV), k, v, mask, impl), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
def test_masks_that_leave_rows_empty(dtype, impl):
    b, t = 3, 70
    q, kc, vc, k, v = problem(b, t, 4, 2, 64, 200, dtype)
    lengths = torch.tensor([0, 130, 0], dtype=torch.int32, device=DEV)
    mask = tree_mask(b, t, 1)
    mask[:, 3] = False
    mask[0, 66:] = False
    mask[2] = False
    got = run(q, kc, vc, lengths, k, v, mask, impl)
    check(got, reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))
    assert (got[0][2] == 0).all() and (got[1][0, :, 3] == -math.inf).all() and got[1][1].isfinite().all()


@pytest.mark.parametrize('dtype, impl', FAMILIES)
@pytest.mark.parametrize('garbage', [math.nan, math.inf, -math.inf, 3e38])
def test_what_nobody_sees_leaves_no_trace(dtype, impl, garbage):
    b, t = 2, 12
    q, kc, vc, k, v = problem(b, t, 8, 2, 128, 400, dtype, seed=4)
    lengths = torch.tensor([333, 64], dtype=torch.int32, device=DEV)
    mask = tree_mask(b, t, 9)
    mask[:, :, 5] = False             # a drafted row that no token sees
    clean = run(q, kc, vc, lengths, k, v, mask, impl)
    kc, vc, k, v = kc.clone(), vc.clone(), k.clone(), v.clone()
    for s, n in enumerate((333, 64)):
        kc[s, :, n:], vc[s, :, n:] = garbage, garbage
    k[:, :, 5], v[:, :, 5] = garbage, garbage
    got = run(q, kc, vc, lengths, k, v, mask, impl)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    # a drafted value that some see: theirs alone is not finite, and only in its column
    if not math.isinf(garbage) or garbage > 0:
        v[0, 1, 2, 17] = garbage
        got = run(q, kc, vc, lengths, k, v, mask, impl)
        hit = torch.zeros_like(clean[0], dtype=torch.bool)
        hit[0, 4:, :, 17] = mask[0, :, 2]
        assert torch.equal(got[0][~hit], clean[0][~hit])
        if math.isfinite(garbage):
            assert got[0][hit].isfinite().all()
        else:
            assert (~got[0][hit].isfinite()).all()


@pytest.mark.parametrize('dtype, impl', FAMILIES)
def test_large_logits(dtype, impl):
    """Queries thirty times as large: maxima that move by hundreds from block to block."""
    q, kc, vc, k, v = problem(2, 5, 8, 2, 64, 900, dtype, seed=8, scale=1.0)
    q = (q.float() * 30).to(dtype)
    kc = (kc.float() * torch.linspace(0.1, 3, 900, device=DEV)[:, None]).to(dtype)
    check(run(q, kc, vc, [900, 900][0], k, v, None, impl), reference(q, kc, vc, [900, 900], k, v, None, weights_rounded=rounded(dtype, impl)))
    check(run(q, kc, vc, 900, k, v, None, impl, scale=0.01), reference(q, kc, vc, [900, 900], k, v, None, scale=0.01, weights_rounded=rounded(dtype, impl)))


@pytest.mark.parametrize('dtype, impl', FAMILIES)
def test_strides(dtype, impl):
    """Caches as rows of all heads, of a larger buffer, shared by all sequences or heads, and on odd boundaries."""
    b, t, hq, hkv, d, n = 3, 4, 8, 2, 64, 300
    q, kc, vc, k, v = problem(b, t, hq, hkv, d, n, dtype, seed=5)
    lengths = torch.tensor([300, 77, 200], dtype=torch.int32, device=DEV)
    mask = tree_mask(b, t, 2)
    rows = randn((b, n + 9, 2 * hkv, d), 6, dtype)[:, 4:4 + n]
    odd = randn((b, hkv, n, d + 3), 7, dtype)[..., 1:1 + d]
    shared, one = randn((1, hkv, n, d), 8, dtype).expand(b, -1, -1, -1), randn((b, 1, n, d), 9, dtype).expand(-1, hkv, -1, -1)
    for kk, vv in ((rows[:, :, :hkv].transpose(1, 2), rows[:, :, hkv:].transpose(1, 2)), (shared, one), (one, shared), (odd, kc)):
        check(run(q, kk, vv, lengths, k, v, mask, 'auto' if kk is odd and impl != 'simt' else impl),
              reference(q, kk, vv, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))
    wide = torch.zeros(b, t, t + 5, dtype=torch.bool, device=DEV)
    wide[:, :, :t] = mask
    check(run(q, kc, vc, lengths, k, v, wide[:, :, :t], impl), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))
    check(run(q, kc, vc, lengths, k, v, mask.transpose(1, 2).contiguous().transpose(1, 2), impl), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=rounded(dtype, impl)))


def test_an_empty_cache_and_empty_calls():
    for dtype in (torch.float32, torch.bfloat16):
        q, kc, vc, k, v = problem(2, 5, 4, 2, 64, 0, dtype)
        check(run(q, kc, vc, None, k, v), reference(q, kc, vc, [0, 0], k, v, None, weights_rounded=dtype == torch.bfloat16))
        q, kc, vc, k, v = problem(2, 0, 4, 2, 64, 10, dtype)
        assert run(q, kc, vc, None, k, v)[0].shape == (2, 4, 0, 64)
        q, kc, vc, k, v = problem(0, 3, 4, 2, 64, 10, dtype)
        assert run(q, kc, vc, None, k, v)[1].shape == (0, 4, 3)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Rows of a cache whose last element lies behind 2^32 elements (bf16) or bytes (fp32) of its start."""
    d, hkv = 128, 4
    capacity = (1 << 32) // (hkv * d) + 1000 if dtype == torch.bfloat16 else (1 << 30) // (hkv * d) + 1000
    kc = torch.zeros(1, capacity, hkv, d, device=DEV, dtype=dtype)
    kc[:, -900:] = randn((1, 900, hkv, d), 1, dtype)
    kc = kc.transpose(1, 2)
    q, _, _, k, v = problem(1, 2, 8, hkv, d, 1, dtype)
    # all keys but the last 900 are zero: their logits are 0, and so are their values
    got = run((q.float() * 8).to(dtype), kc, kc, None, k, v)
    near = kc[:, :, -900:]
    qs = (q.float() * 8).to(dtype).double().view(1, hkv, 2, 2, d)
    keys, vals = torch.cat((near, k), 2).double(), torch.cat((near, v), 2).double()
    logits = torch.einsum('bkgtd,bknd->bkgtn', qs, keys) * d ** -0.5
    logits[..., 0, 901] = -math.inf
    lse = torch.logsumexp(torch.cat((logits, torch.full((1, hkv, 2, 2, 1), math.log(capacity - 900), device=DEV, dtype=torch.float64)), -1), -1)
    out = torch.einsum('bkgtn,bknd->bkgtd', torch.exp(logits - lse[..., None]), vals).reshape(1, 8, 2, d)
    # sums of some 10^7 equal terms, pairwise in threads of 10^5: 10^5 * 2^-24
    tol = 2e-2 if dtype == torch.bfloat16 else 1e-2
    assert (got[1].double() - lse.reshape(1, 8, 2)).abs().max() <= 1e-2
    assert (got[0].double() - out).abs().max() <= tol * out.abs().max()


def test_a_verification_step():
    """The operators together as a serving loop uses them: drafted tokens are normalised and rotated at length + depth, the
    tree attends cache and drafts; then the accepted path, appended to the cache token by token, gives the same rows."""
    b, t, hq, hkv, d, capacity = 2, 10, 8, 2, 64, 300
    dtype = torch.bfloat16
    rotary = RotaryFrequencies(d, layout='half', scaling='yarn', factor=4., original_length=128)
    w = [1 + randn((d,), i, dtype, 0.2) for i in (1, 2)]
    lengths = torch.tensor([250, 31], dtype=torch.int32, device=DEV)
    kc, vc = randn((b, hkv, capacity, d), 3, dtype), randn((b, hkv, capacity, d), 4, dtype)
    qkv = randn((b, t, hq + 2 * hkv, d), 5, dtype).transpose(1, 2)
    mask = tree_mask(b, t, 6)
    depth = mask.sum(-1) - 1
    q, k = norm_rotate_heads(qkv[:, :hq], qkv[:, hq:hq + hkv], *w, rotary, lengths[:, None].long() + depth)
    v = qkv[:, hq + hkv:]
    out, lse = run(q, kc, vc, lengths, k, v, mask)
    check((out, lse), reference(q, kc, vc, lengths, k, v, mask, weights_rounded=True))
    for s in range(b):
        leaf = int(depth[s].argmax())
        path = mask[s, leaf].nonzero()[:, 0]
        n = int(lengths[s])
        one_k, one_v = kc[s:s + 1].clone(), vc[s:s + 1].clone()
        for i, token in enumerate(path.tolist()):
            row = qkv[s:s + 1, :, token:token + 1]
            q1, k1 = norm_rotate_heads(row[:, :hq], row[:, hq:hq + hkv], *w, rotary, offset=n + i)
            assert torch.equal(q1[0, :, 0], q[s, :, token]) and torch.equal(k1[0, :, 0], k[s, :, token])
            got = run(q1, one_k, one_v, n + i, k1, row[:, hq + hkv:])
            ref = reference(q1, one_k, one_v, [n + i], k1, row[:, hq + hkv:], None, weights_rounded=True)
            check(got, ref)
            # both are within their bounds of the same value
            bound = 2 * (ref[2] + 2.0 ** -8 * (ref[0].abs() + ref[2]))
            assert ((got[0].double() - out[s:s + 1, :, token:token + 1].double()).abs() <= bound).all()
            one_k[:, :, n + i], one_v[:, :, n + i] = k1[:, :, 0], row[:, hq + hkv:, 0]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_streams_graphs_and_repeats(dtype):
    """The same call gives the same bits; captured with lengths that change between replays, two graphs in turn."""
    b, t = 3, 6
    q, kc, vc, k, v = problem(b, t, 8, 2, 64, 1500, dtype, seed=2)
    mask = tree_mask(b, t, 3)
    lengths = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([1400, 3, 700], [10, 1500, 0])]
    expected = [run(q, kc, vc, n, k, v, mask) for n in lengths]
    for n, e in zip(lengths, expected):
        for a, r in zip(run(q, kc, vc, n, k, v, mask), e):
            assert torch.equal(a, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree_attend(q, kc, vc, lengths[0], k, v, mask, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], expected[0][0]) and torch.equal(got[1], expected[0][1])
    held, graphs, outs = [torch.zeros_like(lengths[0]) for _ in range(2)], [], []
    for n in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(tree_attend(q, kc, vc, n, k, v, mask, return_lse=True))
        graphs.append(g)
    for i, j in ((0, 0), (1, 1), (0, 1), (1, 0)):
        held[i].copy_(lengths[j])
        graphs[i].replay()
        assert torch.equal(outs[i][0], expected[j][0]) and torch.equal(outs[i][1], expected[j][1])
    ops.check_device_status()


def test_gradients_are_refused_not_dropped():
    args = problem(1, 3, 4, 2, 64, 10, torch.bfloat16)
    expected = tree_attend(*args[:3], None, *args[3:])
    for i in range(5):
        given = [x.clone().requires_grad_(j == i) for j, x in enumerate(args)]
        with pytest.raises(L.NsaError, match='no gradient'):
            tree_attend(*given[:3], None, *given[3:])
        with torch.no_grad():
            assert torch.equal(tree_attend(*given[:3], None, *given[3:]), expected)


def test_refusals_on_the_device():
    q, kc, vc, k, v = problem(2, 3, 4, 2, 64, 10, torch.float32)
    ok = torch.zeros(2, dtype=torch.int32, device=DEV)
    cases = [
        (lambda: tree_attend(q.half(), kc.half(), vc.half(), None, k.half(), v.half()), 'dtype'),
        (lambda: tree_attend(q, kc.bfloat16(), vc, None, k, v), 'device and type'),
        (lambda: tree_attend(q, kc, vc[:, :, :9], None, k, v), 'cached keys'),
        (lambda: tree_attend(q, kc, vc, None, k, v[:, :, :2]), 'drafted tokens'),
        (lambda: tree_attend(q[:, :3], kc, vc, None, k, v), 'multiple'),
        (lambda: tree_attend(q[0], kc, vc, None, k, v), 'batch, heads'),
        (lambda: tree_attend(q, kc, vc, ok[:1], k, v), 'lengths'),
        (lambda: tree_attend(q, kc, vc, ok.float(), k, v), 'lengths'),
        (lambda: tree_attend(q, kc, vc, ok.cpu(), k, v), 'CUDA tensors only'),
        (lambda: tree_attend(q, kc, vc, 11, k, v), 'capacity'),
        (lambda: tree_attend(q, kc, vc, ok, k, v, torch.ones(3, 2, dtype=torch.bool, device=DEV)), 'mask must be'),
        (lambda: tree_attend(q, kc, vc, ok, k, v, torch.ones(3, 3, device=DEV)), 'mask must be'),
        (lambda: tree_attend(q, kc, vc, ok, k, v, impl='sm100'), 'tensor-core'),
        (lambda: tree_attend(q[..., :60], kc[..., :60], vc[..., :60], ok, k[..., :60], v[..., :60]), 'dim_head'),
        (lambda: tree_attend(q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, ok, k, v), 'last axis'),
    ]
    for call, match in cases:
        with pytest.raises(L.NsaError, match=match):
            call()
