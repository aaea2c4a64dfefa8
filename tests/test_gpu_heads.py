"""Rotation of heads by positions, with and without their norm, against the formulas in 64 bits: layouts, parts of a head,
scalings, strides that allow only narrow vectors, weights per head, gradients, far positions.

Bounds, element by element.  A sine or cosine is off by at most pi 2^-25 (the phase as fp32) + 2^-23 (two units of sincospif)
< 4 * 2^-24, twice the magnitude's and the products' and the sum's rounding: 8 * 2^-24 of |u| + |v| of the pair.  The norm adds
the sum of squares (at most 24 additions in a row, halved by the root), two units of rsqrtf and two products: 24 * 2^-24 more.
Behind them one rounding to the type, eps / 2 of the value."""
import itertools

import pytest
import torch

from native_sparse_attention_pytorch_b200 import RMSNorm, RotaryFrequencies, norm_rotate_heads, rotate_heads  # noqa: F401
from native_sparse_attention_pytorch_b200 import _lib as L
from native_sparse_attention_pytorch_b200.rotary import RotaryEmbedding

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def angles(rotary, positions):
    f = torch.tensor(rotary.frequencies, dtype=torch.float64, device=DEV)
    a = positions.double()[..., None] * f
    return a if a.dim() == 2 else a[:, None]


def turned(x, rotary, angle, inverse=False, absolute=False):
    """The rotation in 64 bits; `absolute`: |u| + |v| of every pair in both places instead, times the magnitude."""
    r, x = rotary.rotary_dim, x.double()
    co, si = angle.cos() * rotary.magnitude, angle.sin() * rotary.magnitude
    u, v = (x[..., :r // 2], x[..., r // 2:r]) if rotary.layout == 'half' else (x[..., 0:r:2], x[..., 1:r:2])
    if inverse:
        si = -si
    a, z = u * co - v * si, v * co + u * si
    if absolute:
        a = z = (u.abs() + v.abs()) * rotary.magnitude + 0 * co
    rest = x[..., r:].abs() if absolute else x[..., r:]
    if rotary.layout == 'half':
        return torch.cat((a, z, rest), dim=-1)
    return torch.cat((torch.stack((a, z), dim=-1).flatten(-2), rest), dim=-1)


def assert_within(got, ref, bound, what):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if ref.numel() == 0:
        return
    half = torch.finfo(got.dtype).eps / 2
    excess = (got.double() - ref).abs() - (bound + half * (ref.abs() + bound))
    worst = excess.max().item()
    assert worst <= 0, f'{what}: {worst:.3e} beyond the bound'


def wide_weight(w):
    return w.double()[:, None] if w.dim() == 2 else w.double()


def check_forward(x, w, y, rotary, angle, eps, what):
    n = x.double()
    if w is not None:
        n = n * (n.square().mean(-1, keepdim=True) + eps).rsqrt() * wide_weight(w)
    grow = 8 if w is None else 32
    assert_within(y, turned(n, rotary, angle), grow * U * turned(n, rotary, angle, absolute=True), what)


def check_backward(x, w, dy, dx, dw, rotary, angle, eps, what):
    g, size = turned(dy, rotary, angle, inverse=True), 8 * U * turned(dy, rotary, angle, absolute=True)
    if w is None:
        return assert_within(dx, g, size, what + ' dx')
    n = x.double()
    rstd = (n.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit, wide = n * rstd, wide_weight(w)
    back = g * wide
    ref = rstd * (back - unit * (back * unit).mean(-1, keepdim=True))
    # each of the two terms is off by its factors' errors (24 + 8 for the pair, 64 for the mean's products and sum)
    off = rstd * (32 * U * turned(dy, rotary, angle, absolute=True) * wide.abs() + 96 * U * unit.abs() * (turned(dy, rotary, angle, absolute=True) * wide.abs() * unit.abs()).mean(-1, keepdim=True))
    assert_within(dx, ref, off, what + ' dx')
    dims = (0, 2) if w.dim() == 2 else (0, 1, 2)
    # at most 256 additions in a row (a thread's rows, lanes, warps, blocks) at these sizes
    assert_within(dw, (g * unit).sum(dims), (256 + 32) * U * (turned(dy, rotary, angle, absolute=True) * unit.abs()).sum(dims), what + ' dw')


def run_case(b, n, hq, hk, d, rotary, dtype, weights=None, wdtype=None, fused=True, positions=None, offset=0, eps=1e-6, seed=0, grad=True):
    if fused:       # views of a projection's rows
        rows = randn((b, n, (hq + 2 * hk) * d), seed, dtype).view(b, n, hq + 2 * hk, d).transpose(1, 2)
        q, k = rows[:, :hq].detach(), rows[:, hq:hq + hk].detach()
    else:
        q, k = randn((b, hq, n, d), seed, dtype), randn((b, hk, n, d), seed + 1, dtype)
    wq = wk = None
    if weights:
        wq, wk = (1 + randn((h, d) if weights == 'heads' else (d,), seed + 2 + i, wdtype or dtype, 0.3) for i, h in enumerate((hq, hk)))
        wq, wk = wq.detach().requires_grad_(grad), wk.detach().requires_grad_(grad)
    q, k = q.requires_grad_(grad), k.requires_grad_(grad)
    if weights:
        y, z = norm_rotate_heads(q, k, wq, wk, rotary, positions, offset, eps=eps)
    else:
        y, z = rotate_heads(q, k, rotary, positions, offset)
    assert y.is_contiguous() and z.is_contiguous() and y.dtype == z.dtype == dtype
    angle = angles(rotary, (torch.arange(n, device=DEV) if positions is None else positions) + offset)
    check_forward(q.detach(), wq, y.detach(), rotary, angle, eps, 'q')
    check_forward(k.detach(), wk, z.detach(), rotary, angle, eps, 'k')
    if not grad:
        return
    dy, dz = randn(y.shape, seed + 5, dtype), randn(z.shape, seed + 6, dtype)
    leaves = (q, k, wq, wk) if weights else (q, k)
    g = torch.autograd.grad((y, z), leaves, (dy, dz))
    for x, dx in zip((q, k), g):
        assert dx.dtype == dtype
        if x.numel() and not x.is_contiguous():
            assert dx.transpose(1, 2).is_contiguous()        # in the memory order of the projection
    check_backward(q.detach(), wq, dy, g[0], g[2] if weights else None, rotary, angle, eps, 'q')
    check_backward(k.detach(), wk, dz, g[1], g[3] if weights else None, rotary, angle, eps, 'k')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('layout', ['interleaved', 'half'])
@pytest.mark.parametrize('d, r', [(64, 64), (64, 32), (128, 128), (128, 48), (80, 40), (256, 256), (256, 2), (96, 6), (34, 34), (36, 20), (2, 2), (250, 126), (128, 20), (80, 20)])
@pytest.mark.parametrize('weights', [None, 'shared', 'heads'])
def test_layouts_and_parts(dtype, layout, d, r, weights):
    run_case(2, 13, 6, 2, d, RotaryFrequencies(d, r, layout=layout), dtype, weights)


@pytest.mark.parametrize('b, n, hq, hk', [(1, 1, 1, 1), (8, 1, 32, 4), (1, 517, 8, 8), (3, 129, 12, 4), (1, 2000, 9, 1)])
@pytest.mark.parametrize('weights', [None, 'shared', 'heads'])
@pytest.mark.parametrize('fused', [False, True])
def test_sizes(b, n, hq, hk, weights, fused):
    run_case(b, n, hq, hk, 64, RotaryFrequencies(64, layout='half'), torch.bfloat16, weights, fused=fused, wdtype=torch.float32)


@pytest.mark.parametrize('scaling', [dict(scaling='linear', factor=4.), dict(scaling='ntk', factor=8.), dict(scaling='yarn', factor=16., original_length=2048)])
@pytest.mark.parametrize('layout', ['interleaved', 'half'])
def test_scalings_at_far_positions(scaling, layout):
    rotary = RotaryFrequencies(64, layout=layout, **scaling)
    positions = torch.randint(0, 1 << 20, (3, 17), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    for p in (positions, positions.int(), positions[:1], positions[0]):
        run_case(3, 17, 4, 2, 64, rotary, torch.float32, positions=p)
    run_case(3, 17, 4, 2, 64, rotary, torch.float32, 'shared', positions=positions, offset=(1 << 24) + 1)
    run_case(3, 17, 4, 2, 64, rotary, torch.float32, offset=-100)


def test_positions_past_32_bits():
    # angles in 64-bit floating point are themselves off by 2^-53 of a number up to 2^33: 10^-6
    rotary = RotaryFrequencies(64)
    x = randn((1, 2, 4, 64), 1)
    p = torch.tensor([1 << 32, (1 << 32) + 1, (1 << 33) - 1, 5], device=DEV)
    y, _ = rotate_heads(x, None, rotary, p)
    angle = angles(rotary, p)
    assert_within(y, turned(x, rotary, angle), (8 * U + 2.0 ** -20) * turned(x, rotary, angle, absolute=True), 'far')


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('weights', [None, 'shared'])
@pytest.mark.parametrize('pad, shift', [(1, 0), (2, 2), (4, 4), (0, 1), (3, 5)])
def test_strides_and_boundaries(dtype, weights, pad, shift):
    """Rows that start on narrow boundaries: a slice of rows of d + pad elements, `shift` into the buffer."""
    b, h, n, d = 2, 3, 5, 64
    rotary = RotaryFrequencies(d, 32, layout='half')
    flat = randn((shift + b * h * n * (d + pad),), 3, dtype)
    x = flat[shift:].view(b, h, n, d + pad)[..., :d]
    w = 1 + randn((d,), 4, dtype, 0.3)
    x.requires_grad_()
    y = (norm_rotate_heads(x, None, w, None, rotary) if weights else rotate_heads(x, None, rotary))[0]
    dy = randn((b, n, h, d + pad), 5, dtype)[..., :d].transpose(1, 2)
    angle = angles(rotary, torch.arange(n, device=DEV))
    eps = torch.finfo(torch.float32).eps
    check_forward(x.detach(), w if weights else None, y.detach(), rotary, angle, eps, 'x')
    dx, = torch.autograd.grad(y, x, dy)
    if not weights:
        check_backward(x.detach(), None, dy, dx, None, rotary, angle, eps, 'x')
    last = randn((b, h, d, n), 6, dtype).transpose(2, 3)      # the last axis is not contiguous
    got = (norm_rotate_heads(last, None, w, None, rotary) if weights else rotate_heads(last, None, rotary))[0]
    check_forward(last, w if weights else None, got, rotary, angle, eps, 'transposed')


def test_the_interleaved_whole_head_is_what_the_layer_rotates_by():
    x = randn((2, 4, 33, 64), 7)
    ours, layer = rotate_heads(x, None, RotaryFrequencies(64), offset=5)[0], RotaryEmbedding(64).to(DEV).rotate_queries_or_keys(x, offset=5)
    # the layer's angles are fp32 products of positions up to 37: off by 37 * 2^-24, on top of 8 units of either side
    bound = (16 + 2 * 37) * U * turned(x, RotaryFrequencies(64), angles(RotaryFrequencies(64), torch.arange(5, 38, device=DEV)), absolute=True)
    assert ((ours - layer).abs() <= bound).all()


def test_gradients_are_those_of_differences():
    """Central differences in 64 bits of the formula, at a few elements, against the kernels' gradient."""
    rotary, eps = RotaryFrequencies(16, 8, layout='half'), 1e-5
    x, w, dy = randn((1, 2, 3, 16), 1), 1 + randn((2, 16), 2, scale=0.3), randn((1, 2, 3, 16), 3)
    angle = angles(rotary, torch.arange(3, device=DEV))

    def loss(x, w):
        n = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w[:, None]
        return (turned(n, rotary, angle) * dy.double()).sum()
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = norm_rotate_heads(xg, None, wg, None, rotary, eps=eps)[0]
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    for t, grad, at in ((x, dx, [(0, 0, 0, 0), (0, 1, 2, 15), (0, 1, 1, 5)]), (w, dw, [(0, 0), (1, 7), (1, 12)])):
        for i in at:
            step = torch.zeros_like(t, dtype=torch.float64)
            step[i] = 1e-5
            a = [x.double(), w.double()]
            k = 0 if t is x else 1
            lo, hi = list(a), list(a)
            lo[k], hi[k] = a[k] - step, a[k] + step
            slope = ((loss(*hi) - loss(*lo)) / 2e-5).item()
            # differences: step^2 times third derivatives (10^-10 times a few) and 2^-52 |loss| / step; the kernel: fp32
            assert abs(slope - grad[i].item()) <= 1e-5 * max(1.0, abs(slope)), (i, slope, grad[i].item())


def test_missing_gradients_and_repeats():
    rotary = RotaryFrequencies(64)
    q, k, w = randn((2, 4, 9, 64), 1).requires_grad_(), randn((2, 2, 9, 64), 2).requires_grad_(), randn((64,), 3).requires_grad_()
    y, z = norm_rotate_heads(q, k, w, w, rotary)                 # one weight for both: its gradient is the sum
    both = torch.autograd.grad((y, z), w, (torch.ones_like(y), torch.ones_like(z)), retain_graph=True)[0]
    one = torch.autograd.grad(y, w, torch.ones_like(y), retain_graph=True)[0]
    two = torch.autograd.grad(z, w, torch.ones_like(z), retain_graph=True)[0]
    assert torch.equal(both, one + two)
    assert torch.autograd.grad(y, k, torch.ones_like(y), allow_unused=True, retain_graph=True)[0] is None
    again = torch.autograd.grad((y, z), (q, k, w), (torch.ones_like(y), torch.ones_like(z)), retain_graph=True)
    for a, b in zip(again, torch.autograd.grad((y, z), (q, k, w), (torch.ones_like(y), torch.ones_like(z)))):
        assert torch.equal(a, b)
    y, z = rotate_heads(q, k, rotary)
    (y.sum() + 0 * z.detach().sum()).backward()                  # a gradient of stride 0, and one that never arrives
    assert k.grad is None
    check_backward(None, None, torch.ones_like(y), q.grad, None, rotary, angles(rotary, torch.arange(9, device=DEV)), 0, 'q')
    y, _ = rotate_heads(q, k, rotary)
    g, = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match='differentiate twice'):
        g.sum().backward()


def test_broadcast_inputs_get_the_sum():
    rotary = RotaryFrequencies(64, layout='half')
    one = randn((1, 1, 7, 64), 1).requires_grad_()
    y, _ = rotate_heads(one.expand(3, 5, 7, 64), None, rotary)
    dy = randn(y.shape, 2)
    dx, = torch.autograd.grad(y, one, dy)
    ref = turned(dy, rotary, angles(rotary, torch.arange(7, device=DEV)), inverse=True).sum((0, 1), keepdim=True)
    assert (dx.double() - ref).abs().max() <= 64 * U * dy.abs().sum((0, 1)).max()


def test_outputs_given_and_in_place():
    rotary = RotaryFrequencies(64, 32, layout='half')
    q, k = randn((2, 4, 5, 64), 1, torch.bfloat16), randn((2, 2, 5, 64), 2, torch.bfloat16)
    y, z = rotate_heads(q, k, rotary, offset=11)
    cache = torch.full((2, 2, 40, 64), 7., device=DEV, dtype=torch.bfloat16)
    got = rotate_heads(q, k, rotary, offset=11, out=(None, cache[:, :, 11:16]))
    assert torch.equal(got[0], y) and torch.equal(cache[:, :, 11:16], z) and got[1].data_ptr() == cache[:, :, 11:].data_ptr()
    assert (cache[:, :, :11] == 7).all() and (cache[:, :, 16:] == 7).all()
    w = 1 + randn((64,), 3, torch.bfloat16, 0.3)
    y, z = norm_rotate_heads(q, k, w, w, rotary)
    norm_rotate_heads(q, k, w, w, rotary, out=(q, k))            # in place
    assert torch.equal(q, y) and torch.equal(k, z)


def test_not_finite_values_stay_in_their_pair_or_row():
    rotary = RotaryFrequencies(64, 32, layout='half')
    x = randn((1, 2, 4, 64), 1)
    clean, _ = rotate_heads(x, None, rotary)
    bad = x.clone()
    bad[0, 0, 1, 3], bad[0, 1, 2, 40] = float('nan'), float('inf')     # a rotated feature, one that passes
    y, _ = rotate_heads(bad, None, rotary)
    assert y[0, 0, 1, [3, 19]].isnan().all() and y[0, 1, 2, 40] == float('inf')
    y[0, 0, 1, [3, 19]], y[0, 1, 2, 40] = clean[0, 0, 1, [3, 19]], clean[0, 1, 2, 40]
    assert torch.equal(y, clean)
    w = torch.ones(64, device=DEV)
    clean, y = norm_rotate_heads(x, None, w, None, rotary)[0], norm_rotate_heads(bad, None, w, None, rotary)[0]
    assert y[0, 0, 1].isnan().all()
    others = torch.ones(2, 4, dtype=torch.bool, device=DEV)
    others[0, 1] = others[1, 2] = False
    assert torch.equal(y[0][others], clean[0][others])


@pytest.mark.parametrize('b, n', [(0, 5), (3, 0)])
def test_nothing_to_do(b, n):
    rotary = RotaryFrequencies(64)
    q, w = torch.empty(b, 4, n, 64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True)
    y, _ = norm_rotate_heads(q, None, w, None, rotary)
    dq, dw = torch.autograd.grad(y, (q, w), torch.empty_like(y))
    assert y.shape == q.shape and dq.shape == q.shape and (dw == 0).all()


def test_streams_and_graphs():
    """On a side stream, and captured: a graph replayed on new inputs, two graphs of one operator replayed in turn."""
    rotary = RotaryFrequencies(64, layout='half')
    w = (1 + randn((64,), 9, scale=0.3)).requires_grad_()
    x = [randn((2, 4, 50, 64), s) for s in (1, 2)]
    pos = torch.arange(50, device=DEV)

    def step(x, pos):
        leaf = x.detach().requires_grad_()
        y, _ = norm_rotate_heads(leaf, None, w, None, rotary, pos)
        return (y.detach(), *torch.autograd.grad(y, (leaf, w), y.detach()))
    expected = [step(t, pos + 3) for t in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x[0], pos + 3)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, expected[0]):
        assert torch.equal(a, b)
    held = [(torch.zeros_like(x[0]), torch.zeros_like(pos)) for _ in range(2)]
    graphs, outs = [], []
    for t, p in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(t, p))
        graphs.append(g)
    for order in itertools.permutations(range(2)):
        for i in order:
            held[i][0].copy_(x[i])
            held[i][1].copy_(pos + 3)
        for i in order:
            graphs[i].replay()
        for i in order:
            for a, b in zip(outs[i], expected[i]):
                assert torch.equal(a, b)


def test_a_capture_beside_a_living_eager_graph():
    """A forward and backward recorded while an eager graph of the same tensors is still held.  (Leaves of their own in the
    recording: PyTorch itself keeps the stream of a leaf's first graph as long as that lives, and refuses the capture.)"""
    rotary = RotaryFrequencies(64)
    q, w = randn((2, 4, 9, 64), 1).requires_grad_(), (1 + randn((64,), 2, scale=0.3)).requires_grad_()
    held, _ = norm_rotate_heads(q, None, w, None, rotary)
    expected = torch.autograd.grad(held, (q, w), held.detach(), retain_graph=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        leaves = q.detach().requires_grad_(), w.detach().requires_grad_()
        y, _ = norm_rotate_heads(leaves[0], None, leaves[1], None, rotary)
        got = torch.autograd.grad(y, leaves, y.detach())
    g.replay()
    for a, b in zip(got, expected):
        assert torch.equal(a, b)


def test_refusals_on_the_device():
    rotary = RotaryFrequencies(64)
    q, k, w = randn((2, 4, 5, 64), 1), randn((2, 2, 5, 64), 2), torch.ones(64, device=DEV)
    cases = [
        (lambda: rotate_heads(q.half(), None, rotary), 'dtype'),
        (lambda: rotate_heads(q[..., :32], None, rotary), 'heads of 64'),
        (lambda: rotate_heads(q, k.bfloat16(), rotary), 'device and type'),
        (lambda: rotate_heads(q, k[:, :, :4], rotary), 'share batch'),
        (lambda: rotate_heads(q[0], None, rotary), 'batch, heads, seq'),
        (lambda: rotate_heads(q, None, rotary, torch.zeros(5, device=DEV)), 'int64 or int32'),
        (lambda: rotate_heads(q, None, rotary, torch.zeros(4, device=DEV, dtype=torch.long)), 'positions must be'),
        (lambda: rotate_heads(q, None, rotary, torch.zeros(3, 5, device=DEV, dtype=torch.long)), 'positions must be'),
        (lambda: rotate_heads(q, None, rotary, torch.zeros(5, dtype=torch.long)), 'CUDA tensors only'),
        (lambda: rotate_heads(q, None, rotary, out=(q[:, :2], None)), 'an output'),
        (lambda: rotate_heads(q.clone().requires_grad_(), None, rotary, out=(q, None)), 'gradients'),
        (lambda: norm_rotate_heads(q, k, w, None, rotary), 'weight'),
        (lambda: norm_rotate_heads(q, k, w, w[:32], rotary), 'weight'),
        (lambda: norm_rotate_heads(q, k, w, torch.ones(2, 64, device=DEV), rotary), 'one form'),
        (lambda: norm_rotate_heads(q, k, w.bfloat16(), w.bfloat16(), rotary), "tensor's type"),
    ]
    for call, match in cases:
        with pytest.raises(L.NsaError, match=match):
            call()


def test_outputs_that_overlap_are_refused():
    rotary, w = RotaryFrequencies(64), torch.ones(64, device=DEV)
    q, k = randn((2, 3, 5, 64), 1), randn((2, 3, 5, 64), 2)
    flat = randn((2 * 3 * 5 * 64 + 64,), 3)
    cases = [
        (lambda: rotate_heads(q, k, rotary, out=(k, None)), "overlap the other"),
        (lambda: rotate_heads(q, k, rotary, out=(k, q)), "overlap the other"),
        (lambda: rotate_heads(q, k, rotary, out=(flat[64:].view_as(q), flat[:-64].view_as(q))), "overlap the other"),
        (lambda: rotate_heads(flat[64:].view_as(q), None, rotary, out=(flat[:-64].view_as(q), None)), 'must not overlap it'),
        (lambda: rotate_heads(q, None, rotary, out=(q[:, :1].expand(2, 3, 5, 64), None)), 'broadcast'),
        (lambda: norm_rotate_heads(q, None, w, None, rotary, out=(flat[64:].view_as(q).requires_grad_(), None)), 'wants gradients'),
    ]
    before = q.clone(), k.clone(), flat.clone()
    for call, match in cases:
        with pytest.raises(L.NsaError, match=match):
            call()
    flat = flat.detach()
    assert all(torch.equal(a, b) for a, b in zip(before, (q, k, flat)))
    qkv = randn((2, 5, 9, 64), 4).transpose(1, 2)          # one projection's heads, side by side, each in its own place
    a, b = qkv[:, :6], qkv[:, 6:8]
    y, z = rotate_heads(a.contiguous(), b.contiguous(), rotary)
    rotate_heads(a, b, rotary, out=(a, b))
    assert torch.equal(a, y) and torch.equal(b, z)


def test_what_a_backward_pass_needs_is_not_overwritten_unnoticed():
    rotary = RotaryFrequencies(64)
    x, at = randn((1, 2, 3, 64), 1).requires_grad_(), torch.tensor([4, 5, 9], device=DEV)
    y, _ = rotate_heads(x, None, rotary, at)
    at.add_(1)                                               # the positions of the next step, in the same tensor
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    e = x.exp()                                              # its backward pass needs its result
    with torch.no_grad():
        rotate_heads(e, None, rotary, out=(e, None))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        e.sum().backward()
    with torch.inference_mode():
        then = torch.tensor([4, 5, 9], device=DEV)
        t = torch.zeros(1, 2, 3, 64, device=DEV)
        rotate_heads(t, None, rotary, then, out=(t, None))
    y, _ = rotate_heads(x, None, rotary, then)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    ref = turned(torch.ones_like(y), rotary, angles(rotary, torch.tensor([4, 5, 9], device=DEV)), inverse=True)
    assert (dx.double() - ref).abs().max() <= 64 * U


def test_two_streams_at_once():
    rotary = RotaryFrequencies(128, layout='half')
    w = [(1 + randn((128,), i, torch.bfloat16, 0.2)).requires_grad_() for i in (1, 2)]
    xs = [randn((2, h, n, 128), 3 + n, torch.bfloat16) for h, n in ((8, 700), (4, 900))]

    def step(x):
        leaf = x.detach().requires_grad_()
        y, z = norm_rotate_heads(leaf, leaf, *w, rotary)
        return torch.autograd.grad((y, z), (leaf, *w), (y.detach(), z.detach()))
    expected = [step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(x))
    torch.cuda.synchronize()
    for g, e in zip(got, expected):
        for grads in g:
            for a, b in zip(grads, e):
                assert torch.equal(a, b)


@pytest.mark.parametrize('layout', ['interleaved', 'half'])
def test_weights_on_narrow_boundaries(layout):
    """fp32 weights beside bf16 rows, and bf16 ones, as views into a flat buffer of parameters."""
    rotary, x = RotaryFrequencies(64, layout=layout), randn((1, 3, 6, 64), 1, torch.bfloat16)
    angle = angles(rotary, torch.arange(6, device=DEV))
    for dtype in (torch.float32, torch.bfloat16):
        flat = 1 + randn((64 * 3 + 8,), 2, dtype, 0.3)
        for shift in (0, 1, 2, 4):
            for w in (flat[shift:shift + 64], flat[shift:shift + 192].view(3, 64)):
                y, _ = norm_rotate_heads(x, None, w, None, rotary)
                check_forward(x, w, y, rotary, angle, torch.finfo(torch.float32).eps, f'{dtype} {shift}')
