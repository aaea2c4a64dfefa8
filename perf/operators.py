"""Cases of the operators that prepare and attend drafted or prompted tokens: rotation of queries and keys by their
positions, normalisation of every head with the rotation in the same pass, and attention of a tree of drafted tokens over
a cache.  `run` computes a case in plain PyTorch, or through the package where `own` is set."""
import math

import numpy as np
import torch

own = False
DEV = 'cuda'
EPS = 1e-6
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def _rows(kind, name, batch, seq, heads, kv_heads, d, rotary_dim, layout, scaling, far, grad, dtype='bf16', weights='shared'):
    return dict(name=name, kind=kind, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, d=d, rotary_dim=rotary_dim,
                layout=layout, scaling=scaling, far=far, grad=grad, dtype=dtype, weights=weights)


def _tree(name, batch, tokens, heads, kv_heads, d, length, ragged, shape, dtype='bf16'):
    return dict(name=name, kind='tree', batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, d=d, length=length,
                ragged=ragged, shape=shape, dtype=dtype)


def listed():
    return [
        # the newest token of eight sequences, in a model whose context was stretched: latency alone
        _rows('rotate', 'rotate_token', 8, 1, 32, 4, 64, 64, 'half', 'yarn', 65536, False),
        # a long prompt (64 / 8 heads of 128), the largest forward
        _rows('rotate', 'rotate_prompt', 1, 65536, 64, 8, 128, 128, 'interleaved', 'none', 0, False),
        # a training step that rotates half of every head, forward and gradients
        _rows('rotate', 'rotate_train', 2, 16384, 16, 4, 64, 32, 'half', 'ntk', 0, True),
        # the newest token of sixteen sequences
        _rows('norm_rotate', 'norm_rotate_token', 16, 1, 16, 4, 128, 128, 'half', 'none', 32768, False),
        # a prompt of odd length, with positions stretched linearly
        _rows('norm_rotate', 'norm_rotate_prompt', 1, 16383, 64, 8, 128, 128, 'interleaved', 'linear', 0, False),
        # a training step, forward and gradients, the weights' among them
        _rows('norm_rotate', 'norm_rotate_train', 4, 8192, 32, 4, 64, 64, 'half', 'none', 0, True),
        # 32-bit training of a small model with a weight row for every head, rotary part that is no power of two
        _rows('norm_rotate', 'norm_rotate_train_fp32', 3, 1021, 8, 2, 80, 40, 'interleaved', 'none', 0, True, dtype='fp32', weights='heads'),
        # one token of one sequence over an ordinary cache: latency alone
        _tree('tree_token', 1, 1, 32, 4, 64, 4096, False, 'chain'),
        # one token each of a serving batch over long caches of different lengths: the caches' bytes
        _tree('tree_token_batch', 32, 1, 64, 8, 128, 16384, True, 'chain'),
        # a small tree of drafted tokens for every sequence of a batch
        _tree('tree_verify', 8, 16, 16, 4, 64, 16384, True, 'tree'),
        # a wide tree over the long-context configuration: the tensor cores' arithmetic
        _tree('tree_wide', 4, 64, 64, 8, 128, 65536, True, 'tree'),
        # 32-bit values, odd sizes
        _tree('tree_fp32', 2, 7, 8, 2, 64, 1531, True, 'tree', dtype='fp32'),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(['rotate', 'norm_rotate', 'tree', 'tree'])
    dtype = rng.choice(['bf16', 'bf16', 'bf16', 'fp32'])
    heads, kv = rng.choice([(8, 2), (16, 4), (32, 4), (64, 8), (16, 2), (8, 8), (12, 4), (8, 1)])
    if kind == 'tree':
        d = rng.choice([64, 64, 128, 128, 32, 80])
        batch, tokens = _spread(rng, 1, 16), rng.choice([1, _spread(rng, 2, 16), _spread(rng, 16, 64)])
        # no more than the wide tree's arithmetic nor the batch's bytes; 32-bit values at the sizes of tests and small models
        most = min(65536, int(2.5e8 / (batch * kv * d)), int(8e10 / (batch * heads * tokens * d)) if dtype == 'bf16' else 8192)
        return _tree('', batch, tokens, heads, kv, d, _spread(rng, 16, max(16, most)), rng.random() < 0.7, rng.choice(['tree', 'tree', 'chain']), dtype)
    d = rng.choice([64, 64, 128, 128, 32, 80, 96, 256])
    part = rng.choice([d, d, d // 2, d // 4 * 2])
    layout, scaling, grad = rng.choice(['interleaved', 'half']), rng.choice(['none', 'linear', 'ntk', 'yarn']), rng.random() < 0.5
    weights = rng.choice(['shared', 'shared', 'heads'])
    if rng.random() < 0.25:
        return _rows(kind, '', _spread(rng, 1, 128), _spread(rng, 1, 8), heads, kv, d, part, layout, scaling, _spread(rng, 64, 1 << 20), False, dtype, weights)
    batch = _spread(rng, 1, 8)
    most = max(2, min(65536, int((6e7 if grad else 1.5e8) / (batch * (heads + kv) * d))))
    return _rows(kind, '', batch, _spread(rng, 2, most), heads, kv, d, part, layout, scaling, 0, grad, dtype, weights)


# ---- what a user's program has in hand -------------------------------------------------

THETA, FACTOR, ORIGINAL = 10000., 4., 4096
BETA_FAST, BETA_SLOW = 32., 1.


def _frequencies(c):
    """Angle per position of every rotated pair in 64 bits, and the factor on the rotated features."""
    r, theta, magnitude = c['rotary_dim'], THETA, 1.
    if c['scaling'] == 'ntk':
        theta = THETA * FACTOR ** (r / (r - 2)) if r > 2 else THETA
    f = theta ** (-np.arange(0, r, 2, dtype=np.float64) / r)
    if c['scaling'] == 'linear':
        f = f / FACTOR
    if c['scaling'] == 'yarn':
        keep = np.clip((ORIGINAL * f / (2 * math.pi) - BETA_SLOW) / (BETA_FAST - BETA_SLOW), 0., 1.)
        f, magnitude = f * keep + f / FACTOR * (1. - keep), 0.1 * math.log(FACTOR) + 1.
    return f, magnitude


def _lengths(c):
    """Cached tokens of every sequence: the same, or between half of the largest and the largest."""
    return [c['length'] if not c['ragged'] or b == 0 else max(0, int(c['length'] * (0.5 + 0.5 * (b * 0.6180339887 % 1.)))) for b in range(c['batch'])]


def _ancestors(batch, tokens, rng):
    """[batch, tokens, tokens]: a token sees itself and its ancestors; parents are drawn among the tokens before it."""
    mask = np.zeros((batch, tokens, tokens), dtype=bool)
    for t in range(tokens):
        parent = (rng.random(batch) * (t + 1)).astype(np.int64) - 1      # -1: a child of the last cached token
        mask[:, t] = np.where((parent >= 0)[:, None], mask[np.arange(batch), np.maximum(parent, 0)], False)
        mask[:, t, t] = True
    return mask


def prepare(case, seed):
    c, dtype = case, DTYPES[case['dtype']]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    b, h, kv, d = c['batch'], c['heads'], c['kv_heads'], c['d']

    def randn(*shape, scale=1.):
        return (torch.randn(*shape, device=DEV, generator=gen, dtype=torch.float32) * scale).to(dtype)

    if c['kind'] == 'tree':
        t = c['tokens']
        lengths = _lengths(c)
        capacity = max(lengths) + t + 37                 # a cache has room to grow
        qkv = randn(b, t, (h + 2 * kv) * d).view(b, t, h + 2 * kv, d).transpose(1, 2)
        s = dict(q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], k_cache=randn(b, kv, capacity, d), v_cache=randn(b, kv, capacity, d),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV), mask=None)
        if c['shape'] == 'tree':
            s['mask'] = torch.from_numpy(_ancestors(b, t, np.random.default_rng(seed))).to(DEV)
        return dict(s, case=c)
    n = c['seq']
    # queries and keys are views of a fused projection's rows
    rows = randn(b, n, (h + 2 * kv) * d, scale=1. if c['kind'] == 'rotate' else 3.).view(b, n, h + 2 * kv, d).transpose(1, 2)
    q, k = rows[:, :h], rows[:, h:h + kv]
    positions = torch.arange(n, device=DEV)
    if c['far']:                                         # each sequence somewhere in its context
        positions = positions + torch.randint(0, c['far'], (b, 1), device=DEV, generator=gen)
    s = dict(case=c, q=q, k=k, positions=positions)
    if c['kind'] == 'norm_rotate':
        per_head = c['weights'] == 'heads'
        s['wq'] = 1. + randn(*((h, d) if per_head else (d,)), scale=0.2)
        s['wk'] = 1. + randn(*((kv, d) if per_head else (d,)), scale=0.2)
    if c['grad']:
        s['dq'], s['dk'] = randn(b, h, n, d), randn(b, kv, n, d)
        for name in ('q', 'k', 'wq', 'wk'):
            if name in s:
                s[name] = s[name].detach().requires_grad_()
    f, s['magnitude'] = _frequencies(c)
    s['frequencies'] = torch.from_numpy(f).to(DEV)
    if own:
        from native_sparse_attention_pytorch_b200 import RotaryFrequencies
        scaling = {} if c['scaling'] == 'none' else dict(scaling=c['scaling'], factor=FACTOR)
        if c['scaling'] == 'yarn':
            scaling.update(original_length=ORIGINAL, beta_fast=BETA_FAST, beta_slow=BETA_SLOW)
        s['rotary'] = RotaryFrequencies(d, rotary_dim=c['rotary_dim'], theta=THETA, layout=c['layout'], **scaling)
    return s


# ---- the plain forms ---------------------------------------------------------------------

def _turn(x, s, inverse=False):
    """Rotation of the first features of x [B, H, N, d] in 32 bits, by angles formed in 64."""
    c, r = s['case'], s['case']['rotary_dim']
    angle = s['positions'].double()[..., None] * s['frequencies']
    if angle.dim() == 3:
        angle = angle[:, None]
    co, si = (angle.cos() * s['magnitude']).float(), (angle.sin() * s['magnitude']).float()
    if inverse:
        si = -si
    if c['layout'] == 'half':
        a, z = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((a * co - z * si, z * co + a * si, x[..., r:]), dim=-1)
    a, z = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * co - z * si, z * co + a * si), dim=-1).flatten(-2), x[..., r:]), dim=-1)


def _plain_rows(x, w, dy, s):
    """(y, dx, dw) of one of the two, dx and dw where dy is given and dw where w is."""
    dtype, x = x.dtype, x.detach().float()
    if w is None:
        y = _turn(x, s).to(dtype)
        return (y,) if dy is None else (y, _turn(dy.float(), s, inverse=True).to(dtype), None)
    w32 = w.detach().float()
    w32 = w32[:, None] if w32.dim() == 2 else w32
    rstd = (x.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    unit = x * rstd
    y = _turn(unit * w32, s).to(dtype)
    if dy is None:
        return (y,)
    g = _turn(dy.float(), s, inverse=True)
    dw = (g * unit).sum(dim=(0, 2) if w.dim() == 2 else (0, 1, 2), dtype=torch.float64).to(dtype)
    g = g * w32
    dx = rstd * (g - unit * (g * unit).mean(dim=-1, keepdim=True))
    return y, dx.to(dtype), dw


def _plain_tree(s):
    c = s['case']
    b, h, kv, t, d, cap = c['batch'], c['heads'], c['kv_heads'], c['tokens'], c['d'], s['k_cache'].shape[2]
    q = s['q'].float().reshape(b, kv, h // kv * t, d)
    cached = torch.arange(cap, device=DEV)[None] < s['lengths'][:, None]
    drafted = s['mask'] if s['mask'] is not None else torch.ones(t, t, dtype=torch.bool, device=DEV).tril().expand(b, t, t)
    seen = torch.cat((cached[:, None].expand(b, t, cap), drafted), dim=-1)[:, None].repeat(1, 1, h // kv, 1)
    keys, values = torch.cat((s['k_cache'], s['k']), dim=2).float(), torch.cat((s['v_cache'], s['v']), dim=2).float()
    logits = (q @ keys.transpose(-1, -2)).mul_(d ** -0.5).masked_fill_(~seen, -math.inf)
    top = logits.amax(dim=-1, keepdim=True)
    p = logits.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ values) / total
    return out.reshape(b, h, t, d).to(s['q'].dtype), (top + total.log()).reshape(b, h, t)


def run(state):
    s, c = state, state['case']
    if c['kind'] == 'tree':
        if own:
            from native_sparse_attention_pytorch_b200 import tree_attend
            return tree_attend(s['q'], s['k_cache'], s['v_cache'], s['lengths'], s['k'], s['v'], s['mask'], return_lse=True)
        return _plain_tree(s)
    wq, wk, dq, dk = (s.get(n) for n in ('wq', 'wk', 'dq', 'dk'))
    if own:
        from native_sparse_attention_pytorch_b200 import norm_rotate_heads, rotate_heads
        if wq is None:
            out = rotate_heads(s['q'], s['k'], s['rotary'], s['positions'])
        else:
            out = norm_rotate_heads(s['q'], s['k'], wq, wk, s['rotary'], s['positions'], eps=EPS)
        if dq is None:
            return out
        leaves = (s['q'], s['k']) if wq is None else (s['q'], s['k'], wq, wk)
        return (*(x.detach() for x in out), *torch.autograd.grad(out, leaves, (dq, dk)))
    a, z = _plain_rows(s['q'], wq, dq, s), _plain_rows(s['k'], wk, dk, s)
    return tuple(x for pair in zip(a, z) for x in pair if x is not None)


# ---- in 64 bits, from the definitions -----------------------------------------------------

def _exact_rows(x, w, dy, s):
    """Rotated pairs are complex numbers times magnitude * e^(i angle); gradients by their conjugates."""
    c, r = s['case'], s['case']['rotary_dim']
    turn = torch.polar(torch.full((), s['magnitude'], dtype=torch.float64, device=DEV), s['positions'].double()[..., None] * s['frequencies'])
    turn = turn[:, None] if turn.dim() == 3 else turn

    def rotated(v, by):
        z = torch.complex(v[..., :r // 2], v[..., r // 2:r]) if c['layout'] == 'half' else torch.view_as_complex(v[..., :r].unflatten(-1, (-1, 2)).contiguous())
        z = z * by
        out = v.clone()
        if c['layout'] == 'half':
            out[..., :r // 2], out[..., r // 2:r] = z.real, z.imag
        else:
            out[..., :r] = torch.view_as_real(z).flatten(-2)
        return out

    x = x.detach().double()
    if w is None:
        return (rotated(x, turn), None if dy is None else rotated(dy.double(), turn.conj()), None)
    w = w.detach().double()
    wide = w.unsqueeze(1) if w.dim() == 2 else w
    size = torch.sqrt(torch.einsum('bhnd,bhnd->bhn', x, x) / x.shape[-1] + EPS)[..., None]
    y = rotated(x / size * wide, turn)
    if dy is None:
        return y, None, None
    back = rotated(dy.double(), turn.conj())
    dw = torch.einsum('bhnd,bhnd->hd', back, x / size)
    back = back * wide
    dx = back / size - x * torch.einsum('bhnd,bhnd->bhn', back, x)[..., None] / (x.shape[-1] * size ** 3)
    return y, dx, dw if w.dim() == 2 else dw.sum(dim=0)


def _exact_tree(s):
    c, outs, sums = s['case'], [], []
    h, kv, t, d = c['heads'], c['kv_heads'], c['tokens'], c['d']
    for b, n in enumerate(_lengths(c)):
        q = s['q'][b].double().view(kv, h // kv, t, d)
        k, v = (torch.cat((s[m + '_cache'][b, :, :n], s[m][b]), dim=1).double() for m in 'kv')
        logits = torch.einsum('kgtd,ksd->kgts', q, k) / math.sqrt(d)
        hidden = ~s['mask'][b] if s['mask'] is not None else torch.ones(t, t, dtype=torch.bool, device=DEV).triu(1)
        logits[..., n:][..., hidden] = -math.inf
        lse = torch.logsumexp(logits, dim=-1)
        outs.append(torch.einsum('kgts,ksd->kgtd', torch.exp(logits - lse[..., None]), v).reshape(h, t, d))
        sums.append(lse.reshape(h, t))
    return torch.stack(outs), torch.stack(sums)


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'tree':
        return _exact_tree(s)
    a, z = (_exact_rows(s[n], s.get('w' + n), s.get('d' + n), s) for n in 'qk')
    return tuple(x for pair in zip(a, z) for x in pair if x is not None)


def work(case):
    c, size = case, 2 if case['dtype'] == 'bf16' else 4
    b, h, kv, d = c['batch'], c['heads'], c['kv_heads'], c['d']
    if c['kind'] == 'tree':
        t, cached = c['tokens'], sum(_lengths(c))
        rows = 2 * kv * (cached + b * t) + 2 * h * b * t                       # keys, values; queries, outputs
        return {'bytes': rows * d * size + 4 * b * h * t + (b * t * t if c['shape'] == 'tree' else 0) + 4 * b,
                'flops': 4 * d * h * t * (cached + b * (t + 1) / 2)}
    elements = b * c['seq'] * (h + kv) * d
    moved, ops = 2, 3 if c['kind'] == 'rotate' else 7
    if c['grad']:
        moved, ops = 4, ops + (3 if c['kind'] == 'rotate' else 12)
    return {'bytes': elements * moved * size + 8 * c['seq'] * (b if c['far'] else 1), 'flops': elements * ops}
