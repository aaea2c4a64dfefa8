"""Rotary position embedding used in front of the selected and sliding
branches (upstream call sites NSA:238, NSA:643).  Convention: inverse
frequency theta^(-2m/d) on the adjacent feature pair (2m, 2m+1), angles in
fp32, result in the input dtype.  On CUDA tensors the rotation is one kernel
of the library (`nsa_rotary`) over tables of cos / sin built here; CPU tensors
(host-side tests) take the same formula in plain PyTorch."""
import ctypes as C
import math

import torch
from torch import nn
from torch.autograd import Function, forward_ad

from . import _lib as L


_INV_FREQ = {}


def inverse_frequencies(dim, theta, device):
    """theta^(-2m/dim), always fp32: kept here instead of as a module buffer, which `module.bfloat16()` would round to
    8 bits and so turn positions past a few hundred into wrong angles."""
    key = (dim, theta, device)
    inv_freq = _INV_FREQ.get(key)
    if inv_freq is None:   # computed on the host (as upstream's package does at construction), kept per device
        inv_freq = _INV_FREQ[key] = (theta ** (-torch.arange(0, dim, 2).float() / dim)).to(device)
    return inv_freq


def _tables(dim, theta, n, offset, device):
    """cos / sin of the angles [n, dim/2] in fp32."""
    inv_freq = inverse_frequencies(dim, theta, device)
    pos = torch.arange(n, device=device, dtype=torch.float32) + offset
    ang = pos[:, None] * inv_freq[None, :]
    return ang.cos().contiguous(), ang.sin().contiguous()


class _Rotate(Function):
    """out = rotation of every feature pair of x [B, H, N, d] by the angles of the tables [N, d/2]."""

    @staticmethod
    def forward(ctx, x, cos, sin):
        from .ops import dim_order
        ctx.save_for_backward(cos, sin)
        ctx.order = dim_order(x)
        return _launch(x, cos, sin, inverse=False)

    @staticmethod
    def backward(ctx, grad):
        # the gradient is written in the memory layout of the forward's input (heads as a strided view of the
        # projection output), so that the gradient of that view is a view again instead of a copy
        cos, sin = ctx.saved_tensors
        return _launch(grad, cos, sin, inverse=True, order=ctx.order), None, None


def _launch(x, cos, sin, inverse, order=None):
    from .ops import empty_in_order
    lib = L.load()
    v = 16 // x.element_size()
    if x.stride(-1) != 1 or x.data_ptr() % 16 or any(s % v for s in x.stride()[:-1]):
        x = x.contiguous()
    b, h, n, d = x.shape
    out = empty_in_order((b, h, n, d), order or (0, 1, 2, 3), x.dtype, x.device)
    args = L.RotaryArgs(x=L.t4(x), out=L.ptr(out), cos_table=L.ptr(cos), sin_table=L.ptr(sin), batch=b, heads=h,
                        seq=n, dim_head=d, dtype=L.dtype_code(x), inverse=1 if inverse else 0,
                        out_stride_b=out.stride(0), out_stride_h=out.stride(1), out_stride_n=out.stride(2))
    with torch.cuda.device(x.device):
        L.check(lib.nsa_rotary(C.byref(args), L.stream_of(x)))
    return out


class RotaryEmbedding(nn.Module):
    def __init__(self, dim, theta=10000.0):
        super().__init__()
        self.dim, self.theta = dim, theta

    def rotate_queries_or_keys(self, t, offset=0):
        n = t.shape[-2]
        cos, sin = _tables(self.dim, self.theta, n, offset, t.device)
        if t.is_cuda and t.dim() == 4 and t.dtype in (torch.float32, torch.bfloat16) and \
                t.shape[-1] % (16 // t.element_size()) == 0:
            return _Rotate.apply(t, cos, sin)
        cos, sin = cos.repeat_interleave(2, dim=-1), sin.repeat_interleave(2, dim=-1)
        x = t.float()
        even, odd = x[..., 0::2], x[..., 1::2]
        rotated = torch.stack((-odd, even), dim=-1).flatten(-2)
        return (x * cos + rotated * sin).to(t.dtype)

    def rotate_queries_with_cached_keys(self, q, k):
        nq, nk = q.shape[-2], k.shape[-2]
        return self.rotate_queries_or_keys(q, offset=nk - nq), self.rotate_queries_or_keys(k)


LAYOUTS = ('interleaved', 'half')
SCALINGS = (None, 'linear', 'ntk', 'yarn')


class RotaryFrequencies:
    """The frequencies of a rotary embedding of heads, for `rotate_heads` and `norm_rotate_heads`.

    dim_head      features of a head (even, at most 256); the first `rotary_dim` of them (even; default: all) are rotated
                  in pairs, the others pass unchanged
    theta         base: pair m turns by theta^(-2m / rotary_dim) radians a position
    layout        'interleaved': pairs (2m, 2m+1), as `RotaryEmbedding`; 'half': pairs (m, m + rotary_dim / 2)
    scaling       for contexts longer than the trained one by `factor`:
                  'linear'  every frequency divided by factor;
                  'ntk'     the base becomes theta * factor^(r / (r - 2)), r = rotary_dim: the lowest frequency is divided by
                            factor, the highest stays;
                  'yarn'    a pair that makes at least `beta_fast` turns within `original_length` positions keeps its frequency,
                            one with at most `beta_slow` turns has it divided by factor, linear in the turns between them, and
                            rotated features are multiplied by 0.1 ln(factor) + 1 (Peng et al. 2023, "YaRN: Efficient Context
                            Window Extension of Large Language Models", sections 3.2 to 3.4)
    frequencies   instead of theta and scaling: rotary_dim / 2 radians per position
    magnitude     factor on the rotated features, instead of the scaling's own

    Frequencies are doubles, kept as 64-bit fractions of a turn (`module.bfloat16()` of whatever holds this changes nothing).  An angle
    is off by the rounding of that fraction alone, |position| * (|frequency| * 2^-52 + 2^-62) radians at most: 10^-7 at position
    4 * 10^8 for a frequency of 1, less for lower ones."""

    def __init__(self, dim_head, rotary_dim=None, theta=10000.0, layout='interleaved', scaling=None, factor=1.0,
                 original_length=None, beta_fast=32.0, beta_slow=1.0, frequencies=None, magnitude=None):
        rotary_dim = dim_head if rotary_dim is None else rotary_dim
        if dim_head < 2 or dim_head % 2 or dim_head > 256:
            raise ValueError(f'dim_head must be even and at most 256, got {dim_head}')
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > dim_head:
            raise ValueError(f'rotary_dim must be even, at least 2 and at most dim_head, got {rotary_dim}')
        if layout not in LAYOUTS:
            raise ValueError(f'layout must be one of {LAYOUTS}, got {layout!r}')
        if scaling not in SCALINGS:
            raise ValueError(f'scaling must be one of {SCALINGS}, got {scaling!r}')
        if not factor > 0 or not theta > 0:
            raise ValueError(f'theta and factor must be positive, got {theta} and {factor}')
        if frequencies is not None and scaling is not None:
            raise ValueError('frequencies are taken as they are: no scaling beside them')
        if frequencies is None:
            base = theta * factor ** (rotary_dim / (rotary_dim - 2)) if scaling == 'ntk' and rotary_dim > 2 else theta
            frequencies = [base ** (-2 * m / rotary_dim) for m in range(rotary_dim // 2)]
            if scaling == 'linear':
                frequencies = [f / factor for f in frequencies]
            elif scaling == 'yarn':
                if original_length is None or not original_length > 0 or not beta_fast > beta_slow:
                    raise ValueError('yarn needs original_length, and beta_fast above beta_slow')
                keep = [min(1., max(0., (original_length * f / (2 * math.pi) - beta_slow) / (beta_fast - beta_slow)))
                        for f in frequencies]
                frequencies = [f * k + f / factor * (1 - k) for f, k in zip(frequencies, keep)]
                if magnitude is None:
                    magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != rotary_dim // 2 or not all(math.isfinite(f) for f in frequencies):
            raise ValueError(f'{rotary_dim // 2} finite frequencies are needed, got {len(frequencies)}')
        self.dim_head, self.rotary_dim, self.layout = dim_head, rotary_dim, layout
        self.frequencies = tuple(frequencies)
        self.magnitude = 1.0 if magnitude is None else float(magnitude)
        # 2^64 times the turns per position; whole turns drop out, and the upper half stands for negative numbers
        steps = [round(f / (2 * math.pi) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
        self._steps = torch.tensor([s - 2 ** 64 if s >= 2 ** 63 else s for s in steps], dtype=torch.int64)
        self._on = {}

    def steps(self, device):
        """The table on `device`, copied there once."""
        t = self._on.get(device)
        if t is None:
            if torch.cuda.is_current_stream_capturing():
                raise L.NsaError('the frequencies are not on this device yet: call once before a CUDA graph is recorded')
            t = self._on[device] = self._steps.to(device)
            torch.cuda.current_stream(device).synchronize()     # other streams may read it from now on
        return t


def _rotate(q, k, q_weight, k_weight, rotary, positions, offset, norm, eps, out):
    if forward_ad._current_level >= 0:
        raise L.NsaError('the rotation of heads has no forward-mode derivative')
    if not q.is_cuda:
        L.require_cuda(q)
    if q.shape[-1] != rotary.dim_head:
        raise L.NsaError(f'the frequencies are for heads of {rotary.dim_head}, not {q.shape[-1]}')
    out_q, out_k = (None, None) if out is None else out
    return tuple(L.host().rotate_heads(q, k, q_weight, k_weight, rotary.steps(q.device), rotary.rotary_dim,
                                       rotary.layout == 'half', rotary.magnitude, positions, offset, norm, eps, out_q, out_k))


def rotate_heads(q, k, rotary, positions=None, offset=0, out=None):
    """Queries and keys rotated by their positions, in one launch: q [b, q_heads, n, d], k [b, kv_heads, n, d] (or None) ->
    the same shapes, contiguous; fp32 arithmetic, rounded once.  float32 or bfloat16, any strides with a contiguous last
    axis.  `positions`: int64 or int32, [n] or [b, n] (default 0 .. n-1), `offset` is added to them.  `out`: a pair of
    tensors to write instead (rows of a cache, or q and k themselves, each in its own place), where no gradient is wanted.
    Differentiable in q and k; gradients keep the memory order of their inputs."""
    return _rotate(q, k, None, None, rotary, positions, offset, False, 0.0, out)
