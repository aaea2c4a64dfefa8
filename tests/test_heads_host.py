"""Rotation of heads and norm with rotation, host side: frequencies against their formulas, phases in integers against 64-bit
angles, and what is refused, without a GPU."""
import ctypes as C
import math

import pytest
import torch

from native_sparse_attention_pytorch_b200 import RotaryFrequencies, norm_rotate_heads, rotate_heads
from native_sparse_attention_pytorch_b200 import _lib as L


def test_frequencies_of_the_scalings():
    r, theta, factor = 64, 10000.0, 8.0
    plain = [theta ** (-2 * m / r) for m in range(r // 2)]
    assert RotaryFrequencies(64).frequencies == tuple(plain)
    assert RotaryFrequencies(128, rotary_dim=64).frequencies == tuple(plain)
    linear = RotaryFrequencies(64, scaling='linear', factor=factor)
    assert linear.frequencies == tuple(f / factor for f in plain) and linear.magnitude == 1.0
    ntk = RotaryFrequencies(64, scaling='ntk', factor=factor).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / factor, rel_tol=1e-12)
    yarn = RotaryFrequencies(64, scaling='yarn', factor=factor, original_length=4096)
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, p, t in zip(yarn.frequencies, plain, turns):
        if t >= 32:
            assert f == p
        elif t <= 1:
            assert math.isclose(f, p / factor, rel_tol=1e-15)
        else:
            assert p / factor < f < p
    assert math.isclose(yarn.magnitude, 0.1 * math.log(factor) + 1)
    assert RotaryFrequencies(8, frequencies=[1.0, 0.5, 0.25, -0.125], magnitude=2.0).frequencies == (1.0, 0.5, 0.25, -0.125)


@pytest.mark.parametrize('position', [0, 1, 4095, 1 << 20, (1 << 40) + 12345, -7])
def test_integer_phases_are_the_angles(position):
    """position * step mod 2^64 turns against the angle in rational arithmetic: within position * 2^-65 turns of the frequency
    that the step stands for, and the step within 2^-53 of the frequency."""
    from fractions import Fraction
    rotary = RotaryFrequencies(64)
    for f, step in zip(rotary.frequencies, rotary._steps.tolist()):
        step %= 2 ** 64
        turns = Fraction(f / (2 * math.pi))
        assert abs(Fraction(step, 2 ** 64) - turns) <= Fraction(1, 2 ** 65)
        phase = Fraction(position * step % 2 ** 64, 2 ** 64)
        off = abs(phase - position * turns) % 1
        assert min(off, 1 - off) <= Fraction(abs(position), 2 ** 65)


@pytest.mark.parametrize('kwargs', [dict(dim_head=63), dict(dim_head=258), dict(dim_head=0), dict(dim_head=64, rotary_dim=66), dict(dim_head=64, rotary_dim=31),
                                    dict(dim_head=64, rotary_dim=0), dict(dim_head=64, layout='pairs'), dict(dim_head=64, scaling='cubic'),
                                    dict(dim_head=64, scaling='linear', factor=0.), dict(dim_head=64, theta=-1.), dict(dim_head=64, scaling='yarn', factor=2.),
                                    dict(dim_head=64, scaling='yarn', factor=2., original_length=4096, beta_fast=1., beta_slow=1.),
                                    dict(dim_head=64, frequencies=[1.0]), dict(dim_head=4, frequencies=[1.0, math.inf]),
                                    dict(dim_head=4, frequencies=[1.0, 1.0], scaling='linear')])
def test_frequencies_refuse(kwargs):
    with pytest.raises(ValueError):
        RotaryFrequencies(**kwargs)


def test_no_cpu_path():
    rotary, q, w = RotaryFrequencies(64), torch.randn(1, 2, 3, 64), torch.ones(64)
    with pytest.raises(L.NsaError, match='CUDA tensors only'):
        rotate_heads(q, q, rotary)
    with pytest.raises(L.NsaError, match='CUDA tensors only'):
        norm_rotate_heads(q, q, w, w, rotary)


def test_entry_points_check_their_arguments():
    lib = L.load()
    assert lib.nsa_heads_fwd(None, None) == -1 and lib.nsa_heads_bwd(None, None) == -1 and lib.nsa_heads_workspace_bytes(None) == -1
    a = L.HeadsArgs(batch=1, seq=4, dim_head=64, rotary_dim=64, dtype=7)
    a.part[0].heads = 2
    assert lib.nsa_heads_fwd(C.byref(a), None) == -3
    a.dtype = L.NSA_BF16
    for field, bad in (('dim_head', 63), ('dim_head', 258), ('rotary_dim', 0), ('rotary_dim', 66), ('rotary_dim', 33), ('batch', -1)):
        good = getattr(a, field)
        setattr(a, field, bad)
        assert lib.nsa_heads_fwd(C.byref(a), None) == -2, (field, bad)
        setattr(a, field, good)
    a.batch, a.seq = 1 << 16, 1 << 15
    assert lib.nsa_heads_fwd(C.byref(a), None) == -2        # 2^31 tokens
    a.batch, a.seq = 1, 4
    assert lib.nsa_heads_fwd(C.byref(a), None) == -1        # the frequencies are NULL
    steps = (C.c_uint64 * 32)()
    a.steps = C.addressof(steps)
    assert lib.nsa_heads_fwd(C.byref(a), None) == -1        # x and out are NULL
    a.part[0].x.ptr, a.part[0].out.ptr = 0x1001, 0x1000
    assert lib.nsa_heads_fwd(C.byref(a), None) == -4        # an odd address
    a.part[0].x.ptr, a.norm = 0x1000, 1
    assert lib.nsa_heads_fwd(C.byref(a), None) == -1        # no weight
    a.part[0].weight = 0x1000
    assert lib.nsa_heads_bwd(C.byref(a), None) == -1        # no weight gradient
    a.part[0].dweight, a.part[0].dy.ptr = 0x1000, 0x1000
    assert lib.nsa_heads_bwd(C.byref(a), None) == -5        # no work buffer
    need = lib.nsa_heads_workspace_bytes(C.byref(a))
    assert need > 0
    a.workspace, a.workspace_bytes = 0x1000, need - 1
    assert lib.nsa_heads_bwd(C.byref(a), None) == -5
    a.batch = 0
    assert lib.nsa_heads_fwd(C.byref(a), None) == 0         # nothing to do
