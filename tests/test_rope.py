"""Rotary embedding at given positions without a GPU: the frequencies of each scaling, the
oracle against plain trigonometry, and the refusals of the C entry and of the Python call."""
from __future__ import annotations

import math

import pytest
import torch

import ttcd_amd
from oracle import drafted_ref
from ttcd_amd import _lib, rope_frequencies

INV, UNSUP = _lib.TTCD_ERR_INVALID_ARGUMENT, _lib.TTCD_ERR_UNSUPPORTED
P = 0x10000  # never dereferenced


def test_plain_frequencies_are_the_prologues():
    inv, scale = rope_frequencies(128, 1e6)
    assert scale == 1.0 and inv.dtype == torch.float32
    assert torch.allclose(inv, ttcd_amd.rope_inv_freq(128, 1e6), rtol=1e-5, atol=0)
    assert inv[0] == 1.0 and math.isclose(inv[63].item(), 1e6 ** (-126 / 128), rel_tol=1e-6)


def test_scaled_frequencies():
    plain = rope_frequencies(64, 1e4)[0].double()
    inv, scale = rope_frequencies(64, 1e4, {"type": "linear", "factor": 4})
    assert scale == 1.0 and torch.allclose(inv.double(), plain / 4, rtol=1e-6)
    m = {"original_max_position_embeddings": 2048}
    # dynamic: nothing changes up to m; beyond, the lowest frequency falls by n f / m - f + 1
    for n, by in ((1000, 1.0), (2048, 1.0), (8192, 4 * 4 - 3.0)):
        inv, _ = rope_frequencies(64, 1e4, {"type": "dynamic", "factor": 4, **m}, length=n)
        assert inv[0] == 1.0
        assert math.isclose(inv[31].item(), plain[31].item() / by, rel_tol=1e-5)
    # yarn: pairs that turn often stay, those that hardly turn are stretched
    inv, scale = rope_frequencies(64, 1e4, {"rope_type": "yarn", "factor": 4, **m})
    assert math.isclose(scale, 0.1 * math.log(4) + 1)
    turns = 2048 * plain / (2 * math.pi)
    kept, stretched = turns > 40, turns < 0.8
    assert kept.any() and stretched.any()
    assert torch.allclose(inv.double()[kept], plain[kept], rtol=1e-6)
    assert torch.allclose(inv.double()[stretched], plain[stretched] / 4, rtol=1e-6)
    ratio = inv.double() / plain
    assert (ratio[1:] <= ratio[:-1] + 1e-6).all()
    assert rope_frequencies(64, 1e4, {"rope_type": "yarn", "factor": 4, "attention_factor": 1.5,
                                      **m})[1] == 1.5
    q = {"rope_type": "yarn", "factor": 40, "mscale": 1.0, "mscale_all_dim": 0.5, **m}
    assert math.isclose(rope_frequencies(64, 1e4, q)[1],
                        (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1))
    # llama3: a ramp over the turns
    inv, _ = rope_frequencies(64, 1e4, {"rope_type": "llama3", "factor": 8, "low_freq_factor": 1,
                                        "high_freq_factor": 4, **m})
    keep = ((turns - 1) / 3).clamp(0, 1)
    assert torch.allclose(inv.double(), plain * keep + plain / 8 * (1 - keep), rtol=1e-6)
    for bad in ({"type": "linear"}, {"rope_type": "yarn", "factor": 2}):
        with pytest.raises(ValueError, match="needs"):
            rope_frequencies(64, 1e4, bad)
    with pytest.raises(NotImplementedError):
        rope_frequencies(64, 1e4, {"rope_type": "other"})
    for dim in (0, 7, -2):
        with pytest.raises(ValueError, match="even"):
            rope_frequencies(dim, 1e4)


def test_the_oracle_turns_pairs():
    x = torch.tensor([1.0, 0.0, 0.0, 2.0, 7.0]).view(1, 1, 1, 5)
    f, p = torch.tensor([1.0, 0.5]), torch.tensor([[3]])
    y, _ = drafted_ref.rope(x, f, p)  # pairs (0, 2), (1, 3)
    want = [math.cos(3), -2 * math.sin(1.5), math.sin(3), 2 * math.cos(1.5), 7.0]
    assert torch.allclose(y.flatten(), torch.tensor(want, dtype=torch.float64))
    y, _ = drafted_ref.rope(x, f, p, interleaved=True, inverse=True, scale=2.0)
    want = [2 * math.cos(3), -2 * math.sin(3), 4 * math.sin(1.5), 4 * math.cos(1.5), 7.0]
    assert torch.allclose(y.flatten(), torch.tensor(want, dtype=torch.float64))


def _call(q=P, k=P, qo=P, ko=P, f=P, n=32, B=1, T=2, Hq=2, Hkv=1, D=64, qs=(256, 128, 64, 1),
          ks=(128, 64, 64, 1), scale=1.0, dt=0):
    s = _lib.strides4
    return _lib.lib().ttcd_rope_fwd(q, k, qo, ko, f, n, None, 0, None, 0, B, T, Hq, Hkv, D, s(qs),
                                    s(ks), s(qs), s(ks), 0, 0, scale, dt, None)


def test_bad_arguments():
    assert _call(q=None) == _call(qo=None) == _call(f=None) == _call(k=None) == _call(ko=None) == INV
    assert _call(n=0) == _call(n=33) == _call(B=0) == _call(T=0) == _call(Hq=0) == _call(Hkv=-1) == INV
    assert _call(qs=(256, 128, 64, 2)) == _call(ks=(128, 64, 64, 0)) == _call(dt=3) == INV
    assert _call(scale=math.nan) == _call(scale=math.inf) == INV
    assert _call(D=1, n=1) == _call(D=1026) == _call(B=1 << 20, T=1 << 20) == UNSUP
    assert _call(Hq=1 << 27) == UNSUP
    assert _lib.lib().ttcd_rope_fwd(P, P, P, P, P, 32, P, 0, None, 0, 1, 2, 2, 1, 64,
                                    _lib.strides4((256, 128, 64, 1)),
                                    _lib.strides4((128, 64, 64, 1)),
                                    _lib.strides4((256, 128, 64, 1)),
                                    _lib.strides4((128, 64, 64, 1)), 0, 0, 1.0, 0, None) == INV


def test_python_refuses_the_cpu():
    x = torch.zeros(1, 2, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        ttcd_amd.rope(x, x, torch.ones(32))


def test_the_oracles_far_angles():
    """The oracle's turns of far positions against decimals of 90 digits: the product of a position
    and a frequency passes 53 bits from 2^29 on."""
    from decimal import Decimal, getcontext
    getcontext().prec = 90
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510"
                         "582097494459230781640628620899862803482534211706798")
    f = torch.tensor([1.0, 0.8659643, 0.0123, 1e-5])
    pos = torch.tensor([[5, 2 ** 29 + 1, 2 ** 40 - 1, 2 ** 52 + 12345, 2 ** 53 - 1, -2 ** 53 + 3]])
    x = torch.zeros(1, 6, 1, 8)
    x[..., :4] = 1.0  # (cos, sin) of every pair
    y, _ = drafted_ref.rope(x, f, pos)
    for t, p in enumerate(pos[0].tolist()):
        for i, w in enumerate(f.tolist()):
            a = float((Decimal(p) * Decimal(w)) % two_pi)
            assert abs(y[0, t, 0, i].item() - math.cos(a)) < 1e-14
            assert abs(y[0, t, 0, 4 + i].item() - math.sin(a)) < 1e-14


def test_more_threads_than_a_launch_has():
    """One element an access, 512 tasks a workgroup of 256 threads: 2^33 tasks are 2^32 threads.
    Interleaved or not, and as many with whole vectors."""
    odd = dict(Hq=33, Hkv=31, D=128, n=64, qs=(128, 128 * 33, 128, 1), ks=(129, 128 * 31, 128, 1))
    assert _call(B=1 << 21, T=1, **odd) == UNSUP  # 2^21 * 64 * 64 tasks
    assert _call(B=1 << 20, T=2, **odd) == UNSUP
    even = dict(odd, Hq=512, Hkv=512, qs=(128, 1 << 16, 128, 1), ks=(128, 1 << 16, 128, 1))
    assert _call(B=1 << 20, T=1, **even) == UNSUP  # 2^20 * 1024 * 8


def test_offsets_that_are_no_position():
    for offset, n in ((2 ** 53 + 1, 1), (-2 ** 53 - 1, 1), (2 ** 53 - 3, 5)):
        s = _lib.strides4
        assert _lib.lib().ttcd_rope_fwd(P, None, P, None, P, 32, None, 0, None, offset, 1, n, 2, 0, 64,
                                        s((256, 128, 64, 1)), None, s((256, 128, 64, 1)), None, 0, 0,
                                        1.0, 0, None) == INV
