"""Rotary frequencies (mimir_amd.rotary) against their formulas, and the refusals that need no GPU."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.rotary import RotaryFrequencies, rotary


def test_turns_are_fractions_of_a_turn():
    table = RotaryFrequencies.create(64, base=500000.0, device="cpu")
    assert table.turns.shape == (32,) and table.amplitude == 1.0 and not table.interleaved
    for i, t in enumerate(table.turns.tolist()):
        want = Fraction(500000.0 ** (-2 * i / 64)) / Fraction(2 * math.pi) * 2 ** 64
        # the frequency and the quotient are 64-bit floats: three roundings of 2^-53
        assert abs((t % 2 ** 64) - want) <= want * Fraction(3, 2 ** 53) + 1, i


def test_a_far_position_is_exact():
    turns = RotaryFrequencies.create(8, device="cpu").turns.tolist()
    for pos in (1, 12345, 1 << 30, -77):
        for t, f in zip(turns, RotaryFrequencies.inverse_frequencies(8)[0]):
            got = (pos * t) % 2 ** 64 / 2 ** 64
            want = float(Fraction(f) * pos / Fraction(2 * math.pi) % 1)
            gap = abs(got - want)
            assert min(gap, 1 - gap) <= abs(pos) * (2 ** -64 + f * 2 ** -53) + 2 ** -52


def test_scalings():
    plain, one = RotaryFrequencies.inverse_frequencies(128, base=10000.0)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[63], 10000.0 ** (-126 / 128))
    linear, _ = RotaryFrequencies.inverse_frequencies(128, scaling="linear", factor=4.0)
    assert all(a == b / 4 for a, b in zip(linear, plain))
    ntk, _ = RotaryFrequencies.inverse_frequencies(128, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[63], plain[63] / 4)  # the slowest pair is slowed by the factor
    wave, _ = RotaryFrequencies.inverse_frequencies(128, scaling="wavelength", factor=8.0, original_positions=8192)
    for w, f in zip(wave, plain):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            assert math.isclose(w, f)
        elif turns <= 1:
            assert math.isclose(w, f / 8)
        else:
            assert f / 8 < w < f
    yarn, amplitude = RotaryFrequencies.inverse_frequencies(128, scaling="yarn", factor=16.0, original_positions=4096)
    assert math.isclose(amplitude, 0.1 * math.log(16.0) + 1.0)
    assert yarn[0] == 1.0 and math.isclose(yarn[63], plain[63] / 16)
    assert all(f / 16 <= y * (1 + 1e-12) and y <= f for y, f in zip(yarn, plain))
    assert RotaryFrequencies.create(128, scaling="yarn", factor=16.0, amplitude=1.0, device="cpu").amplitude == 1.0


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, base=1.0),
                                dict(rotary_dim=8, factor=0.0), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                dict(rotary_dim=8, scaling="wavelength", low_turns=4.0, high_turns=4.0),
                                dict(rotary_dim=8, scaling="yarn", slow_turns=40.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        RotaryFrequencies.create(kw.pop("rotary_dim"), device="cpu", **kw)


def test_calls_are_refused_on_the_cpu():
    table = RotaryFrequencies.create(64, device="cpu")
    q = torch.zeros(4, 2, 64)
    pos = torch.arange(4)
    with pytest.raises(RuntimeError, match="ROCm"):
        rotary(q, None, pos, table)
    with pytest.raises(ValueError, match="tokens, heads"):
        rotary(q[0], None, pos, table)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        rotary(q.half(), None, pos, table)
    with pytest.raises(ValueError, match="agree"):
        rotary(q, torch.zeros(5, 2, 64), pos, table)
    with pytest.raises(ValueError, match="agree"):
        rotary(q, q.bfloat16(), pos, table)


def _params(**kw):
    one = 4096  # never read: every call here is refused, or empty
    p = _capi.RotaryParams()
    p.q = p.q_out = p.k = p.k_out = p.turns = p.positions = one
    p.batch, p.seqlen, p.num_q_heads, p.num_kv_heads, p.head_dim, p.rotary_dim, p.dtype, p.amplitude = 1, 1, 2, 1, 64, 64, 1, 1.0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,exc", [
    (dict(dtype=7), TypeError), (dict(batch=-1), ValueError), (dict(num_q_heads=0), ValueError), (dict(rotary_dim=66), ValueError),
    (dict(rotary_dim=3), ValueError), (dict(rotary_dim=0), ValueError), (dict(head_dim=63), ValueError), (dict(q=None), ValueError),
    (dict(k_out=None), ValueError), (dict(turns=None), ValueError), (dict(positions=None), ValueError),
    (dict(amplitude=math.inf), ValueError), (dict(amplitude=math.nan), ValueError), (dict(q=4097), ValueError),
])
def test_c_abi_refusals(kw, exc):
    lib = _capi.load()
    with pytest.raises(exc):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_rotary(ctypes.byref(_params(**kw)), None))


def test_c_abi_empty_calls():
    lib = _capi.load()
    for kw in (dict(batch=0), dict(seqlen=0)):
        assert lib.mimir_prefixlm_rotary(ctypes.byref(_params(**kw)), None) == _capi.OK
    assert lib.mimir_prefixlm_rotary(None, None) == _capi.ERR_INVALID_ARGUMENT


@pytest.fixture
def turned_on_the_cpu(monkeypatch):
    """``rotary`` with the general path's launch replaced by the formula (64-bit angles, interleaved layout or halves)."""
    import mimir_amd.rotary as R

    def turn(query, key, positions, frequencies, inverse, inplace=False):
        angle = positions[..., None, None] * (frequencies.turns.double() * 2.0 ** -64 * 2 * math.pi) * (-1 if inverse else 1)
        z = torch.polar(torch.full_like(angle, frequencies.amplitude), angle)
        out = []
        for x in (query, key):
            if x is None:
                out.append(None)
                continue
            y = torch.view_as_real(torch.complex(*(x.detach().double().unflatten(-1, (2, -1)).unbind(-2))) * z)
            out.append(y.mT.flatten(-2).to(x.dtype))
        return tuple(out)

    monkeypatch.setattr(R, "_turn", turn)
    monkeypatch.setattr(R.P, "_check_device_tensor", lambda name, t: None)


def test_tangents_are_turned(turned_on_the_cpu):
    import torch.autograd.forward_ad as fwd

    table, pos = RotaryFrequencies.create(8, amplitude=1.5, device="cpu"), torch.arange(5) * 100
    gen = torch.Generator().manual_seed(0)
    q, k, tq, tk = (torch.randn(5, h, 8, generator=gen) for h in (3, 2, 3, 2))
    want = rotary(tq, tk, pos, table)
    with fwd.dual_level():
        dual = lambda x, t: fwd.make_dual(x, t)  # noqa: E731
        tangent = lambda x: fwd.unpack_dual(x).tangent  # noqa: E731
        a, b = rotary(dual(q, tq), dual(k, tk), pos, table)
        assert torch.equal(tangent(a), want[0]) and torch.equal(tangent(b), want[1])
        assert torch.equal(fwd.unpack_dual(a).primal, rotary(q, k, pos, table)[0])
        a, none = rotary(dual(q, tq), None, pos, table, inverse=True)
        assert none is None and torch.equal(tangent(a), rotary(tq, None, pos, table, inverse=True)[0])
        a, b = rotary(q, dual(k, tk), pos, table)  # one side alone
        assert (tangent(a) is None or not tangent(a).any()) and torch.equal(tangent(b), want[1])
        with torch.no_grad():
            assert torch.equal(tangent(rotary(dual(q, tq), k, pos, table)[0]), want[0])
        with pytest.raises(ValueError, match="gradient"):
            rotary(dual(q, tq), None, pos, table, inplace=True)
        w = tq.clone().requires_grad_(True)  # the tangent's own gradient is the turn back
        a, _ = rotary(dual(q, w), None, pos, table)
        g, = torch.autograd.grad(tangent(a), w, want[0])
        assert torch.equal(g, rotary(want[0], None, pos, table, inverse=True)[0])


@pytest.mark.parametrize("factor,amplitude", [(0.25, 1.0), (0.999, 1.0), (1.0, 1.0), (math.e, 1.1), (40.0, 0.1 * math.log(40.0) + 1.0)])
def test_yarn_amplitude(factor, amplitude):
    """A range that is not stretched is not amplified, nor damped."""
    freq, got = RotaryFrequencies.inverse_frequencies(64, scaling="yarn", factor=factor, original_positions=4096)
    assert math.isclose(got, amplitude)
    assert RotaryFrequencies.create(64, scaling="yarn", factor=factor, device="cpu").amplitude == got


@pytest.mark.parametrize("kw", [dict(batch=1 << 15, seqlen=1 << 15), dict(seqlen=(1 << 31) - 1, dtype=0)])
def test_launches_of_2_to_32_threads_are_refused(kw):
    p = _params(num_q_heads=1, num_kv_heads=0, q_out=1 << 50, **kw)
    p.q_stride_head = p.q_stride_token = p.q_out_stride_head = p.q_out_stride_token = 64
    p.q_stride_batch = p.q_out_stride_batch = 64 * p.seqlen
    lib = _capi.load()
    with pytest.raises(ValueError, match="too many tokens"):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_rotary(ctypes.byref(p), None))
