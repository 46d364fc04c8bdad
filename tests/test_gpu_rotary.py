"""Rotary positions on the GPU (mimir_amd.rotary) against complex multiplication in 64 bits.

A kernel's cosine and sine are off by at most 2^-22: the angle (at most pi / 4 after the quarter turns) has two
roundings, 2 * 2^-24 * pi / 4 < 2^-23, and 2^-34 of a turn; the series' last operations one or two more of 2^-24 each.
With the products' and the sum's roundings and the amplitude's a turned column is off by at most
2^-21 * amplitude (|a| + |b|); rounding to bf16 adds 2^-8 of it."""

import pytest
import torch

from mimir_amd.rotary import RotaryFrequencies, rotary
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


def _near(got, want, size, name):
    off = 2.0 ** -21 * size
    if got.dtype == torch.bfloat16:
        off = off + 2.0 ** -8 * (want.abs() + off)
    else:
        off = off + 2.0 ** -24 * want.abs()
    bad = (got.cpu().double() - want).abs() > off
    assert not bad.any(), (name, int(bad.sum()), (got.cpu().double() - want).abs().max())


def _check(device, lead, hq, hkv, d, rd, dtype, interleaved, scaling="none", max_pos=5000, index=torch.int64, grad=True, **kw):
    gen = torch.Generator().manual_seed(rd * 7 + d)
    tokens = 1
    for n in lead:
        tokens *= n
    qkv = torch.randn(*lead, hq + 2 * hkv, d, generator=gen).to(dtype).to(device)
    q, k = qkv[..., :hq, :], qkv[..., hq:hq + hkv, :]
    pos = torch.randint(0, max_pos, lead, generator=gen).to(index)
    freq, amplitude = RotaryFrequencies.inverse_frequencies(rd, scaling=scaling, **kw)
    table = RotaryFrequencies.create(rd, interleaved=interleaved, scaling=scaling, device=device, **kw)
    if grad:
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    out = rotary(q, k, pos.to(device), table)
    flat = lambda t: t.detach().reshape(tokens, -1, d)  # noqa: E731
    for name, x, y in (("q", q, out[0]), ("k", k, out[1])):
        assert y.shape == x.shape and y.dtype == dtype
        want, size = O.rotary(flat(x), pos.reshape(-1), freq, amplitude, interleaved)
        _near(flat(y), want, size, name)
    if grad:
        dout = [torch.randn(y.shape, generator=gen).to(dtype).to(device) for y in out]
        got = torch.autograd.grad(out, (q, k), dout)
        for name, g, y in (("dq", dout[0], got[0]), ("dk", dout[1], got[1])):
            want, size = O.rotary(flat(g), pos.reshape(-1), freq, amplitude, interleaved, inverse=True)
            _near(flat(y), want, size, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(128, 128), (64, 64), (64, 20), (128, 64), (96, 96), (80, 32), (64, 2), (128, 26), (6, 4), (128, 126)])
def test_layouts_and_parts(device, dtype, interleaved, d, rd):
    _check(device, (3, 37), 4, 2, d, rd, dtype, interleaved)


@pytest.mark.parametrize("lead", [(1,), (1, 1), (5, 1), (1, 700), (4099,), (2, 3)])
def test_token_counts(device, lead):
    _check(device, lead, 16, 4, 128, 128, torch.bfloat16, False, index=torch.int32)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (32, 8), (7, 1), (40, 8)])
def test_heads(device, hq, hkv):
    _check(device, (2, 65), hq, hkv, 64, 64, torch.float32, True)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "wavelength", "yarn"])
def test_scalings_at_far_positions(device, scaling):
    _check(device, (2, 50), 4, 2, 128, 128, torch.float32, False, scaling=scaling, factor=16.0, original_positions=4096,
           max_pos=1 << 28)


def test_no_key_and_inverse(device):
    x = torch.randn(33, 4, 64, device=device)
    table = RotaryFrequencies.create(64, device=device)
    pos = torch.arange(33, device=device)
    y, none = rotary(x, None, pos, table)
    assert none is None
    back, _ = rotary(y, None, pos, table, inverse=True)
    assert (back - x).abs().max() <= 2.0 ** -20 * 2 * x.abs().max()  # both turns' 2^-21 (|a| + |b|)


def test_in_place_and_broadcast_positions(device):
    q, k = torch.randn(3, 9, 4, 96, device=device).bfloat16(), torch.randn(3, 9, 2, 96, device=device).bfloat16()
    table = RotaryFrequencies.create(48, interleaved=True, device=device)
    pos = torch.arange(100, 109, device=device)
    want = rotary(q, k, pos.expand(3, 9).contiguous(), table)
    q0, k0 = q.clone(), k.clone()
    got = rotary(q, k, pos, table, inplace=True)
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(q[..., 48:], q0[..., 48:]) and torch.equal(k[..., 48:], k0[..., 48:])


def test_strides_and_odd_addresses(device):
    """Transposed heads and rows off their 16 bytes take narrower accesses, a strided head_dim a copy."""
    base = torch.randn(5, 8, 41, 68, device=device).bfloat16()
    pos = torch.randint(0, 999, (5, 41), device=device)
    table = RotaryFrequencies.create(64, device=device)
    turned = torch.randn(5, 8, 64, 41, device=device).bfloat16().transpose(2, 3)
    for x in (base[..., :64], base[..., 1:65], base[..., 2:66], turned):
        x = x.transpose(1, 2)  # [batch, tokens, heads, d]
        want = rotary(x.contiguous(), None, pos, table)[0]
        assert torch.equal(rotary(x, None, pos, table)[0], want)


def test_gradient_of_the_gradient_and_of_differences(device):
    x = torch.randn(7, 2, 32, device=device, requires_grad=True)
    table = RotaryFrequencies.create(16, scaling="yarn", factor=4.0, original_positions=64, device=device)
    pos = torch.arange(7, device=device) * 5
    f = lambda t: rotary(t, None, pos, table)[0]  # noqa: E731
    w, v = torch.randn(7, 2, 32, device=device), torch.randn(7, 2, 32, device=device)
    g, = torch.autograd.grad((f(x) * w).sum(), x, create_graph=True)
    # linear in x: a difference of any step is the derivative
    diff = ((f(x + v) - f(x)) * w).sum()
    assert abs((g * v).sum() - diff) <= 1e-4 * (w.norm() * v.norm())
    w2 = w.clone().requires_grad_(True)
    g2, = torch.autograd.grad((f(x) * w2).sum(), x, create_graph=True)
    gg, = torch.autograd.grad((g2 * v).sum(), w2)
    assert (gg - f(v)).abs().max() <= 1e-5


def test_shared_leaf_and_one_sided_gradients(device):
    x = torch.randn(9, 4, 64, device=device, requires_grad=True)
    table = RotaryFrequencies.create(64, device=device)
    pos = torch.arange(9, device=device)
    q, k = rotary(x, x, pos, table)
    both, = torch.autograd.grad((q.sum() + 2 * k.sum()), x, retain_graph=True)
    one, = torch.autograd.grad(q.sum(), x, retain_graph=True)
    assert (both - 3 * one).abs().max() <= 1e-5
    k2 = torch.randn(9, 1, 64, device=device)  # needs no gradient
    q, k2 = rotary(x, k2, pos, table)
    assert torch.autograd.grad(q.sum(), x)[0].shape == x.shape


def test_refusals(device):
    q = torch.zeros(4, 2, 64, device=device)
    table = RotaryFrequencies.create(64, device=device)
    pos = torch.arange(4, device=device)
    with pytest.raises(TypeError, match="int32 or int64"):
        rotary(q, None, pos.float(), table)
    with pytest.raises(ValueError, match="do not fit"):
        rotary(q, None, torch.arange(5, device=device), table)
    with pytest.raises(ValueError, match="frequencies"):
        rotary(q[..., :32], None, pos, table)
    with pytest.raises(ValueError, match="int64 vector"):
        rotary(q, None, pos, table._replace(turns=table.turns.cpu()))
    with pytest.raises(ValueError, match="gradient"):
        rotary(q.clone().requires_grad_(True), None, pos, table, inplace=True)
    with pytest.raises(ValueError, match="in-place"):
        rotary(q.expand(4, 2, 64)[:, :1].expand(4, 3, 64), None, pos, table, inplace=True)
    empty = rotary(q[:0], None, pos[:0], table)[0]
    assert empty.shape == (0, 2, 64)


def test_captured_and_on_another_stream(device):
    q, k = torch.randn(8, 1, 16, 128, device=device).bfloat16(), torch.randn(8, 1, 4, 128, device=device).bfloat16()
    pos = torch.zeros(8, 1, dtype=torch.int64, device=device)
    table = RotaryFrequencies.create(128, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary(q, k, pos, table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = rotary(q, k, pos, table)
    for step in range(3):
        pos.fill_(1000 * step + 7)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = rotary(q, k, pos, table)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_one_tensor_in_place_as_query_and_key(device):
    x = torch.randn(4, 3, 64, device=device)
    table, pos = RotaryFrequencies.create(64, device=device), torch.arange(4, device=device)
    for key in (x, x[:, :1]):
        with pytest.raises(ValueError, match="memory of their own"):
            rotary(x, key, pos, table, inplace=True)
    want, _ = rotary(x, None, pos, table)
    rotary(x[:, :2], x[:, 2:], pos, table, inplace=True)
    assert torch.equal(x, want)


def test_captured_forward_and_backward(device):
    """The whole step in a graph, replayed beside eager steps of the same leaves, and a backward on a side stream."""
    q, k = (torch.randn(3, 37, h, 64, device=device).bfloat16().requires_grad_(True) for h in (6, 2))
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    pos = torch.arange(37, device=device).expand(3, 37).contiguous()
    table = RotaryFrequencies.create(48, interleaved=True, device=device)

    def step():  # no graph of the leaves lives on after it
        out = rotary(q, k, pos, table)
        return (*torch.autograd.grad(out, (q, k), (dq, dk)), *(x.detach() for x in out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for a, b in zip(eager, step()):
        assert torch.equal(a, b)
    for i in range(3):
        pos.add_(1000 + i)
        with torch.no_grad():
            for x in (q, k, dq, dk):
                x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b), i


def test_in_place_is_seen_by_autograd(device):
    pos, table = torch.arange(5, device=device), RotaryFrequencies.create(64, device=device)
    for at in (pos, pos[3:4]):  # one position for all tokens: the general path
        x = torch.randn(5, 2, 64, device=device, requires_grad=True) * 1
        y = (x * x).sum()
        want, _ = rotary(x.detach().clone(), None, at, table)
        with torch.no_grad():
            rotary(x, None, at, table, inplace=True)
        assert torch.equal(x.detach(), want)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()


def test_in_place_views_that_overlap(device):
    base = torch.randn(6, 5, 64, device=device)
    table, pos = RotaryFrequencies.create(64, device=device), torch.arange(6, device=device)
    half = RotaryFrequencies.create(32, device=device)
    for at, freq, views in ((pos, table, lambda x: (x[:, :3], x[:, 2:])), (pos[:5], table, lambda x: (x[:5], x[1:])),
                            (pos[3:4], table, lambda x: (x[:, :3], x[:, 2:])),  # one position for all: the general path
                            (pos, half, lambda x: (x[:, :2, :32], x[:, :2, 16:48])),
                            (pos, table, lambda x: (torch.as_strided(x, (6, 2, 64), (128, 32, 1)), None))):
        x = base.clone()
        with pytest.raises(ValueError, match="memory of their own"):
            rotary(*views(x), at, freq, inplace=True)
        assert torch.equal(x, base) and x._version == 0
    for at in (pos, pos[3:4]):  # heads in turn share no element
        x = base.clone()
        want, _ = rotary(x, None, at, table)
        rotary(x[:, ::2], x[:, 1::2], at, table, inplace=True)
        assert torch.equal(x, want)


def test_forward_mode(device):
    import torch.autograd.forward_ad as fwd

    table, pos = RotaryFrequencies.create(48, interleaved=True, scaling="yarn", factor=4.0, device=device), torch.arange(9, device=device) * 50
    for dtype in (torch.float32, torch.bfloat16):
        q, k, tq, tk = (torch.randn(9, h, 64, device=device, dtype=dtype) for h in (4, 2, 4, 2))
        want, value = rotary(tq, tk, pos, table), rotary(q, k, pos, table)
        for needs in (False, True):  # beside a reverse gradient too
            with fwd.dual_level():
                out = rotary(*(fwd.make_dual(x.detach().clone().requires_grad_(needs), t) for x, t in ((q, tq), (k, tk))), pos, table)
                for got, y, t in zip(out, value, want):
                    primal, tangent = fwd.unpack_dual(got)
                    assert torch.equal(primal, y) and torch.equal(tangent, t) and primal.requires_grad == needs
