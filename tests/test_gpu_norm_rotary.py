"""Normed rotary heads on the GPU (mimir_amd.rotary.norm_rotary) against 64 bits.

The kernel's r = 1 / sqrt(mean(x^2) + eps): the sum's chain is at most 16 products a lane and 6 adds across lanes,
24 roundings of 2^-24 with the mean and eps, which the root halves, and rsqrt's 2^-23: below 2^-20.  With r w, x (r w) and the
turn's 2^-21 of |a| + |b| (test_gpu_rotary.py) an output is off by at most 2^-19 of its pair's size.  The gradient holds r
three times, two sums and the turn: below 2^-18 of the same formula with magnitudes.  A weight's gradient sums at most 70 terms
in a chain here (16 in registers, 32 groups, 16 rows, 6 levels), 70 * 2^-24 < 2^-17, on top of its terms' 2^-18: 2^-16.
Rounding to bf16 adds half a step, 2^-8."""

import pytest
import torch

from mimir_amd.rotary import RotaryFrequencies, norm_rotary, rotary
from oracle import generation_oracle as O

pytestmark = pytest.mark.gpu


def _near(got, want_size, rel, name):
    want, size = want_size
    off = rel * size
    off = off + (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24) * (want.abs() + off)
    bad = ~((got.cpu().double() - want).abs() <= off)
    assert not bad.any(), (name, int(bad.sum()), float((got.cpu().double() - want).abs().max()))


def _check(device, lead, hq, hkv, d, rd, dtype, interleaved=False, wtype=None, eps=1e-6, max_pos=5000, index=torch.int64, grad=True, **kw):
    gen = torch.Generator().manual_seed(rd * 7 + d)
    tokens = 1
    for n in lead:
        tokens *= n
    rand = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    qkv = (rand(*lead, hq + 2 * hkv, d) * torch.exp(2.0 * rand(*lead, 1, 1))).to(dtype).to(device)
    q, k = qkv[..., :hq, :].detach(), qkv[..., hq:hq + hkv, :].detach()
    wq, wk = ((1.0 + 0.3 * rand(d)).to(wtype or dtype).to(device) for _ in range(2))
    pos = torch.randint(0, max_pos, lead, generator=gen).to(index)
    freq, amplitude = RotaryFrequencies.inverse_frequencies(rd, **kw)
    table = RotaryFrequencies.create(rd, interleaved=interleaved, device=device, **kw)
    leaves = [t.requires_grad_(grad) for t in (q, k, wq, wk)]
    out = norm_rotary(q, k, pos.to(device), table, wq, wk, eps=eps)
    flat = lambda t: t.detach().reshape(tokens, -1, d)  # noqa: E731
    args = (pos.reshape(-1), freq, amplitude, interleaved, eps)
    for name, x, w, y in (("q", q, wq, out[0]), ("k", k, wk, out[1])):
        assert y.shape == x.shape and y.dtype == dtype and y.is_contiguous()
        _near(flat(y), O.norm_rotary(flat(x), w, *args), 2.0 ** -19, name)
    if grad:
        dout = [rand(*y.shape).to(dtype).to(device) for y in out]
        got = torch.autograd.grad(out, leaves, dout)
        for name, g, x, w, dx, dw in (("q", dout[0], q, wq, got[0], got[2]), ("k", dout[1], k, wk, got[1], got[3])):
            assert dx.dtype == dtype and dw.dtype == w.dtype
            want_x, want_w = O.norm_rotary_grad(flat(g), flat(x), w, *args)
            _near(flat(dx), want_x, 2.0 ** -18, "d" + name)
            _near(dw, want_w, 2.0 ** -16, "weight of " + name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rd", [(128, 128), (64, 64), (64, 20), (128, 64), (96, 96), (80, 32), (64, 2), (128, 26), (6, 4), (128, 126),
                                  (256, 128), (2, 2)])
def test_layouts_and_parts(device, dtype, interleaved, d, rd):
    _check(device, (3, 37), 4, 2, d, rd, dtype, interleaved)


@pytest.mark.parametrize("lead", [(1,), (1, 1), (5, 1), (1, 700), (4099,), (2, 3)])
def test_token_counts(device, lead):
    _check(device, lead, 16, 4, 128, 128, torch.bfloat16, index=torch.int32, wtype=torch.float32)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (32, 8), (7, 1), (40, 8), (1, 8)])
def test_heads(device, hq, hkv):
    _check(device, (2, 65), hq, hkv, 64, 64, torch.float32, True)


@pytest.mark.parametrize("scaling", ["linear", "yarn"])
def test_scaled_ranges(device, scaling):
    _check(device, (2, 50), 4, 2, 128, 128, torch.float32, scaling=scaling, factor=16.0, original_positions=4096, max_pos=1 << 20)


def test_large_eps_and_zero_rows(device):
    _check(device, (2, 9), 4, 2, 64, 64, torch.float32, eps=0.5)
    table, pos = RotaryFrequencies.create(64, device=device), torch.arange(5, device=device)
    x = torch.zeros(5, 2, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    y, _ = norm_rotary(x, None, pos, table, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert not y.any() and not dw.any() and torch.isfinite(dx).all()
    want, _ = O.norm_rotary_grad(torch.ones(5, 2, 64), torch.zeros(5, 2, 64), None, pos, RotaryFrequencies.inverse_frequencies(64)[0], 1.0,
                                 False, 1e-6)
    _near(dx, want, 2.0 ** -18, "dx")


def test_without_weights_or_key(device):
    gen = torch.Generator(device=device).manual_seed(3)
    q = torch.randn(33, 4, 64, device=device, generator=gen)
    table, pos = RotaryFrequencies.create(32, device=device), torch.arange(33, device=device)
    freq = RotaryFrequencies.inverse_frequencies(32)[0]
    y, none = norm_rotary(q, None, pos, table)
    assert none is None
    _near(y, O.norm_rotary(q, None, pos, freq, 1.0, False, 1e-6), 2.0 ** -19, "y")
    q.requires_grad_(True)
    y, _ = norm_rotary(q, None, pos, table)
    dx, = torch.autograd.grad(y, q, torch.ones_like(y))
    _near(dx, O.norm_rotary_grad(torch.ones_like(y), q, None, pos, freq, 1.0, False, 1e-6)[0], 2.0 ** -18, "dx")
    # a weight on one side only
    wk = torch.rand(64, device=device, requires_grad=True)
    yq, yk = norm_rotary(q, q.detach(), pos, table, None, wk)
    dw, = torch.autograd.grad((yq, yk), wk, (torch.ones_like(yq), torch.ones_like(yk)))
    _near(dw, O.norm_rotary_grad(torch.ones_like(y), q, None, pos, freq, 1.0, False, 1e-6)[1], 2.0 ** -16, "dw")


def test_unused_output(device):
    q, k = (torch.randn(9, 2, 64, device=device, requires_grad=True) for _ in range(2))
    w = torch.ones(64, device=device, requires_grad=True)
    table, pos = RotaryFrequencies.create(64, device=device), torch.arange(9, device=device)
    y, _ = norm_rotary(q, k, pos, table, w, w)
    dq, dk, dw = torch.autograd.grad(y.sum(), (q, k, w))
    assert dq.any() and not dk.any()
    want = O.norm_rotary_grad(torch.ones(9, 2, 64), q, None, pos, RotaryFrequencies.inverse_frequencies(64)[0], 1.0, False, 1e-6)[1]
    _near(dw, want, 2.0 ** -16, "dw")


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_strides(device, offset):
    """Heads in front of tokens, rows of odd length, addresses off 16 bytes, a broadcast gradient."""
    gen = torch.Generator().manual_seed(offset)
    hold = torch.randn(2, 3, 21, 70, generator=gen).to(device)
    q = hold[..., offset:offset + 64].transpose(1, 2)           # [2, 21, 3, 64]
    k = hold[:, :1, :, offset:offset + 64].transpose(1, 2).expand(2, 21, 2, 64)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    table, pos = RotaryFrequencies.create(64, interleaved=True, device=device), torch.arange(21, device=device)
    freq = RotaryFrequencies.inverse_frequencies(64)[0]
    y, z = norm_rotary(q, k, pos, table)
    dq, dk = torch.autograd.grad((y.sum(), z.sum()), (q, k))  # gradients are expanded scalars
    both = pos.cpu().repeat(2)
    for x, out, dx in ((q, y, dq), (k, z, dk)):
        flat = x.detach().reshape(42, -1, 64)
        _near(out.detach().reshape(flat.shape), O.norm_rotary(flat, None, both, freq, 1.0, True, 1e-6), 2.0 ** -19, "y")
        _near(dx.reshape(flat.shape), O.norm_rotary_grad(torch.ones_like(flat), flat, None, both, freq, 1.0, True, 1e-6)[0], 2.0 ** -18, "dx")


def test_empty(device):
    w = torch.ones(64, device=device, requires_grad=True)
    q = torch.zeros(2, 0, 4, 64, device=device, requires_grad=True)
    y, _ = norm_rotary(q, None, torch.zeros(2, 0, dtype=torch.long, device=device), RotaryFrequencies.create(64, device=device), w)
    dq, dw = torch.autograd.grad(y.sum(), (q, w))
    assert y.shape == q.shape and dq.shape == q.shape and not dw.any()


def test_weight_one_is_rotary_of_the_normed(device):
    x = torch.randn(50, 4, 128, device=device)
    table, pos = RotaryFrequencies.create(128, device=device), torch.arange(50, device=device)
    y, _ = norm_rotary(x, None, pos, table, torch.ones(128, device=device))
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    # 2^-19 on this side, the norm's rounding 2^-20 and the turn's 2^-21 on the other, of pairs of at most 2 max |n|
    assert (y - rotary(n, None, pos, table)[0]).abs().max() <= 2.0 ** -18 * 2 * n.abs().max()


def test_captured_and_on_a_side_stream(device):
    gen = torch.Generator(device=device).manual_seed(5)
    q, k = (torch.randn(64, h, 128, device=device, dtype=torch.bfloat16, generator=gen, requires_grad=True) for h in (8, 2))
    wq, wk = (torch.rand(128, device=device, generator=gen, requires_grad=True) for _ in range(2))
    table, pos = RotaryFrequencies.create(128, device=device), torch.arange(64, device=device)

    def step():
        out = norm_rotary(q, k, pos, table, wq, wk)
        return (*out, *torch.autograd.grad(out, (q, k, wq, wk), [torch.ones_like(t) for t in out]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, device=device, generator=gen))
            wk.copy_(torch.rand(128, device=device, generator=gen))
        want = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), seed


def test_same_result_every_time(device):
    gen = torch.Generator(device=device).manual_seed(6)
    q = torch.randn(3000, 8, 128, device=device, dtype=torch.bfloat16, generator=gen, requires_grad=True)
    w = torch.rand(128, device=device, generator=gen, requires_grad=True)
    table, pos = RotaryFrequencies.create(128, device=device), torch.arange(3000, device=device)
    first = None
    for _ in range(3):
        y, _ = norm_rotary(q, None, pos, table, w)
        got = torch.autograd.grad(y, (q, w), torch.ones_like(y))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_misaligned_heads_past_the_lanes_are_refused(device):
    x = torch.randn(4, 2, 256, device=device, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="columns at a time"):
        norm_rotary(x, None, torch.arange(4, device=device), RotaryFrequencies.create(2, device=device))


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 256), (torch.bfloat16, 640), (torch.float32, 256), (torch.float32, 512), (torch.bfloat16, 128)])
def test_gradients_off_their_alignment(device, monkeypatch, native, dtype, d):
    """A forward that ran has a backward, whatever the layout of the gradients that come."""
    from mimir_amd import _capi

    if not native:
        monkeypatch.setattr(_capi, "_host", _capi._GeneralPath)
    gen = torch.Generator(device=device).manual_seed(d)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device).to(dtype)  # noqa: E731
    leaves = [rand(7, 3, d).requires_grad_(True), rand(7, 1, d).requires_grad_(True), rand(d).requires_grad_(True)]
    table, pos = RotaryFrequencies.create(d, device=device), torch.arange(7, device=device)
    out = norm_rotary(leaves[0], leaves[1], pos, table, leaves[2], leaves[2])
    dout = [rand(*y.shape) for y in out]
    want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    odd = [torch.zeros(1 + 7 * (y.shape[1] * d + 3), dtype=dtype, device=device)[1:].view(7, -1)[:, :y.shape[1] * d].view(y.shape) for y in out]
    fine = [torch.zeros(7, d, y.shape[1], dtype=dtype, device=device).transpose(1, 2) for y in out]  # no unit stride
    # Past 128 columns the copies are read as the aligned gradients were.  Up to there they are read by other accesses, whose sums
    # add in another order: 2^-18 of sizes below 16 either way, and each rounded once, to neighbours 2^-7 apart at most.
    for views in (odd, fine):
        for view, g in zip(views, dout):
            view.copy_(g)
        got = torch.autograd.grad(out, leaves, views, retain_graph=True)
        assert all(torch.equal(a, b) if d > 128 else torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -13) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_of_one_entry(device, dtype):
    """[tokens, D, 1] transposed, and any stride for a dim of one entry: read as if it were contiguous."""
    gen = torch.Generator(device=device).manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device).to(dtype)  # noqa: E731
    table = RotaryFrequencies.create(256, device=device)
    for tokens, strides in ((5, (256, 1, 1)), (5, (264, 3, 1)), (1, (1, 7, 1))):
        q, k, dq, dk = (rand(tokens, 1, 256) for _ in range(4))
        odd = [torch.zeros(1 << 12, dtype=dtype, device=device).as_strided(q.shape, strides).copy_(t) for t in (q, k, dq, dk)]
        pos = torch.arange(tokens, device=device)
        results = []
        for a, b, da, db in ((q, k, dq, dk), odd):
            leaves = [a.detach().requires_grad_(True), b.detach().requires_grad_(True)]
            out = norm_rotary(*leaves, pos, table)
            results.append([*out, *torch.autograd.grad(out, leaves, (da, db))])
        assert all(torch.equal(x, y) for x, y in zip(*results))
