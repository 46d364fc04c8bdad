"""Cross attention on the GPU (mimir_amd.cross) against 64 bits.

With u = 2^-8, half a step of bf16: P is rounded to bf16 for P V (u of sum p |v|, the size), the scores' fp32 sums and exp2
add below 2^-12 of P for the inputs here (|s| <= 40 in base 2: 40 * 2^-22 and a few roundings), the sums a few 2^-20; the output
is rounded once (u |out|).  dV: P again (u of sum p |dO|) and its own rounding.  dS is rounded once (u of its size, which
takes dP and delta by their magnitudes) and holds P's 2^-12 and delta, from O with its low half (u^2 of sum |dO| |out|) but
with P's rounding in O (u of sum |dO| sum p |v|, within the size's delta part): 2.1 u of the size together; dQ and dK then
round once (u)."""

import math

import pytest
import torch

from mimir_amd import set_validate_metadata
from mimir_amd.cache import Cache
from mimir_amd.cross import attention_to_states, cross_attention
from oracle import generation_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -8
MORE = 2.0 ** -11  # of the smaller errors


def _near(got, want_size, rel, name):
    want, size = want_size
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    off = (rel * U + MORE) * size + U * want.abs() * 1.02
    bad = ~((got.cpu().double() - want).abs() <= off + 1e-30)
    assert not bad.any(), (name, int(bad.sum()), float((got.cpu().double() - want).abs().max()))


def _make(device, pairs, hq, hkv, d, lead=(0, 0), pad=(0, 0), size=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed + 31 * len(pairs) + d)
    cu_q, cu_k = [lead[0]], [lead[1]]
    for n, m in pairs:
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    rand = lambda *s: torch.randn(*s, generator=gen).clamp_(-4, 4)  # noqa: E731
    q = (size * rand(cu_q[-1] + pad[0], hq, d)).bfloat16().to(device)
    kv = rand(cu_k[-1] + pad[1], 2 * hkv, d).bfloat16().to(device)
    do = rand(q.shape[0], hq, d).bfloat16().to(device)
    return q, kv[:, :hkv], kv[:, hkv:], do, cu_q, cu_k


def _check(device, pairs, hq, hkv, d, grad=True, scale=None, index=torch.int32, **kw):
    q, k, v, do, cu_q, cu_k = _make(device, pairs, hq, hkv, d, **kw)
    lists = [torch.tensor(c, dtype=index, device=device) for c in (cu_q, cu_k)]
    s = 1.0 / math.sqrt(d) if scale is None else scale
    if grad:
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = cross_attention(q, k, v, *lists, softmax_scale=scale)
    want = O.cross_attention(q, k, v, cu_q, cu_k, s, do if grad else None)
    _near(out.detach(), want[0], 1.0, "out")
    if grad:
        got = torch.autograd.grad(out, (q, k, v), do)
        for name, g, w, rel in zip(("dq", "dk", "dv"), got, want[1:], (2.1, 2.1, 1.0)):
            _near(g, w, rel, name)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pairs", [
    [(1, 1)], [(1, 64)], [(3, 65)], [(128, 128)], [(129, 127)], [(33, 200), (200, 33)], [(1, 700)], [(700, 1)], [(64, 63), (65, 64), (31, 129)],
    [(300, 500), (5, 2), (130, 257)]])
def test_lengths(device, d, pairs):
    _check(device, pairs, 4, 2, d)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (8, 1), (16, 4), (6, 3), (12, 4), (9, 3)])
@pytest.mark.parametrize("d", [64, 128])
def test_heads(device, hq, hkv, d):
    _check(device, [(70, 90), (40, 150)], hq, hkv, d)


@pytest.mark.parametrize("d", [64, 128])
def test_empty_sequences_and_padding(device, d):
    _check(device, [(0, 0), (5, 0), (0, 7), (40, 33), (0, 0), (17, 0)], 4, 2, d, pad=(9, 21))
    _check(device, [(0, 70), (130, 0)], 4, 2, d, lead=(3, 5), pad=(1, 1))
    _check(device, [(12, 0)], 2, 1, d)
    _check(device, [(0, 12)], 2, 1, d)
    _check(device, [(20, 30)], 2, 1, d, lead=(140, 200), pad=(300, 131), index=torch.int64)
    _check(device, [], 2, 1, d, pad=(20, 30))
    _check(device, [], 2, 1, d)


def test_many_sequences(device):
    gen = torch.Generator().manual_seed(2)
    pairs = [(int(n), int(m)) for n, m in torch.randint(0, 9, (1500, 2), generator=gen)]
    _check(device, pairs, 2, 1, 64)


def test_larger(device):
    _check(device, [(1100, 1500), (513, 2049)], 8, 2, 128)
    _check(device, [(1100, 1500), (513, 2049)], 4, 4, 64)


@pytest.mark.parametrize("d", [64, 128])
def test_sharp_and_flat_softmax(device, d):
    _check(device, [(80, 300)], 4, 2, d, size=3.0, scale=0.05)
    _check(device, [(80, 300)], 4, 2, d, scale=1e-6)
    _check(device, [(80, 300)], 4, 2, d, scale=1e-20)


def test_low_scores_do_not_overflow_past_the_end(device):
    """All scores near -200 in base 2: a state past the last tile's end would have P = exp2(200)."""
    d = 64
    q = torch.full((40, 2, d), 4.0, device=device, dtype=torch.bfloat16)
    k = torch.full((70, 2, d), -4.0, device=device, dtype=torch.bfloat16)
    k[::3] = -4.03125
    gen = torch.Generator().manual_seed(1)
    v, do = (torch.randn(n, 2, d, generator=gen).bfloat16().to(device) for n in (70, 40))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, *(torch.tensor([0, n], device=device) for n in (40, 70)))
    got = torch.autograd.grad(out, leaves, do)
    want = O.cross_attention(q, k, v, [0, 40], [0, 70], 1 / 8, do)
    for name, g, w, rel in zip(("out", "dq", "dk", "dv"), (out.detach(), *got), want, (1.0, 2.1, 2.1, 1.0)):
        _near(g, w, rel, name)


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 64), (2, 2, 128), (16, 4, 128)])
def test_one_state_has_no_score_gradient(device, hq, hkv, d):
    """P is 1 whatever the score: dQ and dK are exactly 0, beside sequences with more states too."""
    pairs = [(300, 1), (1, 1), (130, 1), (70, 129), (64, 2)]
    q, k, v, do, cu_q, cu_k = _make(device, pairs, hq, hkv, d, lead=(3, 5), pad=(9, 4))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, *(torch.tensor(c, device=device) for c in (cu_q, cu_k)))
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    assert not dq[:cu_q[3]].any() and not dk[:cu_k[3]].any()
    assert dq[cu_q[3]:cu_q[5]].any() and dk[cu_k[3]:cu_k[5]].any() and dv[5:8].any()
    _check(device, pairs, hq, hkv, d, lead=(3, 5), pad=(9, 4))


def test_nan_and_inf_stay_in_their_sequence(device):
    pairs = [(70, 90), (70, 90), (70, 90)]
    q, k, v, do, cu_q, cu_k = _make(device, pairs, 4, 2, 64, pad=(10, 10))
    lists = [torch.tensor(c, device=device) for c in (cu_q, cu_k)]
    clean = cross_attention(q, k, v, *lists)
    k, v = k.clone(), v.clone()
    k[100], v[120] = float("nan"), float("inf")
    k[270:], v[270:], q[210:] = float("nan"), float("nan"), float("nan")
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, *lists)
    grads = torch.autograd.grad(out, leaves, do)
    assert torch.equal(out[:70], clean[:70]) and torch.equal(out[140:210], clean[140:210]) and not out[210:].any()
    assert not torch.isfinite(out[70:140]).any()
    assert torch.isfinite(grads[0][:70]).all() and torch.isfinite(grads[0][140:]).all() and not grads[0][210:].any()
    for g in grads[1:]:
        assert torch.isfinite(g[:90]).all() and torch.isfinite(g[180:]).all() and not g[270:].any()


def test_layouts(device):
    """Heads in front of tokens, rows off their 16 bytes, an expanded gradient, one tensor as query, key and value."""
    gen = torch.Generator().manual_seed(3)
    hold = torch.randn(4, 90, 72, generator=gen).bfloat16().to(device)
    cu = torch.tensor([0, 40, 90], device=device)
    for x in (hold[..., :64].transpose(0, 1), hold[..., 1:65].transpose(0, 1)):
        x = x.detach().requires_grad_(True)
        out = cross_attention(x, x, x, cu, cu)
        dx, = torch.autograd.grad(out.sum(), x)
        want = O.cross_attention(x, x, x, [0, 40, 90], [0, 40, 90], 1 / 8, torch.ones(90, 4, 64))
        _near(out.detach(), want[0], 1.0, "out")
        # three gradients in bf16, added in bf16: two more roundings of the sum so far
        total = sum(w for w, _ in want[1:])
        size = sum(s * r for (_, s), r in zip(want[1:], (2.1, 2.1, 1.0)))
        off = (U + MORE) * size + U * sum(w.abs() for w, _ in want[1:]) * 3.1
        assert ((dx.cpu().double() - total).abs() <= off).all()


def test_only_some_gradients(device):
    q, k, v, do, cu_q, cu_k = _make(device, [(50, 60)], 2, 1, 64)
    lists = [torch.tensor(c, device=device) for c in (cu_q, cu_k)]
    v = v.detach().requires_grad_(True)
    dv, = torch.autograd.grad(cross_attention(q, k, v, *lists), v, do)
    _near(dv, O.cross_attention(q, k, v, cu_q, cu_k, 1 / 8, do)[3], 1.0, "dv")


def test_captured(device):
    q, k, v, do, cu_q, cu_k = _make(device, [(70, 130), (150, 40)], 4, 2, 128)
    lists = [torch.tensor(c, device=device, dtype=torch.int32) for c in (cu_q, cu_k)]
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]

    def step():
        out = cross_attention(*leaves, *lists)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    gen = torch.Generator(device=device).manual_seed(5)
    for i, split in enumerate((100, 10, 220)):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=gen, device=device))
        lists[0].copy_(torch.tensor([0, split, 220]))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), i


def test_same_result_every_time(device):
    q, k, v, do, cu_q, cu_k = _make(device, [(700, 900), (40, 1500), (300, 7)], 8, 2, 128)
    lists = [torch.tensor(c, device=device) for c in (cu_q, cu_k)]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    first = None
    for _ in range(3):
        out = cross_attention(*leaves, *lists)
        got = (out.detach(), *torch.autograd.grad(out, leaves, do))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_refusals(device):
    q, k, v, do, cu_q, cu_k = _make(device, [(5, 6)], 4, 2, 64)
    a, b = (torch.tensor(c, device=device) for c in (cu_q, cu_k))
    for args, error in [((q.float(), k, v, a, b), TypeError), ((q[0], k, v, a, b), ValueError), ((q[:, :3], k, v, a, b), ValueError),
                        ((q, k[:3], v, a, b), ValueError), ((q[..., :32], k, v, a, b), ValueError), ((q, k, v, a[:1], b), ValueError),
                        ((q, k, v, a.float(), b), ValueError), ((q, k.cpu(), v, a, b), ValueError), ((q, k, v, a[:0], b[:0]), ValueError),
                        ((q[..., :32], k[..., :32], v[..., :32], a, b), ValueError), ((q.cpu(), k, v, a, b), RuntimeError)]:
        with pytest.raises(error):
            cross_attention(*args)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softmax_scale"):
            cross_attention(q, k, v, a, b, softmax_scale=scale)
    set_validate_metadata(True)
    try:
        cross_attention(q, k, v, a, b)
        for bad in ([1, 0], [0, 7], [-1, 3]):
            with pytest.raises(ValueError, match="decrease"):
                cross_attention(q, k, v, a, torch.tensor(bad, device=device))
    finally:
        set_validate_metadata(False)


# ---------------------------------------------------------------- rows of a cache of states

def _states(device, requests, beams, S, hq, hkv, d, pool, length, lens, rows, index=torch.int32, seed=0):
    gen = torch.Generator().manual_seed(seed + length)
    rand = lambda *s: torch.randn(*s, generator=gen).bfloat16().to(device)  # noqa: E731
    q, cache = rand(requests * beams, S, hq, d), Cache(rand(pool, length, hkv, d), rand(pool, length, hkv, d))
    return q, cache, torch.tensor(lens, dtype=index, device=device), None if rows is None else torch.tensor(rows, dtype=index, device=device)


def _check_states(q, cache, lens, rows):
    out = attention_to_states(q, cache, lens, rows)
    named = list(range(cache.keys.shape[0])) if rows is None else rows.tolist()
    want = O.attention_to_states(q, cache.keys, cache.values, lens.tolist(), named, 1 / math.sqrt(q.shape[3]))
    _near(out, want, 1.0, "out")
    return out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(4, 4), (16, 4), (8, 1), (9, 3)])
@pytest.mark.parametrize("beams,S", [(1, 1), (4, 1), (3, 5), (16, 1)])
def test_states(device, d, hq, hkv, beams, S):
    lens = [300, 0, 64, 65, 1, 127, 300]
    _check_states(*_states(device, 5, beams, S, hq, hkv, d, 7, 300, lens, [6, 1, 3, 4, 5]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 64, 1000, 5000])
def test_state_lengths(device, d, length):
    _check_states(*_states(device, 3, 2, 1, 8, 2, d, 3, length, [length, length // 2, max(length - 1, 0)], None, index=torch.int64))


@pytest.mark.parametrize("requests", [1, 63, 64, 65, 200])
def test_many_requests(device, requests):
    gen = torch.Generator().manual_seed(requests)
    lens = torch.randint(0, 260, (requests,), generator=gen).tolist()
    rows = torch.randperm(requests, generator=gen).tolist()
    _check_states(*_states(device, requests, 2, 1, 4, 2, 64, requests, 256, lens, rows))  # some lengths past the cache


def test_rows_outside_and_shared(device):
    q, cache, lens, rows = _states(device, 6, 2, 1, 4, 2, 64, 3, 100, [100, 50, -4], [0, -1, 3, 0, 1, 2], index=torch.int64)
    out = _check_states(q, cache, lens, rows)
    assert not out[2:6].any() and not out[10:].any() and out[:2].any()
    rows[1] = (1 << 32) + 1
    _check_states(q, cache, lens, rows)


@pytest.mark.parametrize("d", [64, 128])
def test_many_queries(device, d):
    """More than 128 query rows per kv head: the tile kernel, in place where keys and values lie alike."""
    q, cache, lens, rows = _states(device, 3, 2, 50, 8, 2, d, 4, 400, [400, 0, 130, 77], [2, 0, 1])
    a = _check_states(q, cache, lens, rows)
    hold = torch.randn(4, 2, 400, 2, d, device=device).bfloat16()
    hold[:, 0], hold[:, 1] = cache.keys, cache.values
    assert torch.equal(attention_to_states(q, Cache(hold[:, 0], hold[:, 1]), lens, rows), a)
    wide = torch.zeros(4, 500, 2, d, device=device, dtype=torch.bfloat16)  # keys further apart than values
    wide[:, :400] = cache.keys
    _check_states(q, Cache(wide[:, :400], cache.values), lens, rows)


def test_state_layouts(device):
    gen = torch.Generator().manual_seed(4)
    hold = torch.randn(3, 2, 200, 128, generator=gen).bfloat16().to(device)  # heads in front of positions
    cache = Cache(hold.transpose(1, 2)[..., :64], hold.transpose(1, 2)[..., 64:])
    lens = torch.tensor([200, 150, 3], device=device, dtype=torch.int32)
    q = torch.randn(4, 6, 5, 64, generator=gen).bfloat16().to(device)
    _check_states(q.transpose(1, 2)[:3], cache, lens, None)
    _check_states(q[:3, :1, :2], cache, lens, None)
    odd = torch.randn(3 * 2 * 4 * 64 + 1, generator=gen).bfloat16().to(device)[1:].view(3, 2, 4, 64)  # off 16 bytes
    _check_states(odd, cache, lens, None)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lost", [(0, 64), (0, 700), (32, 64), (100, 900), (300, 1000)])
def test_states_with_scores_of_minus_infinity(device, d, lost):
    """Keys that give -inf take no part, in one part of the states or over whole parts of them."""
    q, cache, lens, _ = _states(device, 1, 2, 1, 4, 2, d, 1, 1000, [1000], None)
    q[..., 0] = 1.0
    cache.keys[:, lost[0]:lost[1], :, 0] = -float("inf")
    _check_states(q, cache, lens, None)
    lists = [torch.tensor([0, n], device=device) for n in (2, 1000)]
    _near(cross_attention(q[:, 0], cache.keys[0], cache.values[0], *lists),
          tuple(t[:, 0] for t in O.attention_to_states(q, cache.keys, cache.values, [1000], [0], 1 / math.sqrt(d))), 1.0, "out")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("requests", [1, 700])
def test_states_past_the_caches(device, d, requests):
    """A cache of 2^28 bytes and more (by its rows and positions) of which little is held, or all by one request."""
    length = (1 << 28) // (requests * 4 * d) + 1
    if requests == 1:
        q, cache, lens, _ = _states(device, 1, 1, 1, 1, 1, d, 1, length, [length], None)
        keys, values = cache.keys[0, :, 0].double().cpu(), cache.values[0, :, 0].double().cpu()
        p = torch.softmax(keys @ q[0, 0, 0].double().cpu() / math.sqrt(d), dim=0)
        _near(attention_to_states(q, cache, lens)[0, 0, 0], (p @ values, p @ values.abs()), 1.0, "out")
        return
    lens = [min(length, (37 * i) % 300) for i in range(requests)]
    _check_states(*_states(device, requests, 2, 1, 2, 1, d, requests, length, lens, None))


def test_expanded_queries(device):
    """One query for all batch rows, for all tokens, for all heads: strides of 0 (read as given)."""
    q, cache, lens, _ = _states(device, 3, 2, 1, 4, 2, 64, 3, 90, [90, 5, 70], None)
    a = _check_states(q[:1].expand(6, -1, -1, -1), cache, lens, None)
    assert torch.equal(a, attention_to_states(q[:1].repeat(6, 1, 1, 1), cache, lens))
    _check_states(q.expand(-1, 5, -1, -1), cache, lens, None)
    _check_states(q[:1].expand(6, 5, -1, -1), cache, lens, None)
    _check_states(q[:, :, :1].expand(-1, -1, 4, -1), cache, lens, None)
    one = Cache(*(t[:, :1].expand(-1, 90, -1, -1) for t in cache))  # one state at all positions
    with pytest.raises(ValueError, match="position stride"):
        attention_to_states(q, one, lens)


def test_states_agree_with_packed_queries(device):
    q, cache, lens, rows = _states(device, 2, 4, 1, 16, 4, 128, 2, 600, [600, 345], None)
    out = attention_to_states(q, cache, lens)
    cu_q, cu_k = torch.tensor([0, 4, 8], device=device), torch.tensor([0, 600, 945], device=device)
    k, v = (torch.cat((t[0], t[1, :345])) for t in cache)
    other = cross_attention(q[:, 0], k, v, cu_q, cu_k)
    # both within u of sum p |v|, twice, and two roundings of the output
    size = O.attention_to_states(q, cache.keys, cache.values, [600, 345], [0, 1], 1 / math.sqrt(128))[1]
    assert ((out[:, 0].double() - other.double()).cpu().abs() <= 2 * (U + MORE) * size[:, 0] + 2.04 * U * out[:, 0].double().cpu().abs()).all()


def test_states_captured(device):
    q, cache, lens, rows = _states(device, 3, 2, 1, 8, 2, 128, 5, 700, [700, 1, 350, 0, 64], [0, 2, 4])
    attention_to_states(q, cache, lens, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = attention_to_states(q, cache, lens, rows)
    gen = torch.Generator(device=device).manual_seed(1)
    for new in ([1, 3, 0], [4, 4, 2], [0, 1, 2]):
        q.copy_(torch.randn(q.shape, device=device, generator=gen))
        rows.copy_(torch.tensor(new))
        lens.add_(3)
        want = attention_to_states(q, cache, lens, rows)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_states_refusals(device):
    q, cache, lens, rows = _states(device, 2, 2, 1, 4, 2, 64, 3, 10, [1, 2, 3], [0, 1])
    for args, error in [((q[0], cache, lens, rows), ValueError), ((q.float(), cache, lens, rows), TypeError), ((q, cache, lens[:2], rows), ValueError),
                        ((q, cache, lens, None), ValueError), ((q, cache, lens, rows[:0]), ValueError), ((q, cache, lens.float(), rows), ValueError),
                        ((q, cache, lens.cpu(), rows), ValueError), ((q[:, :, :3], cache, lens, rows), ValueError),
                        ((q, Cache(cache.keys[..., :32], cache.values), lens, rows), ValueError),
                        ((q, Cache(cache.keys, cache.values[:, :5]), lens, rows), ValueError),
                        ((q[..., :56], Cache(cache.keys[..., 1:57], cache.values[..., 1:57]), lens, rows), ValueError),
                        ((q.cpu(), Cache(*(t.cpu() for t in cache)), lens.cpu(), rows.cpu()), RuntimeError)]:
        with pytest.raises(error):
            attention_to_states(*args)
    with pytest.raises(ValueError, match="no gradient"):
        attention_to_states(q.clone().requires_grad_(True), cache, lens, rows)
    set_validate_metadata(True)
    try:
        with pytest.raises(IndexError):
            attention_to_states(q, cache, lens, torch.tensor([0, 3], device=device))
    finally:
        set_validate_metadata(False)


def test_lists_that_decrease_stay_in_their_workspace(device):
    """Lists up and down name more tiles than 32 bits count (2^18 sequences of 2^20 rows, 8192 tiles each): nothing is listed,
    nothing around the workspace is written, and calls after it are right."""
    import ctypes

    from mimir_amd import _capi

    total, n = 1 << 20, (1 << 19) + 2
    q = torch.zeros(total, 1, 64, dtype=torch.bfloat16, device=device)
    k, v = (torch.randn(200, 1, 64, device=device).bfloat16() for _ in range(2))
    up_down = torch.arange(n + 1, device=device) % 2
    cu_q, cu_k = (total * up_down).int(), (200 * up_down).int()
    out, lo = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.zeros(1, total, device=device)
    p = _capi.CrossParams()
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    for name, t in zip(("q", "k", "v", "out", "dout", "dq", "dk", "dv"), (q, k, v, out, q, *grads)):
        setattr(p, name, t.data_ptr())
        setattr(p, name + "_stride_token", 64)
    p.out_lo, p.lse2, p.cu_seqlens_q, p.cu_seqlens_k = lo.data_ptr(), lse.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr()
    p.total_q, p.total_k, p.numseqs, p.num_q_heads, p.num_kv_heads, p.head_dim = total, 200, n, 1, 1, 64
    p.dtype, p.softmax_scale = _capi.DTYPE_BFLOAT16, 0.125
    lib = _capi.load()
    for backward, entry in ((0, lib.mimir_prefixlm_cross_fwd), (1, lib.mimir_prefixlm_cross_bwd)):
        size = lib.mimir_prefixlm_cross_workspace_bytes(ctypes.byref(p), backward)
        hold = torch.full((size + (1 << 21),), 0x5a, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = hold.data_ptr() + (1 << 20), size
        _capi.raise_for_status(lib, entry(ctypes.byref(p), torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert (hold[:1 << 20] == 0x5a).all() and (hold[(1 << 20) + size:] == 0x5a).all()
        assert not hold[1 << 20:(1 << 20) + 16 * (total // 128 + n)].any()  # the list of query tiles: nothing
    assert not out.any()
    _check(device, [(1100, 1500), (513, 2049)], 4, 4, 64)


@pytest.mark.parametrize("native", [True, False])
def test_rows_far_apart(device, monkeypatch, native):
    """The last tokens of sequences of 2^22 elements and more, one of each: queries, states and gradients 2^22 apart and further."""
    from mimir_amd import _capi

    if not native:
        monkeypatch.setattr(_capi, "_host", _capi._GeneralPath)
    gen = torch.Generator().manual_seed(8)
    hold = torch.zeros(4, 2 << 22, dtype=torch.bfloat16, device=device)

    def far(n, heads, step):
        t = hold.as_strided((n, heads, 64), (step, 64, 1), 64 * far.used)
        far.used += heads
        return t.copy_(torch.randn(n, heads, 64, generator=gen).bfloat16())

    for step, n in ((1 << 22, 5), ((1 << 22) + 64, 5), (1 << 23, 1)):
        far.used = 0
        q, k, v, do = (far(n, h, step).detach().requires_grad_(True) for h in (4, 2, 2, 4))
        near = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in (q, k, v, do)]
        cu = torch.tensor([0, n // 2, n], dtype=torch.int32, device=device)
        results = []
        for leaves in ((q, k, v, do), near, (*near[:3], do)):
            out = cross_attention(*leaves[:3], cu, cu)
            results.append([out, *torch.autograd.grad(out, leaves[:3], leaves[3])])
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*results))
        states = Cache(torch.randn(n, 40, 2, 64, device=device).bfloat16(), torch.randn(n, 40, 2, 64, device=device).bfloat16())
        lens = torch.full((n,), 33, device=device)
        assert torch.equal(*(attention_to_states(t.detach()[:, None], states, lens) for t in (q, near[0])))
