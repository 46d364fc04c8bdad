"""The 8-bit paged cache and its attention (mimir_amd.paged) against the 64-bit oracle.

Codes and exponents must be the oracle's exactly, and every page that the call does not append
to as it was.  Outputs: the bound that the oracle derives element by element (its ``attend``).
The pool starts full of NaN codes but for the tokens held, so anything read past them shows."""

import pytest
import torch

import mimir_amd
from mimir_amd.paged import PAGE_TOKENS, PagedCache, attention_with_pages
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _pool(lens, room, hkv, d, layers, gen, extra=3, spread=1.0):
    """A pool whose rows hold lens tokens in scattered pages with room for `room` more; unwritten slots are NaN codes."""
    need = [-(-(n + r) // PAGE_TOKENS) for n, r in zip(lens, room)]
    pages = torch.randperm(sum(need) + extra, generator=gen).tolist()
    width = max(max(need), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    shape = (len(pages), layers, hkv)
    keys = torch.full((*shape, PAGE_TOKENS, d), 127, dtype=torch.uint8)
    values = torch.full((*shape, d, PAGE_TOKENS), 127, dtype=torch.uint8)
    exps = [torch.randint(-8, -3, shape, generator=gen, dtype=torch.int8) for _ in range(2)]
    at = 0
    for b, n in enumerate(need):
        for i in range(n):
            p = pages[at]
            at += 1
            table[b, i] = p
            held = max(0, min(PAGE_TOKENS, lens[b] - i * PAGE_TOKENS))
            x = torch.randn(2, layers, hkv, held, d, generator=gen) * 200 * spread
            codes = x.clamp(-440, 440).to(torch.float8_e4m3fn).view(torch.uint8)
            keys[p, :, :, :held] = codes[0]
            values[p, :, :, :, :held] = codes[1].transpose(-1, -2)
    f8 = torch.float8_e4m3fn
    return PagedCache(keys.view(f8), values.view(f8), *exps), table


def _move(x, device):
    return x.view(torch.uint8).to(device).view(x.dtype) if x.dtype == torch.float8_e4m3fn else x.to(device)


def _compare(cache, want, label):
    for name, got, x in zip(PagedCache._fields, cache, (want.keys, want.values, want.ke, want.ve)):
        g = got.detach().cpu()
        g = (g.view(torch.uint8) if g.dtype == torch.float8_e4m3fn else g).numpy()
        if x.dtype == "uint8":  # NaN codes of either sign are one
            g, x = (g | (0x80 * ((g & 127) == 127)).astype("uint8")), (x | (0x80 * ((x & 127) == 127)).astype("uint8"))
        assert (g == x).all(), (label, name, int((g != x).sum()))


def _near(out, want, tol, label):
    import numpy as np

    got = out.detach().cpu().double().numpy()
    assert (np.isnan(got) == np.isnan(want)).all(), (label, "NaN", int(np.isnan(got).sum()), int(np.isnan(want).sum()))
    bad = ~(np.abs(got - want) <= tol + 1e-30) & ~np.isnan(want)
    assert not bad.any(), (label, int(bad.sum()), np.abs(got - want)[bad].max())


def _run(device, S, hq, hkv, d, lens, causal=True, new=None, rows=None, layers=1, layer=0, seed=0, index=torch.int32, edit=None,
         scale=None, extra_rows=0, grow=1.0, width=None, room=None):
    gen = torch.Generator().manual_seed(seed)
    B = len(lens)
    cache, table = _pool(lens, room or [S] * B, hkv, d, layers, gen)
    if width is not None:
        table = torch.cat((table, torch.full((B, max(0, width - table.shape[1])), -1, dtype=torch.int32)), 1)[:, :width].contiguous()
    order = None
    if rows is not None:  # batch row b is table row rows[b]
        order = torch.tensor(rows, dtype=index)
        big = torch.full((max(rows) + 1 + extra_rows, table.shape[1]), -1, dtype=torch.int32)
        for b, r in enumerate(rows):
            if r >= 0:
                big[r] = table[b]
        table = big
    q = torch.randn(B, S, hq, d, generator=gen).to(BF16)
    k, v = ((torch.randn(B, S, hkv, d, generator=gen) * grow).to(BF16) for _ in range(2))
    lengths = torch.tensor(lens, dtype=index)
    fresh = None if new is None else torch.tensor(new, dtype=index)
    if edit is not None:
        edit(locals())
    want = O.Cache(*cache)
    ref, tol = want.attend(q, k, v, layer, table, lengths, causal, order, fresh, scale)
    dev = PagedCache(*(_move(x, device) for x in cache))
    to = lambda x: None if x is None else x.to(device)  # noqa: E731
    label = f"S={S} hq={hq} hkv={hkv} d={d} lens={lens[:8]} causal={causal} new={new and new[:8]} seed={seed}"
    print("[paged]", label, flush=True)
    out = attention_with_pages(q.to(device), k.to(device), v.to(device), dev, layer, to(table), to(lengths), causal, to(order),
                               new_lengths=to(fresh), softmax_scale=scale)
    torch.cuda.synchronize()
    _compare(dev, want, label)
    _near(out, ref, tol, label)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("hq,hkv", [(16, 4), (8, 8), (2, 2), (8, 1), (16, 1)])
def test_decode(device, d, hq, hkv):
    _run(device, 1, hq, hkv, d, [0, 1, 62, 63, 64, 65, 777, 1499], seed=hq + hkv)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("S,causal", [(2, True), (3, False), (4, True), (5, True), (8, False)])
def test_short_chunks(device, d, S, causal):
    """Up to 32 query rows per kv head: the decode kernel with one or two row tiles; 4 rows a token."""
    _run(device, S, 8, 2, d, [0, 61, 63, 64, 130, 900], causal, seed=S)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("S,causal,lens", [(9, True, [0, 1, 63, 64, 500]), (17, False, [63, 40]), (64, True, [0, 64, 33]), (65, False, [0, 63, 100]),
                                           (130, True, [5, 0, 700]), (257, True, [60])])
def test_prefill(device, d, S, causal, lens):
    _run(device, S, 8, 2, d, lens, causal, seed=S)


@pytest.mark.parametrize("hq,hkv", [(3, 1), (6, 6), (5, 5), (40, 1), (12, 4)])
@pytest.mark.parametrize("S", [1, 21])
def test_odd_heads(device, S, hq, hkv):
    _run(device, S, hq, hkv, 64, [30, 64, 191], seed=hq)


@pytest.mark.parametrize("S,new", [(1, [1, 0, 1, 0]), (4, [4, 0, 1, 3]), (40, [40, 0, 1, 23]), (129, [5, 129, 0, 64])])
@pytest.mark.parametrize("causal", [True, False])
def test_padded_batches(device, S, new, causal):
    """Queries past new_lengths give zeros, their keys are not appended, rows of 0 are left alone."""
    def poison(x):
        for b, n in enumerate(new):
            for t in ("q", "k", "v"):
                x[t][b, n:] = float("nan")
    _run(device, S, 8, 2, 128, [100, 50, 0, 64], causal, new=new, edit=poison)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_table_rows_layers_and_index_types(device, index):
    _run(device, 1, 8, 2, 128, [5, 100, 64], rows=[4, 0, 2], layers=3, layer=1, index=index, extra_rows=2)
    _run(device, 20, 8, 2, 64, [5, 100, 64], rows=[4, 0, 2], layers=3, layer=2, index=index, new=[20, 3, 0])


@pytest.mark.parametrize("S", [1, 30])
def test_rows_outside(device, S):
    """Rows outside the table, negative lengths, missing pages and lengths past the table: zeros, dropped
    tokens and unseen keys, and nothing else is touched."""
    def edit(x):
        x["order"][1] = 77
        x["order"][2] = -1
        x["lengths"][3] = -5
        x["table"][4, 1] = -1
        x["table"][5, 0] = 1 << 20
    _run(device, S, 8, 2, 128, [10, 20, 30, 40, 300, 90, 10], rows=[0, 1, 2, 3, 4, 5, 6], edit=edit)
    _run(device, S, 8, 2, 128, [128, 125, 64, 1000], width=2, room=[0, 3, 64, 0])


@pytest.mark.parametrize("batch,hkv", [(300, 2), (256, 1), (257, 4)])
def test_many_rows(device, batch, hkv):
    """Past 256 batch rows a pair of row and head takes a workgroup; up to there the pages are dealt out."""
    gen = torch.Generator().manual_seed(batch)
    _run(device, 1, 4 * hkv, hkv, 64, torch.randint(0, 700, (batch,), generator=gen).tolist(), seed=batch)


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("S", [1, 3, 8])
def test_wide_tables(device, S, d):
    """Tables much wider than the rows are long: their pages are dealt to shares whatever their number, with new
    tokens in the last page of a share, padded rows, rows without keys, and NaN tokens."""
    lens = [0, 1, 62, 63, 64, 65, 777, 1499, 255, 256, 257]
    _run(device, S, 8, 2, d, lens, width=1100, seed=S)
    _run(device, S, 8, 2, d, lens, False, new=[S, 0, 1, S, 0, S, S, max(S - 1, 1), S, 0, S], width=1100, seed=S)

    def edit(x):
        x["v"][6, S - 1, 1, 5] = float("nan")
        x["k"][7, S // 2, 0] = float("inf")
        x["order"][2] = -1
        x["lengths"][5] = -1
        x["table"][6, 3] = -1
    _run(device, S, 8, 2, d, lens, rows=list(range(11)), width=1100, edit=edit, grow=20.0)


@pytest.mark.parametrize("batch", [64, 65, 129, 256])
def test_many_rows_in_a_wide_table(device, batch):
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 900, (batch,), generator=gen).tolist()
    new = torch.randint(0, 2, (batch,), generator=gen).tolist()
    _run(device, 1, 4, 1, 64, lens, seed=batch, width=600)
    _run(device, 1, 4, 1, 64, lens, seed=batch, width=600, new=new)


@pytest.mark.parametrize("S,hq", [(1, 8), (3, 8), (6, 8), (33, 8)])
def test_long_rows(device, S, hq):
    """A long row cut into many shares (more than 64 pages for a wave), beside short ones."""
    _run(device, S, hq, 2, 64, [30011, 3, 0, 500], seed=S)


@pytest.mark.parametrize("S", [1, 7, 50])
@pytest.mark.parametrize("grow", [1e-3, 30.0, 1e5, 1e30, 1e-30])
def test_scales_grow(device, S, grow):
    """New tokens of other magnitudes: a page's older codes are rounded again, or its new ones fall below its scale."""
    _run(device, S, 8, 2, 64, [60, 10, 64], grow=grow, seed=3)


@pytest.mark.parametrize("S", [2, 8, 12, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nan_and_infinite_tokens(device, S, bad):
    """Stored as NaN; a causal query before such a token does not see it, one after it does."""
    def edit(x):
        x["v"][0, S // 2, 0, 3] = bad
        x["v"][1, S - 1, 1, 63] = bad
        x["k"][2, S // 2, 1, 0] = bad
        x["k"][3, S - 1] = bad
        x["v"][3, 0] = bad
    _run(device, S, 8, 2, 64, [63, 0, 100, 64], edit=edit)


def test_nan_queries_stay_in_their_rows(device):
    def edit(x):
        x["q"][0, 0, 3] = float("nan")
        x["q"][1, 0, 5, 2] = float("nan")
    _run(device, 1, 8, 2, 128, [700, 70], edit=edit)
    _run(device, 40, 8, 2, 128, [700, 70], edit=edit)


def test_zeros_and_tiny_scales(device):
    def edit(x):
        x["k"].zero_()
        x["v"].zero_()
    _run(device, 1, 8, 2, 128, [0, 64, 63], edit=edit)
    _run(device, 1, 8, 2, 128, [100, 64], scale=1e-38)
    _run(device, 40, 8, 2, 128, [100, 64], scale=1e-38)
    _run(device, 1, 8, 2, 128, [100, 64], scale=3.0)


def test_strided_operands(device):
    """q, k, v as views of a fused projection; a page table that is a view of a wider one."""
    gen = torch.Generator().manual_seed(5)
    cache, table = _pool([100, 7], [30, 30], 2, 64, 1, gen)
    for S in (1, 30):
        qkv = torch.randn(2, S, 12, 64, generator=gen).to(BF16)
        want = O.Cache(*cache)
        ref, tol = want.attend(qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:], 0, table, torch.tensor([100, 7]), True)
        dev = PagedCache(*(_move(x, device) for x in cache))
        x = qkv.to(device)
        wide = torch.full((2, 9), -1, dtype=torch.int32, device=device)
        wide[:, 2:2 + table.shape[1]] = table.to(device)
        out = attention_with_pages(x[:, :, :8], x[:, :, 8:10], x[:, :, 10:], dev, 0, wide[:, 2:2 + table.shape[1]],
                                   torch.tensor([100, 7], device=device), True)
        _compare(dev, want, S)
        _near(out, ref, tol, S)


def test_pages_past_four_gib(device):
    """Page numbers whose bytes pass 32 bits, keys and values."""
    pages, hkv, d = 300_000, 2, 128  # 16 KiB a page
    cache = PagedCache.create(pages, 1, hkv, d, device=device)
    gen = torch.Generator().manual_seed(1)
    small, small_table = _pool([150], [1], hkv, d, 1, gen)
    far = torch.tensor([299_999, 262_144, 280_001])
    for x, y in zip(cache, small):
        raw, src = (t.view(torch.uint8) for t in (x, y))
        raw[far.to(device)] = src[small_table[0, :3].long()].to(device)
    q, k, v = (torch.randn(1, 1, h, d, generator=gen).to(BF16) for h in (8, hkv, hkv))
    want = O.Cache(*small)
    ref, tol = want.attend(q, k, v, 0, small_table, torch.tensor([150]), True)
    table = far.int()[None].to(device)
    out = attention_with_pages(q.to(device), k.to(device), v.to(device), cache, 0, table, torch.tensor([150], device=device), True)
    _near(out, ref, tol, "far")
    q, k, v = (torch.randn(1, 20, h, d, generator=gen).to(BF16) for h in (8, hkv, hkv))
    ref, tol = want.attend(q, k, v, 0, small_table, torch.tensor([150]), True)
    out = attention_with_pages(q.to(device), k.to(device), v.to(device), cache, 0, table, torch.tensor([150], device=device), True)
    _near(out, ref, tol, "far prefill")


@pytest.mark.parametrize("S", [1, 48])
def test_captured_in_two_graphs(device, S):
    """Two graphs of the call (two layers), replayed in turn beside eager work, as the eager calls."""
    gen = torch.Generator().manual_seed(9)
    lens = [130, 64, 5, 900]
    cache, table = _pool(lens, [200] * 4, 2, 64, 2, gen)
    dev = PagedCache(*(_move(x, device) for x in cache))
    table, lengths = table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
    q, k, v = (torch.randn(4, S, h, 64, generator=gen).to(BF16).to(device) for h in (8, 2, 2))
    shadow = PagedCache(*(_move(x.view(torch.uint8).clone().view(x.dtype), device) for x in cache))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for layer in range(2):
            attention_with_pages(q, k, v, PagedCache(*(x.view(torch.uint8).clone().view(x.dtype) for x in dev)), layer, table, lengths, True)
        for layer in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(attention_with_pages(q, k, v, dev, layer, table, lengths, True))
            graphs.append(graph)
    torch.cuda.synchronize()
    for step in range(4):
        for x in (q, k, v):
            x.normal_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            want = attention_with_pages(q, k, v, shadow, layer, table, lengths, True)
            assert torch.equal(outs[layer], want), (step, layer)
        for a, b in zip(dev, shadow):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        lengths += S if step < 3 else 0


def test_same_result_every_time(device):
    gen = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 3000, (64,), generator=gen).tolist()
    cache, table = _pool(lens, [1] * 64, 2, 64, 1, gen)
    dev = PagedCache(*(_move(x, device) for x in cache))
    q, k, v = (torch.randn(64, 1, h, 64, generator=gen).to(BF16).to(device) for h in (8, 2, 2))
    lengths = torch.tensor(lens, device=device)
    first = attention_with_pages(q, k, v, dev, 0, table.to(device), lengths, True)
    for _ in range(5):
        assert torch.equal(attention_with_pages(q, k, v, dev, 0, table.to(device), lengths, True), first)


def test_refusals(device):
    cache = PagedCache.create(4, 2, 2, 64, device=device)
    table = torch.zeros(1, 2, dtype=torch.int32, device=device)
    lens = torch.zeros(1, dtype=torch.int32, device=device)
    q, k = torch.zeros(1, 1, 4, 64, device=device, dtype=BF16), torch.zeros(1, 1, 2, 64, device=device, dtype=BF16)
    call = lambda q=q, k=k, v=k, cache=cache, layer=0, table=table, lens=lens, **kw: attention_with_pages(  # noqa: E731
        q, k, v, cache, layer, table, lens, True, **kw)
    assert call().shape == q.shape
    for exc, kw in [(TypeError, dict(q=q.float())), (ValueError, dict(k=k.float())), (ValueError, dict(q=q[0])),
                    (ValueError, dict(k=k[..., :32])), (ValueError, dict(q=q[:, :, :3])), (IndexError, dict(layer=2)),
                    (IndexError, dict(layer=-1)), (ValueError, dict(table=table.long())), (ValueError, dict(table=table[0])),
                    (ValueError, dict(lens=lens.float())), (ValueError, dict(lens=torch.zeros(2, dtype=torch.int32, device=device))),
                    (ValueError, dict(new_lengths=torch.zeros(2, dtype=torch.int32, device=device))),
                    (ValueError, dict(cache=PagedCache.create(4, 2, 3, 64, device=device))),
                    (ValueError, dict(cache=PagedCache.create(0, 2, 2, 64, device=device))),
                    (ValueError, dict(softmax_scale=0.0)), (ValueError, dict(softmax_scale=float("nan"))),
                    (TypeError, dict(cache=cache._replace(keys=cache.keys.view(torch.uint8)))),
                    (TypeError, dict(cache=cache._replace(key_exponents=cache.key_exponents.view(torch.uint8)))),
                    (ValueError, dict(cache=cache._replace(values=cache.values[:2]))),
                    (ValueError, dict(cache=cache._replace(keys=cache.keys.transpose(1, 2)))),
                    (RuntimeError, dict(q=q.cpu()))]:
        with pytest.raises(exc):
            call(**kw)
    assert call(q=q[:0], k=k[:0], v=k[:0], lens=lens[:0]).shape == (0, 1, 4, 64)
    assert call(q=q[:, :0], k=k[:, :0], v=k[:, :0]).shape == (1, 0, 4, 64)


def test_validation(device):
    cache = PagedCache.create(4, 1, 2, 64, device=device)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = ints([0, 1], [0, 2])
    q, k = torch.ones(2, 1, 4, 64, device=device, dtype=BF16), torch.ones(2, 1, 2, 64, device=device, dtype=BF16)
    mimir_amd.set_validate_metadata(True)
    try:
        attention_with_pages(q, k, k, cache, 0, table, ints(64, 65), True)  # the shared page 0 is only read
        attention_with_pages(q, k, k, cache, 0, table, ints(3, 5), True, new_lengths=ints(1, 0))
        for exc, lens, kw in [(ValueError, ints(3, 5), {}), (ValueError, ints(-1, 64), {}), (IndexError, ints(128, 64), {}),
                              (ValueError, ints(64, 65), dict(new_lengths=ints(2, 0))),
                              (IndexError, ints(64, 65), dict(cache_batch_indices=ints(0, 2)))]:
            with pytest.raises(exc):
                attention_with_pages(q, k, k, cache, 0, table, lens, True, **kw)
        with pytest.raises(IndexError, match="no page"):
            attention_with_pages(q, k, k, cache, 0, ints([0, 1], [3, -1]), ints(64, 65), True)
    finally:
        mimir_amd.set_validate_metadata(False)


@pytest.mark.parametrize("S", [1, 40])
def test_two_streams_at_once(device, S):
    """Calls of two layers that overlap on two streams, as the calls one after another."""
    gen = torch.Generator().manual_seed(12)
    lens = [900, 64, 5, 2030]
    cache, table = _pool(lens, [8 * S] * 4, 2, 64, 2, gen)
    one, two = (PagedCache(*(_move(x, device) for x in cache)) for _ in range(2))
    table, lengths = table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
    q, k, v = (torch.randn(4, S, h, 64, generator=gen).to(BF16).to(device) for h in (8, 2, 2))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs, wants = [[], []], [[], []]
    torch.cuda.synchronize()
    for step in range(6):
        at = lengths + S * step
        torch.cuda.synchronize()
        for layer in range(2):
            with torch.cuda.stream(streams[layer]):
                outs[layer].append(attention_with_pages(q, k, v, one, layer, table, at, True))
        for layer in range(2):
            wants[layer].append(attention_with_pages(q, k, v, two, layer, table, at, True))
    torch.cuda.synchronize()
    for a, b in zip(outs[0] + outs[1], wants[0] + wants[1]):
        assert torch.equal(a, b)
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("d,hq,hkv", [(128, 16, 4), (64, 8, 8), (128, 2, 2)])
@pytest.mark.parametrize("lens,new,S", [
    ([0, 0, 0, 0], [0, 0, 0, 0], 300), ([2000], [77], 200), ([3000, 5, 0, 640], [40, 0, 333, 64], 333),
    ([130, 64, 900], [513, 0, 1], 513), ([0, 63, 64, 65, 200, 1], [128, 129, 127, 1, 0, 256], 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_padded_chunks(device, d, hq, hkv, lens, new, S, causal):
    """Row tiles without queries, rows cut into many and into few runs of pages, lengths on both sides of a tile."""
    def poison(x):
        for b, n in enumerate(new):
            for t in ("q", "k", "v"):
                x[t][b, n:] = float("nan")
    _run(device, S, hq, hkv, d, lens, causal, new=new, edit=poison, seed=S + d)


@pytest.mark.parametrize("batch,S", [(64, 40), (65, 40), (63, 130), (64, 700)])
def test_padded_batches_of_many_rows(device, batch, S):
    """Up to 64 batch rows and 1024 row tiles are dealt by their pages, more are not: both as the oracle says."""
    gen = torch.Generator().manual_seed(batch + S)
    lens = torch.randint(0, 200, (batch,), generator=gen).tolist()
    new = [[0, S, 1, n][n % 4] for n in torch.randint(0, S + 1, (batch,), generator=gen).tolist()]
    _run(device, S, 8, 4, 64, lens, new=new, seed=batch)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("S", [1, 40, 300])
def test_small_probabilities_that_carry_the_output(device, d, S):
    """One token of each page takes nearly all of the softmax and holds zeros; the others, e^-16 of it, hold the output."""
    from mimir_amd.paged import PagedCache, PageTable, reserve_pages

    n, hkv = 192, 1
    cache, table = PagedCache.create(12, 1, hkv, d, device=device), PageTable.create(1, 12, 12, device=device)
    k, v = torch.zeros(1, n, hkv, d), torch.full((1, n, hkv, d), 2.0 ** 23)
    k[..., 0] = -16.0
    k[:, ::64], v[:, ::64] = 0.0, 0.0
    v[:, 1::2] *= 1.5
    k, v = (x.bfloat16().to(device) for x in (k, v))
    lens = torch.zeros(1, dtype=torch.int32, device=device)
    reserve_pages(table, torch.tensor([n + S], device=device))
    attention_with_pages(torch.zeros(1, n, 2, d, device=device).bfloat16(), k, v, cache, 0, table.pages, lens, True)
    q = torch.zeros(1, S, 2, d, device=device).bfloat16()
    q[..., 0] = 1.0
    far = torch.zeros(1, S, hkv, d, device=device).bfloat16()
    far[..., 0] = -240.0  # the call's own tokens: nothing
    lens.fill_(n)
    pool = O.Cache(*cache)
    got = attention_with_pages(q, far, far * 0, cache, 0, table.pages, lens, True, softmax_scale=1.0)
    want, tol = pool.attend(q, far, far * 0, 0, table.pages, lens, True, scale=1.0)
    assert want.min() > 50 and tol.max() < 1
    assert (abs(got.cpu().double().numpy() - want) <= tol).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("S", [1, 40, 300])
def test_small_query_elements_beside_far_larger_ones(device, d, S):
    """A column 2^20 times the others, at which every key is zero: the others decide, also in prefill, whose queries are
    scaled by the largest of 32 columns (two runs of 16, 32 apart)."""
    from mimir_amd.paged import PagedCache, PageTable, reserve_pages

    n, hkv = 130, 2
    gen = torch.Generator().manual_seed(d + S)
    for big in (0, 37, d - 1):
        cache, table = PagedCache.create(8, 1, hkv, d, device=device), PageTable.create(1, 8, 8, device=device)
        q, k, v = (torch.randn(1, S, h, d, generator=gen) for h in (4, hkv, hkv))
        block = lambda c: (c // 64, c // 16 % 2)  # noqa: E731
        small = torch.tensor([block(c) != block(big) for c in range(d)])  # the columns that decide
        q = torch.where(small, q, 0.0)
        q[..., big] = 2.0 ** 20
        k[..., big] = 0.0
        lens = torch.zeros(1, dtype=torch.int32, device=device)
        kn, vn = (torch.randn(1, n, hkv, d, generator=gen) for _ in range(2))
        kn[..., big] = 0.0
        reserve_pages(table, torch.tensor([n + S], device=device))
        q, k, v, kn, vn = (x.bfloat16().to(device) for x in (q, k, v, kn, vn))
        attention_with_pages(torch.zeros(1, n, 4, d, device=device).bfloat16(), kn, vn, cache, 0, table.pages, lens, True)
        lens.fill_(n)
        pool = O.Cache(*cache)
        got = attention_with_pages(q, k, v, cache, 0, table.pages, lens, True)
        plain = q.clone()
        plain[..., big] = 0.0  # what the large column adds is zero: the bound of a call without it
        want, tol = pool.attend(plain, k, v, 0, table.pages, lens, True)
        assert (abs(got.cpu().double().numpy() - want) <= tol).all(), big
