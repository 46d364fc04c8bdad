"""The bookkeeping of a paged cache (mimir_amd.paged) against lists that follow each call's
definition (oracle.paged_oracle.Table), and a run of all of them around the attention."""

import random

import numpy as np
import pytest
import torch

import mimir_amd
from mimir_amd.paged import (PAGE_TOKENS, PagedCache, PageTable, attention_with_pages, compact_pages, copy_pages, fork_rows,
                             release_rows, reserve_pages)
from mimir_amd.rotary import RotaryFrequencies, rotary
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


def _random_cache(device, pages, layers, heads, d, seed):
    gen = torch.Generator().manual_seed(seed)
    shape = (pages, layers, heads)
    codes = lambda a, b: torch.randint(0, 256, (*shape, a, b), generator=gen, dtype=torch.uint8).to(device).view(torch.float8_e4m3fn)  # noqa: E731
    exps = lambda: torch.randint(-90, 90, shape, generator=gen, dtype=torch.int8).to(device)  # noqa: E731
    return PagedCache(codes(PAGE_TOKENS, d), codes(d, PAGE_TOKENS), exps(), exps())


def _random_table(device, rows, width, pages, seed, shared=True, fill=0.7):
    """Rows of tokens in scattered pages; some share their first pages, some have one reserved past their tokens."""
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    table, lens, counts = [], [], [0] * pages
    for r in range(rows):
        n = rng.choice([0, rng.randint(0, width * PAGE_TOKENS), PAGE_TOKENS * rng.randint(0, width)])
        head = []
        if shared and r and rng.random() < 0.5:
            o = rng.randrange(r)
            head = table[o][:rng.randint(0, min(lens[o], n) // PAGE_TOKENS)]
        need = -(-n // PAGE_TOKENS) + (rng.random() < 0.2)
        need = max(len(head), min(need, width, len(head) + max(0, len(free) - int(pages * (1 - fill)))))
        n = min(n, need * PAGE_TOKENS)
        row = head + [free.pop() for _ in range(need - len(head))]
        for p in row:
            counts[p] += 1
        table.append(row + [-1] * (width - need))
        lens.append(n)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return PageTable(t(table).view(rows, width), t(lens), t(counts), t([0]))


def _same_table(table, want, label=""):
    assert table.pages.tolist() == want.pages, label
    assert table.lengths.tolist() == want.lengths and table.counts.tolist() == want.counts, label
    assert int(table.missing[0]) == want.missing, label


def _same_cache(cache, want, label=""):
    for got, x in zip(cache, (want.keys, want.values, want.ke, want.ve)):
        g = got.cpu()
        assert np.array_equal((g.view(torch.uint8) if g.dtype == torch.float8_e4m3fn else g).numpy(), x), label


def _counted(table):
    """Every page counts the entries that name it."""
    n = torch.zeros_like(table.counts)
    held = table.pages[table.pages >= 0].long()
    n.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    return torch.equal(n, table.counts)


@pytest.mark.parametrize("rows,width,pages", [(1, 1, 1), (3, 4, 20), (17, 9, 120), (256, 40, 9000), (5, 300, 5000), (700, 3, 2500)])
def test_release_and_reserve(device, rows, width, pages):
    for seed in range(4):
        table = _random_table(device, rows, width, pages, seed)
        want = O.Table(*table)
        rng = random.Random(seed)
        out = [rng.randint(-2, rows + 1) for _ in range(rng.randint(1, rows))]
        release_rows(table, torch.tensor(out, device=device))
        want.release(out)
        _same_table(table, want, "release")
        new = [rng.choice([0, -3, 1, rng.randint(0, 64 * width), rng.randint(0, 90 * width)]) for _ in range(rows)]
        reserve_pages(table, torch.tensor(new, device=device))
        want.reserve(new)
        _same_table(table, want, "reserve")
        assert _counted(table)


def test_a_row_listed_twice_is_released_once(device):
    table = _random_table(device, 4, 6, 40, 3)
    want = O.Table(*table)
    release_rows(table, torch.tensor([2, 2, 1, 2], device=device))
    want.release([2, 1])
    _same_table(table, want)
    release_rows(table, torch.empty(0, dtype=torch.int64, device=device))
    _same_table(table, want)


def test_an_exhausted_pool(device):
    table = PageTable.create(4, 5, 6, device=device)
    want = O.Table(*table)
    for new in ([100, 0, 200, 64], [0, 1000, 0, 300], [64, 64, 64, 64]):
        reserve_pages(table, torch.tensor(new, device=device))
        want.reserve(new)
        _same_table(table, want, new)
    assert int(table.missing[0]) > 0
    release_rows(table, torch.tensor([0], device=device))  # the pages go to the places that lack one
    want.release([0])
    reserve_pages(table, torch.tensor([0, 1000, 0, 300], device=device))
    want.reserve([0, 1000, 0, 300])
    _same_table(table, want)


@pytest.mark.parametrize("rows,width,pages", [(2, 1, 4), (8, 5, 60), (64, 20, 1200), (1100, 2, 3500), (300, 250, 9000)])
@pytest.mark.parametrize("layers,heads,d", [(1, 1, 64), (2, 3, 64)])
def test_fork(device, rows, width, pages, layers, heads, d):
    """Permutations, one source for many, self entries, entries outside, destinations named twice."""
    for seed in range(3):
        cache, table = _random_cache(device, pages, layers, heads, d, seed), _random_table(device, rows, width, pages, seed)
        pool, want = O.Cache(*cache), O.Table(*table)
        rng = random.Random(seed)
        dst = list(range(rows))
        rng.shuffle(dst)
        if seed == 0:
            src = sorted(dst)  # a permutation
        elif seed == 1:
            src, dst = [rng.choice([0, rows // 2]) for _ in dst], dst[:rng.randint(1, rows)]
            src = src[:len(dst)]
        else:
            n = rng.randint(1, 2 * rows)
            src, dst = [rng.randint(-1, rows) for _ in range(n)], [rng.randint(-1, rows) for _ in range(n)]
        fork_rows(cache, table, torch.tensor(src, device=device), torch.tensor(dst, device=device))
        pool.move(want.fork(src, dst))
        _same_table(table, want, (seed, rows))
        _same_cache(cache, pool, (seed, rows))
        assert _counted(table)


def test_fork_without_free_pages(device):
    cache = _random_cache(device, 6, 1, 1, 64, 0)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = PageTable(t([[0, 1], [2, 3], [4, -1], [-1, -1]]), t([70, 100, 10, 0]), t([1, 1, 1, 1, 1, 0]), t([0]))
    pool, want = O.Cache(*cache), O.Table(*table)
    src, dst = [0, 0, 1], [3, 2, 0]
    fork_rows(cache, table, t(src), t(dst))
    pool.move(want.fork(src, dst))
    _same_table(table, want)
    _same_cache(cache, pool)


@pytest.mark.parametrize("rows,width,pages", [(1, 1, 1), (4, 6, 50), (60, 30, 5000), (3, 2, 9001)])
@pytest.mark.parametrize("layers,heads,d", [(1, 2, 64), (3, 1, 128)])
def test_compact(device, rows, width, pages, layers, heads, d):
    for seed in range(3):
        cache, table = _random_cache(device, pages, layers, heads, d, seed), _random_table(device, rows, width, pages, seed)
        pool, want = O.Cache(*cache), O.Table(*table)
        used = compact_pages(cache, table)
        n, moves = want.compact()
        pool.move(moves)
        assert used.tolist() == [n]
        _same_table(table, want, (seed, rows))
        _same_cache(cache, pool, (seed, rows))
        again = compact_pages(cache, table)
        assert again.tolist() == [n]
        _same_table(table, want)
        _same_cache(cache, pool)


def test_compact_large_pools_and_odd_tables(device):
    """More pages than the scan holds at once, counts that are not 16-byte aligned, and a row that names a
    free page or none at all: such entries stay."""
    for pages, offset in ((40_000, 0), (16_385, 1), (20_000, 3)):
        cache = _random_cache(device, pages, 1, 1, 64, pages)
        table = _random_table(device, 30, 60, pages, 7)
        table.pages[3, 59], table.pages[4, 58], table.pages[5, 57] = pages - 1, pages + 5, -7
        room = torch.zeros(pages + 4, dtype=torch.int32, device=device)
        room[offset:offset + pages] = table.counts
        room[offset + pages - 1] = 0
        table = table._replace(counts=room[offset:offset + pages])
        pool, want = O.Cache(*cache), O.Table(*table)
        used = compact_pages(cache, table)
        n, moves = want.compact()
        pool.move(moves)
        assert used.tolist() == [n] and len(moves) > 0
        _same_table(table, want, pages)
        _same_cache(cache, pool, pages)
        new = torch.full((30,), 200, device=device)
        reserve_pages(table, new)
        want.reserve([200] * 30)
        _same_table(table, want, pages)


@pytest.mark.parametrize("n", [0, 1, 37, 600])
def test_copy(device, n):
    cache = _random_cache(device, 1300, 2, 1, 64, n)
    pool = O.Cache(*cache)
    order = torch.randperm(1300, generator=torch.Generator().manual_seed(n))
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    if n > 5:
        src[2], dst[3], src[4] = -1, 1300, 5000
    copy_pages(cache, src.to(device), dst.to(device))
    pool.move([(a, b) for a, b in zip(src.tolist(), dst.tolist()) if 0 <= a < 1300 and 0 <= b < 1300])
    _same_cache(cache, pool)


def test_layers_apart_and_pages_past_four_gib(device):
    """A pool that is a view of a wider one, moved across page numbers whose bytes pass 32 bits."""
    wide = PagedCache.create(300_000, 1, 2, 128, device=device)
    cache = PagedCache(*(x[::2] for x in wide))
    gen = torch.Generator().manual_seed(1)
    data = torch.randint(0, 256, (3, 1, 2, 64, 128), generator=gen, dtype=torch.uint8).to(device)
    src, dst = torch.tensor([5, 149_999, 140_000], device=device), torch.tensor([149_998, 7, 149_000], device=device)
    cache.keys.view(torch.uint8)[src] = data
    cache.values.view(torch.uint8)[src] = data.transpose(-1, -2)
    cache.key_exponents[src] = 7
    copy_pages(cache, src, dst)
    assert torch.equal(cache.keys.view(torch.uint8)[dst], data) and torch.equal(cache.values.view(torch.uint8)[dst], data.transpose(-1, -2))
    assert (cache.key_exponents[dst] == 7).all()
    assert int(wide.keys[1::2].view(torch.uint8).sum(dtype=torch.int64)) == 0  # the pages between are left alone


def test_refusals(device):
    cache, table = PagedCache.create(8, 1, 1, 64, device=device), PageTable.create(3, 2, 8, device=device)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    for call in (lambda: fork_rows(cache, table, ints(0, 1), ints(0)), lambda: copy_pages(cache, ints(0, 1), ints(0)),
                 lambda: reserve_pages(table, ints(1, 2)), lambda: release_rows(table, ints(1).float()),
                 lambda: release_rows(table, ints([1])), lambda: compact_pages(PagedCache.create(9, 1, 1, 64, device=device), table),
                 lambda: release_rows(table._replace(pages=table.pages.long()), ints(0)),
                 lambda: release_rows(table._replace(lengths=table.lengths[:2]), ints(0)),
                 lambda: release_rows(table._replace(pages=table.pages.t()), ints(0)),
                 lambda: compact_pages(cache._replace(keys=cache.keys.expand(8, 2, 1, 64, 64)), table)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="ROCm"):
        release_rows(PageTable.create(3, 2, 8, device="cpu"), ints(0))
    mimir_amd.set_validate_metadata(True)
    try:
        copy_pages(cache, ints(0, 0), ints(1, 2))
        for src, dst in ((ints(0, 1), ints(2, 2)), (ints(0, 1), ints(1, 3))):
            with pytest.raises(ValueError, match="named twice"):
                copy_pages(cache, src, dst)
    finally:
        mimir_amd.set_validate_metadata(False)


def test_captured(device):
    """reserve, fork, release and compact in one graph, replayed beside eager work."""
    cache, table = _random_cache(device, 400, 1, 2, 64, 1), _random_table(device, 12, 8, 400, 1)
    src, dst = torch.arange(12, device=device, dtype=torch.int32), torch.arange(12, device=device, dtype=torch.int32)
    out, new = torch.zeros(2, dtype=torch.int32, device=device), torch.zeros(12, dtype=torch.int32, device=device)

    def step():
        release_rows(table, out)
        reserve_pages(table, new)
        table.lengths.add_(new)
        fork_rows(cache, table, src, dst)
        return compact_pages(cache, table)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pool, want = O.Cache(*cache), O.Table(*table)
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            used = step()
    rng = random.Random(5)
    for _ in range(5):
        o, n = [rng.randrange(12) for _ in range(2)], [rng.randint(0, 20) for _ in range(12)]
        s = [rng.randrange(12) for _ in range(12)]
        for dev, x in ((out, o), (new, n), (src, s)):
            dev.copy_(torch.tensor(x, dtype=torch.int32))
        n = [min(a, 8 * PAGE_TOKENS - b) for a, b in zip(n, [0 if r in o else t for r, t in enumerate(want.lengths)])]
        new.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want.release(o)
        want.reserve(n)
        want.lengths = [a + b for a, b in zip(want.lengths, n)]
        pool.move(want.fork(s, list(range(12))))
        count, moves = want.compact()
        pool.move(moves)
        assert used.tolist() == [count]
        _same_table(table, want)
        _same_cache(cache, pool)


def test_serving_run(device):
    """Prompts prefilled, one forked into beams, decoded with rotary positions, beams permuted, the pool packed
    and a conversation replaced: two layers, every output against the oracle."""
    rows, hq, hkv, d, layers, pages = 6, 8, 2, 64, 2, 80
    cache, table = PagedCache.create(pages, layers, hkv, d, device=device), PageTable.create(rows, 12, pages, device=device)
    for x in cache[:2]:
        x.view(torch.uint8).fill_(127)  # whatever lies in free pages must not show
    pool, want = O.Cache(*cache), O.Table(*table)
    freq, amplitude = RotaryFrequencies.inverse_frequencies(32, scaling="yarn", factor=4.0, original_positions=256)
    turns = RotaryFrequencies.create(32, scaling="yarn", factor=4.0, original_positions=256, device=device)
    gen = torch.Generator().manual_seed(0)

    def step(S, new, causal):
        reserve_pages(table, torch.tensor(new, device=device))
        want.reserve(new)
        for layer in range(layers):
            qkv = torch.randn(rows, S, hq + 2 * hkv, d, generator=gen).to(torch.bfloat16).to(device)
            q, k, v = qkv.split((hq, hkv, hkv), dim=2)
            positions = table.lengths[:, None] + torch.arange(S, device=device, dtype=torch.int32)
            q, k = rotary(q, k, positions, turns)
            fresh = torch.tensor(new, dtype=torch.int32, device=device)
            out = attention_with_pages(q, k, v, cache, layer, table.pages, table.lengths, causal, new_lengths=fresh)
            ref, tol = pool.attend(q, k, v, layer, torch.tensor(want.pages), torch.tensor(want.lengths), causal, None, torch.tensor(new))
            assert (np.abs(out.cpu().double().numpy() - ref) <= tol + 1e-30).all(), (S, new, layer)
        table.lengths.add_(fresh)
        want.lengths = [a + b for a, b in zip(want.lengths, new)]
        _same_table(table, want)

    def fork(src, dst):
        fork_rows(cache, table, torch.tensor(src, device=device), torch.tensor(dst, device=device))
        pool.move(want.fork(src, dst))
        _same_table(table, want)

    step(100, [100, 0, 0, 37, 0, 64], False)            # prompts, bidirectional
    fork([0, 0], [1, 2])                                # three beams of the first
    for _ in range(3):
        step(1, [1] * 4 + [0, 1], True)
    fork([1, 0, 0], [0, 1, 2])                          # the beams change places
    for _ in range(2):
        step(1, [1] * 4 + [0, 1], True)
    release_rows(table, torch.tensor([3], device=device))
    want.release([3])
    assert compact_pages(cache, table).tolist() == [(moved := want.compact())[0]]
    pool.move(moved[1])
    _same_table(table, want)
    step(70, [0, 0, 0, 70, 51, 0], True)                # two more prompts
    for _ in range(2):
        step(1, [1] * 6, True)
    assert _counted(table)
    for got, x in zip(cache[:2], (pool.keys, pool.values)):  # NaN codes of either sign are one
        g = got.cpu().view(torch.uint8).numpy()
        assert ((g == x) | ((g & 127 == 127) & (x & 127 == 127))).all()


def test_numbers_past_32_bits_name_no_row(device):
    table = _random_table(device, 4, 6, 40, 3)
    want = O.Table(*table)
    far = torch.tensor([1 << 32, (1 << 32) + 2, -(1 << 32)], device=device)
    release_rows(table, far)
    cache = PagedCache.create(40, 1, 1, 64, device=device)
    fork_rows(cache, table, far, torch.tensor([0, 1, 2], device=device))
    _same_table(table, want)
    for bad in (torch.ones(4, dtype=torch.bool, device=device), torch.ones(4, device=device)):
        with pytest.raises(ValueError, match="whole numbers"):
            release_rows(table, bad)


@pytest.mark.parametrize("rows,width,pages", [(257, 40, 12000), (256, 120, 30000), (1025, 5, 4000), (65, 9, 700),
                                              (64, 128, 9000), (64, 129, 9000), (1, 700, 900), (60, 65, 70000)])
def test_reserve_in_one_launch_two_and_three(device, rows, width, pages):
    """On both sides of 64 and 256 rows and of 8192 table entries, from few asking rows to all, and out of pages."""
    for seed in range(3):
        table = _random_table(device, rows, width, pages, seed)
        want = O.Table(*table)
        rng = random.Random(seed)
        for ask in (0.1, 1.0):
            new = [rng.choice([1, 64, rng.randint(0, 64 * width)]) if rng.random() < ask else 0 for _ in range(rows)]
            reserve_pages(table, torch.tensor(new, dtype=torch.int32, device=device))
            want.reserve(new)
            _same_table(table, want, (seed, ask))
        assert _counted(table)


def _forked(device, rows, width, pages, layers, seed, table, lens, counts, src, dst):
    cache = _random_cache(device, pages, layers, 1, 64, seed)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = PageTable(t(table), t(lens), t(counts), t([0]))
    pool, want = O.Cache(*cache), O.Table(*table)
    fork_rows(cache, table, t(src), t(dst))
    pool.move(want.fork(src, dst))
    _same_table(table, want, (seed, rows))
    _same_cache(cache, pool, (seed, rows))
    assert _counted(table)


@pytest.mark.parametrize("rows,width,pages", [(2, 1, 3), (7, 3, 20), (40, 6, 150), (1300, 2, 2400)])
def test_fork_of_shared_last_pages(device, rows, width, pages):
    """Lengths set back into pages that several rows share: one that all give back goes to the first that goes on from
    it, and no page that is copied is handed out.  More entries than a workgroup has threads, pools nearly full."""
    from test_paged_cpu import _entries, _set_back

    for seed in range(6):
        for layers in (1, 5):
            _forked(device, rows, width, pages, layers, seed, *_set_back(rows, width, pages, seed), *_entries(rows, seed))


def test_fork_after_lengths_set_back(device):
    """By the package's own calls: a fork, lengths set back into its shared page, and every holder replaced."""
    cache, table = _random_cache(device, 8, 3, 2, 64, 1), PageTable.create(4, 2, 8, device=device)
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    reserve_pages(table, t(128, 0, 0, 100))
    table.lengths.copy_(t(128, 0, 0, 100))
    fork_rows(cache, table, t(0), t(1))
    table.lengths.copy_(t(100, 100, 0, 100))
    pool, want = O.Cache(*cache), O.Table(*table)
    fork_rows(cache, table, t(3, 0, 3), t(0, 2, 1))
    pool.move(want.fork([3, 0, 3], [0, 2, 1]))
    _same_table(table, want)
    _same_cache(cache, pool)
    assert _counted(table) and int(table.missing[0]) == 0
