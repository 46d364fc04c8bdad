"""The paged cache without a GPU: the oracle's 8-bit codes, refusals of the C ABI and of CPU tensors."""

import ctypes
import math

import numpy as np
import pytest
import torch

from mimir_amd import _capi
from mimir_amd.paged import PagedCache, PageTable, attention_with_pages, compact_pages, copy_pages, fork_rows, release_rows, reserve_pages
from oracle import paged_oracle as O


def test_oracle_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.VALUES, want, equal_nan=True)
    gen = torch.Generator().manual_seed(0)
    x = torch.cat((torch.randn(20000, generator=gen) * 100, torch.randn(20000, generator=gen) * 0.01, torch.from_numpy(O._MID).float(),
                   -torch.from_numpy(O._MID).float(), torch.tensor([0.0, -0.0, 448.0, -448.0, 1e-9, math.nan]))).clamp(-448, 448)
    got = O.encode(x.double().numpy())
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    nan = want & 127 == 127
    assert np.array_equal(got[~nan], want[~nan]) and (got[nan] & 127 == 127).all()


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.5, 1), (1.0, -8), (0.875, -9), (0.876, -8), (0.0, -100), (2.0 ** -140, -100), (3.3e38, 120)])
def test_oracle_exponents(amax, e):
    assert O.exponent(amax) == e


def _attn(**kw):
    one = 4096  # never read: every call here is refused, or empty
    p = _capi.PagedAttnParams()
    for name in ("q", "k_new", "v_new", "out", "cache_k", "cache_v", "k_exponents", "v_exponents", "page_table", "cache_lengths"):
        setattr(p, name, one)
    p.batch, p.seqlen, p.num_pages, p.table_rows, p.table_width = 1, 1, 4, 1, 4
    p.num_q_heads, p.num_kv_heads, p.head_dim, p.dtype, p.softmax_scale = 4, 2, 64, _capi.DTYPE_BFLOAT16, 0.1
    p.k_stride_page = p.v_stride_page = 2 * 64 * 64
    p.ke_stride_page = p.ve_stride_page = 2
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw,exc", [
    (dict(dtype=0), TypeError), (dict(batch=-1), ValueError), (dict(num_kv_heads=0), ValueError), (dict(num_q_heads=5), ValueError),
    (dict(head_dim=96), ValueError), (dict(softmax_scale=0.0), ValueError), (dict(softmax_scale=math.inf), ValueError),
    (dict(num_pages=0), ValueError), (dict(table_width=0), ValueError), (dict(table_width=1 << 25), ValueError),
    (dict(page_table=None), ValueError), (dict(cache_lengths=None), ValueError), (dict(q=None), ValueError), (dict(k_new=4098), ValueError),
    (dict(out_stride_head=3), ValueError), (dict(q_stride_batch=-8), ValueError), (dict(cache_v=None), ValueError),
    (dict(cache_k=4100), ValueError), (dict(k_stride_page=100), ValueError), (dict(v_stride_page=4096), ValueError),
    (dict(ke_stride_page=1), ValueError), (dict(table_stride=-1), ValueError),
    (dict(table_width=64, workspace=None), ValueError), (dict(table_width=64, workspace=4096, workspace_bytes=8), ValueError),
    (dict(batch=1 << 20, seqlen=1 << 20), ValueError),
])
def test_attention_refusals(kw, exc):
    lib = _capi.load()
    with pytest.raises(exc):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_paged_attn(ctypes.byref(_attn(**kw)), None))


def test_attention_empty_calls_and_workspace():
    lib = _capi.load()
    for kw in (dict(batch=0), dict(seqlen=0)):
        assert lib.mimir_prefixlm_paged_attn(ctypes.byref(_attn(**kw)), None) == _capi.OK
        assert lib.mimir_prefixlm_paged_attn_workspace_bytes(ctypes.byref(_attn(**kw))) == 0
    assert lib.mimir_prefixlm_paged_attn(None, None) == _capi.ERR_INVALID_ARGUMENT
    assert lib.mimir_prefixlm_paged_attn_workspace_bytes(None) == 0
    for kw in (dict(num_kv_heads=0), dict(num_q_heads=3), dict(table_width=-1)):
        assert lib.mimir_prefixlm_paged_attn_workspace_bytes(ctypes.byref(_attn(**kw))) == 0
    # decode: two slots of S * Hq / Hkv rows (D floats of O, a maximum, a sum) per workgroup
    need = lib.mimir_prefixlm_paged_attn_workspace_bytes(ctypes.byref(_attn(table_width=64, seqlen=3)))
    assert need % (2 * 3 * 2 * 66 * 4) == 0 and need > 0
    assert lib.mimir_prefixlm_paged_attn_workspace_bytes(ctypes.byref(_attn(table_width=2))) == 0


def _pages(**kw):
    one = 4096
    p = _capi.PagesParams()
    p.pages = p.lengths = p.counts = p.missing = p.workspace = one
    p.pages_stride, p.rows, p.width, p.num_pages, p.workspace_bytes = 4, 3, 4, 9, 1 << 20
    for i in range(4):
        p.data[i], p.data_bytes[i], p.data_stride[i] = one, 64, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_page_refusals():
    lib = _capi.load()
    calls = {
        "copy": lambda p, n=2, x=4096: lib.mimir_prefixlm_pages_copy(p, x, x, n, None),
        "fork": lambda p, n=2, x=4096: lib.mimir_prefixlm_pages_fork(p, x, x, n, None),
        "compact": lambda p, n=2, x=4096: lib.mimir_prefixlm_pages_compact(p, x, None),
        "release": lambda p, n=2, x=4096: lib.mimir_prefixlm_pages_release(p, x, n, None),
        "reserve": lambda p, n=2, x=4096: lib.mimir_prefixlm_pages_reserve(p, x, None),
    }
    tables = [dict(rows=-1), dict(width=-1), dict(num_pages=-1), dict(pages_stride=3), dict(pages=None), dict(counts=None),
              dict(lengths=None), dict(missing=None)]
    for name, call in calls.items():
        assert call(None) == _capi.ERR_INVALID_ARGUMENT
        for kw in tables if name != "copy" else tables[2:3]:
            with pytest.raises(ValueError):
                _capi.raise_for_status(lib, call(ctypes.byref(_pages(**kw))))
        assert call(ctypes.byref(_pages()), x=None) == _capi.ERR_INVALID_ARGUMENT, name
        if name in ("copy", "fork", "release"):
            assert call(ctypes.byref(_pages()), n=-1) == _capi.ERR_INVALID_ARGUMENT
            assert call(ctypes.byref(_pages()), n=0) == _capi.OK
        if name in ("fork", "compact", "reserve"):
            for kw in (dict(workspace=None), dict(workspace_bytes=16), dict(workspace=4100)):
                assert call(ctypes.byref(_pages(**kw))) == _capi.ERR_INVALID_ARGUMENT, (name, kw)
        if name in ("copy", "fork", "compact"):
            for i in range(4):
                p = _pages()
                p.data[i] = None
                assert call(ctypes.byref(p)) == _capi.ERR_INVALID_ARGUMENT
                p = _pages()
                p.data_stride[i] = 48
                assert call(ctypes.byref(p)) == _capi.ERR_UNSUPPORTED_SHAPE
            p = _pages()
            p.data_bytes[0] = 40
            assert call(ctypes.byref(p)) == _capi.ERR_UNSUPPORTED_SHAPE
    assert lib.mimir_prefixlm_pages_workspace_bytes(None, 3) == 0
    assert lib.mimir_prefixlm_pages_workspace_bytes(ctypes.byref(_pages()), -1) == 0


def test_cpu_tensors_are_refused():
    cache, table = PagedCache.create(4, 1, 2, 64, device="cpu"), PageTable.create(2, 3, 4, device="cpu")
    assert cache.keys.shape == (4, 1, 2, 64, 64) and cache.values.dtype == torch.float8_e4m3fn and cache.key_exponents.dtype == torch.int8
    assert table.pages.tolist() == [[-1] * 3] * 2 and table.counts.tolist() == [0] * 4
    ints = torch.zeros(2, dtype=torch.int32)
    q, k = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: attention_with_pages(q, k, k, cache, 0, table.pages, ints, True), lambda: copy_pages(cache, ints, ints),
                 lambda: fork_rows(cache, table, ints, ints), lambda: compact_pages(cache, table), lambda: release_rows(table, ints),
                 lambda: reserve_pages(table, ints)):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()


@pytest.mark.parametrize("cls,name", [(_capi.RotaryParams, "MimirRotaryParams"), (_capi.PagedAttnParams, "MimirPagedAttnParams"),
                                      (_capi.PagesParams, "MimirPagesParams")])
def test_structs_match_the_header(cls, name):
    from test_capi import _c_layout

    fields = [f for f, _ in cls._fields_]
    size, offsets = _c_layout(name, fields)
    assert ctypes.sizeof(cls) == size
    assert [getattr(cls, f).offset for f in fields] == list(offsets)


@pytest.mark.parametrize("table,lens,new,bad", [
    ([[0, 1], [0, 2]], [64, 65], None, None),           # page 0 is only read
    ([[0, 1], [0, 2]], [3, 64], None, ValueError),      # appended to by row 0, read for row 1
    ([[0, 1], [0, 2]], [64, 3], None, ValueError),
    ([[0, 1], [0, 2]], [3, 64], [1, 0], None),          # row 1 is left alone
    ([[0, 1], [2, 2]], [3, 64], None, ValueError),      # twice in one row
    ([[0, 1], [2, 0]], [3, 5], None, None),             # behind row 1's last token: not looked at
    ([[0, 1], [2, 3]], [63, 63], [2, 1], None),
    ([[0, 1], [1, 3]], [63, 63], [2, 1], ValueError),   # row 0's second new token, row 1's page
])
def test_appended_pages_are_one_rows(table, lens, new, bad):
    from mimir_amd.paged import _validate
    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    call = lambda rows=None: _validate(PagedCache.create(4, 1, 2, 64, device="cpu"), ints(table), ints(lens), rows,  # noqa: E731
                                       None if new is None else ints(new), 2 if new else 1)
    if bad is None:
        call()
    else:
        with pytest.raises(bad, match="held twice"):
            call()


def test_validation_of_rows():
    from mimir_amd.paged import _validate
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cache, table = PagedCache.create(4, 1, 2, 64, device="cpu"), ints([0, 1], [2, 3])
    with pytest.raises(ValueError, match="held twice"):
        _validate(cache, table, ints(3, 3), ints(1, 1), None, 1)
    with pytest.raises(IndexError, match="without rows"):
        _validate(cache, table[:0], ints(3, 3), None, None, 1)


def test_lists_of_rows():
    from mimir_amd.paged import _row_list
    far = torch.tensor([0, 1 << 32, -(1 << 32), (1 << 32) + 1, -1])
    assert _row_list("rows", far, "cpu").tolist() == [0, (1 << 31) - 1, -(1 << 31), (1 << 31) - 1, -1]  # none of them row 0 or 1 but the first
    assert _row_list("rows", torch.tensor([3, 250], dtype=torch.uint8), "cpu").tolist() == [3, 250]
    for bad in (torch.tensor([True, False]), torch.tensor([1.0]), torch.tensor([1j]), torch.tensor(1), torch.tensor([[1]])):
        with pytest.raises(ValueError, match="whole numbers"):
            _row_list("rows", bad, "cpu")


def _set_back(rows, width, pages, seed):
    """A table of rows whose partly filled last pages several rows share, as after a fork and lengths set back."""
    import random
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    table, lens, counts = [], [], [0] * pages
    for r in range(rows):
        if r and rng.random() < 0.7:  # another's pages, all or the first ones, and within their last one
            o = rng.randrange(r)
            held = [p for p in table[o] if p >= 0]
            row = held[:rng.randint(0, len(held))]
        else:
            row = [free.pop() for _ in range(min(rng.randint(0, width), len(free)))]
        n = rng.randint(max(0, 64 * len(row) - 63), 64 * len(row))
        if rng.random() < 0.2:
            n = rng.randint(0, n)
        for p in row:
            counts[p] += 1
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    return table, lens, counts


def _entries(rows, seed):
    """All rows replaced in some order, or a few, some by each other, with repeats and numbers outside."""
    import random
    rng = random.Random(seed)
    dst = list(range(rows))
    rng.shuffle(dst)
    if seed % 3 == 0:
        return [rng.randrange(rows) for _ in dst], dst
    if seed % 3 == 1:
        return sorted(dst), dst
    n = rng.randint(1, 2 * rows)
    return [rng.randint(-1, rows) for _ in range(n)], [rng.randint(-1, rows) for _ in range(n)]


@pytest.mark.parametrize("seed", range(60))
def test_no_page_of_a_fork_is_read_and_written(seed):
    """A page that a fork copies is held after the call, so it is none of those handed out, and every row's tokens
    are the source's."""
    rows, width, pages = 7, 3, 18 + seed % 7
    t = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table, lens, counts = _set_back(rows, width, pages, seed)
    want = O.Table(t(table), t(lens), t(counts), t([0]))
    src, dst = _entries(rows, seed)
    moves = want.fork(src, dst)
    assert not {a for a, _ in moves} & {b for _, b in moves}
    assert all(want.counts[a] > 0 and want.counts[b] == 1 for a, b in moves)
    named = [p for row in want.pages for p in row if p >= 0]
    assert want.counts == [named.count(p) for p in range(pages)]
    origin = dict((b, a) for a, b in moves)
    last = {d: s for s, d in zip(src, dst) if 0 <= s < rows and 0 <= d < rows}
    lost = 0
    for d, s in last.items():
        for i in range(-(-lens[s] // 64)):
            p = want.pages[d][i]
            lost += p < 0
            assert p < 0 or origin.get(p, p) == table[s][i], (d, s, i)
    assert lost == want.missing  # (no row here lacks a page that its tokens need)


def test_a_last_page_given_up_by_all_goes_to_the_first():
    t = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    # rows 0 and 2 hold page 0, 40 tokens of it; every row that held it goes on from another
    want = O.Table(t([[0], [3], [0], [-1]]), t([40, 10, 40, 0]), t([2, 0, 0, 1]), t([0]))
    # row 0 goes on in page 3, which row 1 alone held; row 2 in page 0; rows 3 and 1 in copies of it
    assert want.fork([1, 0, 2, 2], [0, 2, 3, 1]) == [(0, 1), (0, 2)]
    assert want.pages == [[3], [2], [0], [1]] and want.counts == [1, 1, 1, 1] and want.missing == 0
    # no page left: the first still has it
    want = O.Table(t([[0], [0]]), t([40, 40]), t([2]), t([0]))
    assert want.fork([1, 0], [0, 1]) == [] and want.pages == [[0], [-1]] and want.missing == 1 and want.counts == [1]


@pytest.mark.parametrize("kw", [
    dict(batch=1 << 22, num_kv_heads=4),                            # decode: a workgroup of 256 threads for each row and head
    dict(batch=1 << 24, num_q_heads=1, num_kv_heads=1),
    dict(batch=1 << 18, seqlen=2000, num_q_heads=4, num_kv_heads=4),   # prefill: its append, and its row tiles
])
def test_attention_refuses_launches_of_2_to_32_threads(kw):
    lib, p = _capi.load(), _attn(**kw)
    page = p.num_kv_heads * 64 * 64
    p.k_stride_page, p.v_stride_page, p.ke_stride_page, p.ve_stride_page = page, page, p.num_kv_heads, p.num_kv_heads
    with pytest.raises(ValueError, match="too many"):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_paged_attn(ctypes.byref(p), None))


def test_page_calls_refuse_launches_of_2_to_32_threads():
    lib, n = _capi.load(), 1 << 24
    for status in (lib.mimir_prefixlm_pages_fork(ctypes.byref(_pages(workspace_bytes=1 << 40)), 4096, 4096, n, None),
                   lib.mimir_prefixlm_pages_release(ctypes.byref(_pages()), 4096, n, None),
                   lib.mimir_prefixlm_pages_reserve(ctypes.byref(_pages(rows=1 << 26, workspace_bytes=1 << 40)), 4096, None)):
        with pytest.raises(ValueError, match="too many rows"):
            _capi.raise_for_status(lib, status)
