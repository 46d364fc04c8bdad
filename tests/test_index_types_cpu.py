"""Lengths and row numbers of the cached attention in one call may be of different types: none is narrowed."""

import ctypes
import types

import pytest
import torch

from mimir_amd import _capi, cache, paged
from mimir_amd import prefixlm as P

FAR = 1 << 32


def _read(address, B, wide):
    return list(((ctypes.c_int64 if wide else ctypes.c_int32) * B).from_address(address)) if address else None


@pytest.fixture
def seen(monkeypatch):
    """What the C entry would be given: (lengths, rows, new lengths)."""
    calls = []

    def entry(p):
        wide = bool(p.index_int64)
        calls.append((_read(p.cache_lengths, p.batch, wide), _read(p.batch_indices, p.batch, wide),
                      _read(getattr(p, "new_lengths", None), p.batch, wide), wide))
        return _capi.OK

    monkeypatch.setattr(P, "_check_device_tensor", lambda name, t: None)
    monkeypatch.setattr(P, "_stream", lambda device: 0)
    monkeypatch.setattr(paged, "_call", lambda name, device, p: entry(p))
    monkeypatch.setattr(_capi, "load", lambda: types.SimpleNamespace(
        mimir_prefixlm_cache_attn=lambda p, stream: entry(p._obj), mimir_prefixlm_cache_attn_workspace_bytes=lambda p: 0,
        mimir_prefixlm_paged_attn_workspace_bytes=lambda p: 0))
    return calls


TYPES = [torch.int32, torch.int64, torch.int16, torch.uint8]


@pytest.mark.parametrize("lens", TYPES)
@pytest.mark.parametrize("rows", TYPES + [None])
@pytest.mark.parametrize("new", TYPES + [None])
def test_paged(seen, lens, rows, new):
    q, k = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    pool, table = paged.PagedCache.create(4, 1, 2, 64, device="cpu"), torch.zeros(3, 2, dtype=torch.int32)
    make = lambda t, x: None if t is None else torch.tensor(x, dtype=torch.int64).clamp(max=torch.iinfo(t).max).to(t)  # noqa: E731
    given = make(lens, [5, FAR]), make(rows, [FAR, 1]), make(new, [1, FAR + 1])
    paged.attention_with_pages(q, k, k, pool, 0, table, given[0], True, given[1], new_lengths=given[2])
    assert seen[0][:3] == tuple(None if t is None else t.tolist() for t in given)
    assert seen[0][3] == (torch.int64 in (lens, rows, new))


@pytest.mark.parametrize("lens", TYPES)
@pytest.mark.parametrize("rows", TYPES + [None])
def test_static(seen, lens, rows):
    q, k = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    rolled = cache.Cache.create(3, 16, 2, 64, dtype=torch.bfloat16)
    make = lambda t, x: None if t is None else torch.tensor(x, dtype=torch.int64).clamp(max=torch.iinfo(t).max).to(t)  # noqa: E731
    given = make(lens, [5, FAR]), make(rows, [FAR, 1])
    cache.attention_with_cache(q, k, k, rolled, given[0], True, given[1])
    assert seen[0][:2] == tuple(None if t is None else t.tolist() for t in given)
