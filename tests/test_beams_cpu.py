"""Beam selection and row reordering without a GPU: the oracle's selection against a plain search, and the refusals."""

import ctypes
import math

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.beams import reorder_rows, select_beams
from mimir_amd.cache import Cache
from oracle import generation_oracle as O


def test_oracle_selection_by_enumeration():
    gen = torch.Generator().manual_seed(0)
    x, s = torch.randn(2, 3, 4, generator=gen), -torch.rand(2, 3, generator=gen)
    x[0, 1] = x[0, 0]
    s[0, 1] = s[0, 0]
    done = torch.tensor([[False, False, False], [True, False, False]])
    best, token, rows, ended = O.select_beams(x, s, 5, done, 2)
    for r in range(2):
        every = []
        for w in range(3):
            total = math.log(sum(math.exp(v) for v in x[r, w].tolist()))
            for t in range(4):
                p = x[r, w, t].item() - total if not done[r, w] else (0.0 if t == 2 else -math.inf)
                every.append((-(s[r, w].item() + p), w, t))
        every.sort(key=lambda e: (round(e[0], 9), e[1], e[2]))
        for i, (score, w, t) in enumerate(every[:5]):
            assert math.isclose(best[r, i], -score, rel_tol=1e-6) and (rows[r, i], token[r, i]) == (3 * r + w, t)
            assert ended[r, i] == (t == 2 or bool(done[r, w]))


def test_oracle_reordering():
    t = torch.arange(24).view(4, 6, 1, 1)
    (y,), lens = O.reorder_rows([t], torch.tensor([1, 2, 3, 4]), torch.tensor([[1, 0], [0, 2]]))
    assert y.flatten(1).tolist() == [[6, 7, 2, 3, 4, 5], [0, 7, 8, 9, 10, 11], [12, 13, 14, 15, 16, 17], [12, 13, 14, 21, 22, 23]]
    assert lens.tolist() == [2, 1, 3, 3]


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm"):
        select_beams(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="ROCm"):
        reorder_rows(Cache(torch.zeros(2, 4, 1, 8), torch.zeros(2, 4, 1, 8)), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32))


@pytest.mark.parametrize("logits,error", [(torch.zeros(2, 8), ValueError), (torch.zeros(1, 2, 8, dtype=torch.float16), TypeError)])
def test_select_refusals(logits, error):
    with pytest.raises(error):
        select_beams(logits, torch.zeros(1, 2))


def _select(**kw):
    p = _capi.BeamSelectParams()
    values = dict(logits=4096, scores=4096, out_scores=4096, out_tokens=4096, out_rows=4096, requests=2, beams=3, vocab=100, count=3,
                  end_token=-1, dtype=_capi.DTYPE_FLOAT32, workspace=4096, workspace_bytes=1 << 20)
    for name, value in {**values, **kw}.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("kw,error", [
    (dict(dtype=9), TypeError), (dict(beams=0), ValueError), (dict(beams=33), ValueError), (dict(count=0), ValueError), (dict(count=65), ValueError),
    (dict(beams=1, vocab=2), ValueError), (dict(vocab=0), ValueError), (dict(vocab=1 << 30), ValueError), (dict(requests=-1), ValueError),
    (dict(requests=0x7fffffff), ValueError), (dict(logits=None), ValueError), (dict(out_rows=None), ValueError), (dict(logits=4097), ValueError),
    (dict(end_token=100), ValueError), (dict(finished=4096), ValueError), (dict(workspace=None), ValueError), (dict(workspace=4100), ValueError),
    (dict(workspace_bytes=2 * 3 * (8 + 3 * 8) - 1), ValueError)])
def test_c_select_refusals(kw, error):
    lib = _capi.load()
    with pytest.raises(error):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_beam_select(ctypes.byref(_select(**kw)), None))


def test_select_of_no_requests():
    lib = _capi.load()
    assert lib.mimir_prefixlm_beam_select(ctypes.byref(_select(requests=0, logits=None)), None) == _capi.OK


def _reorder(data=(1 << 20, 2 << 20), stride=(4096, 4096), **kw):
    p = _capi.ReorderParams()
    values = dict(lengths=4096, source=4096, position_bytes=256, count=len(data), rows=4, group=2, max_length=16)
    for name, value in {**values, **kw}.items():
        setattr(p, name, value)
    for i, (d, s) in enumerate(zip(data, stride)):
        p.data[i], p.stride[i] = d, s
    return p


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=5), dict(group=0), dict(group=33, rows=33), dict(count=17), dict(position_bytes=8), dict(position_bytes=0),
    dict(position_bytes=1 << 25), dict(lengths=None), dict(source=None), dict(data=(8, 1 << 20)), dict(data=(None, 1 << 20)),
    dict(stride=(4096, 4104)), dict(stride=(4096, 4080)), dict(data=(1 << 20, 1 << 20)), dict(data=(1 << 20, (1 << 20) + 4096)),
    dict(max_length=-1)])
def test_c_reorder_refusals(kw):
    lib = _capi.load()
    with pytest.raises(ValueError):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_reorder_rows(ctypes.byref(_reorder(**kw)), None))


def test_structs_match_the_header():
    from tests.test_capi import _c_layout

    for cls, name in ((_capi.BeamSelectParams, "MimirBeamSelectParams"), (_capi.ReorderParams, "MimirReorderParams")):
        fields = [f[0] for f in cls._fields_]
        size, offsets = _c_layout(name, fields)
        assert ctypes.sizeof(cls) == size
        assert [getattr(cls, f).offset for f in fields] == offsets


def test_c_reorder_launches_of_2_to_the_32_threads_are_refused():
    """The lengths' launch has a wave for each group; without caches there is no other that would be too large."""
    lib = _capi.load()
    for kw in (dict(rows=1 << 26, group=1), dict(rows=1 << 30, group=16)):
        with pytest.raises(ValueError, match="too many"):
            _capi.raise_for_status(lib, lib.mimir_prefixlm_reorder_rows(ctypes.byref(_reorder((), (), update_lengths=1, max_length=0, **kw)), None))
