"""Normed rotary heads, cross attention and beam search on operands whose offsets pass 2^32 elements, in views of one
buffer, with the tolerances of the operators' own tests."""

import math

import pytest
import torch

from mimir_amd.beams import reorder_rows, select_beams
from mimir_amd.cache import Cache
from mimir_amd.cross import attention_to_states, cross_attention
from mimir_amd.rotary import RotaryFrequencies, norm_rotary
from oracle import generation_oracle as O
from test_gpu_beams import _check as _check_select
from test_gpu_cross import _near

pytestmark = pytest.mark.gpu
FAR = 1 << 32


@pytest.fixture(scope="module")
def hold(device):
    t = torch.empty(FAR + (1 << 27), dtype=torch.bfloat16, device=device)
    yield t
    del t
    torch.cuda.empty_cache()


def _view(hold, shape, strides, start=0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = hold.as_strided(shape, strides, start)
    t.copy_(torch.randn(shape, generator=gen).clamp_(-4, 4).bfloat16())
    return t


@pytest.mark.parametrize("d", [64, 128])
def test_far_states(hold, d):
    lens = torch.tensor([300, 0, 70], dtype=torch.int32, device=hold.device)
    q = torch.randn(2, 3, 4, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(hold.device)
    # rows 2^31 elements apart: the third starts at 2^32
    cache = Cache(*(_view(hold, (3, 300, 2, d), (1 << 31, 2 * d, d, 1), n * 2 * 300 * d, n) for n in (0, 1)))
    rows = torch.tensor([2, 0], device=hold.device)
    _near(attention_to_states(q, cache, lens, rows), O.attention_to_states(q, *cache, lens.tolist(), rows.tolist(), 1 / math.sqrt(d)), 1.0, "out")
    # positions 2^21 apart: those from 2048 on lie behind 2^32; few and many query rows
    one = Cache(*(_view(hold, (1, 2060, 2, d), (FAR, 1 << 21, d, 1), n * 2 * d, 2 + n) for n in (0, 1)))
    for tokens in (1, 100):
        q = torch.randn(1, tokens, 4, d, generator=torch.Generator().manual_seed(tokens)).bfloat16().to(hold.device)
        _near(attention_to_states(q, one, torch.tensor([2060], device=hold.device)), O.attention_to_states(q, *one, [2060], [0], 1 / math.sqrt(d)),
              1.0, "out")


@pytest.mark.parametrize("d", [64, 128])
def test_far_cross_attention(hold, d):
    q, k, v = (_view(hold, (2060, h, d), (1 << 21, d, 1), n * 4 * d, n).detach().requires_grad_(True) for n, h in enumerate((4, 2, 2)))
    do = _view(hold, (2060, 4, d), (1 << 21, d, 1), 12 * d, 7)
    cu_q, cu_k = [0, 2000, 2060], [0, 1990, 2060]  # the second sequences pass 2^32 on the way
    out = cross_attention(q, k, v, *(torch.tensor(c, device=hold.device) for c in (cu_q, cu_k)))
    got = torch.autograd.grad(out, (q, k, v), do)
    want = O.cross_attention(q, k, v, cu_q, cu_k, 1 / math.sqrt(d), do)
    for name, g, w, rel in zip(("out", "dq", "dk", "dv"), (out.detach(), *got), want, (1.0, 2.1, 2.1, 1.0)):
        _near(g, w, rel, name)


def test_far_norm_rotary(hold):
    q = _view(hold, (3, 40, 4, 64), (1 << 31, 1000, 64, 1), 0, 1).detach().requires_grad_(True)
    dy = _view(hold, (3, 40, 4, 64), (1 << 31, 1000, 64, 1), 400, 2)
    w = torch.ones(64, device=hold.device)
    table, pos = RotaryFrequencies.create(64, device=hold.device), torch.arange(120, device=hold.device).view(3, 40)
    y, _ = norm_rotary(q, None, pos, table, w)
    (dq,) = torch.autograd.grad(y, q, dy)
    near = q.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
    z, _ = norm_rotary(near, None, pos, table, w)
    (dnear,) = torch.autograd.grad(z, near, dy.clone(memory_format=torch.contiguous_format))
    assert y.any() and torch.equal(y, z) and torch.equal(dq, dnear)


def test_far_select(hold):
    logits = _view(hold, (3, 2, 5003), (1 << 31, 6000, 1), 1, 3)
    scores = -torch.rand(3, 2, generator=torch.Generator().manual_seed(4)).to(hold.device)
    _check_select(logits, scores, 5)
    got = select_beams(logits, scores, 5)
    want = select_beams(logits.clone(memory_format=torch.contiguous_format), scores, 5)
    assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))


def test_far_reorder(hold):
    caches = [Cache(*(_view(hold, (3, 50, 2, 64), (1 << 31, 128, 64, 1), n * 50 * 128, n) for n in (0, 1)))]
    lengths = torch.tensor([50, 7, 33], device=hold.device)
    source = torch.tensor([[2, 0, 0]], device=hold.device)
    want, lens = O.reorder_rows(list(caches[0]), lengths, source.cpu())
    reorder_rows(caches, lengths, source)
    assert all(torch.equal(t.cpu(), y) for t, y in zip(caches[0], want)) and torch.equal(lengths.cpu(), lens)
