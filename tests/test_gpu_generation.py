"""Normed rotary heads, cached and cross attention, beam selection and reordering used together on the GPU, and
their native host calls against the general path."""

import math

import pytest
import torch

from mimir_amd import _capi, prefixlm_attn_fwd
from mimir_amd.beams import reorder_rows, select_beams
from mimir_amd.cache import Cache, attention_with_cache
from mimir_amd.cross import attention_to_states, cross_attention
from mimir_amd.paged import PagedCache, PageTable, attention_with_pages, fork_rows, reserve_pages
from mimir_amd.rotary import RotaryFrequencies, norm_rotary
from oracle import generation_oracle as O

pytestmark = pytest.mark.gpu
U, MORE = 2.0 ** -8, 2.0 ** -11


class _Layer:
    """A decoder layer's attention over its own tokens and over encoded states, and the logits of both."""

    def __init__(self, device, hq, hkv, d, vocab, gen):
        rand = lambda *s: torch.randn(*s, generator=gen).to(device)  # noqa: E731
        self.hq, self.hkv, self.d = hq, hkv, d
        self.qkv = rand(vocab, hq + 2 * hkv, d).bfloat16()  # of each token
        self.cross_q = rand(vocab, hq, d).bfloat16()
        self.wq, self.wk = (0.5 + torch.rand(d, generator=gen)).to(device), (0.5 + torch.rand(d, generator=gen)).to(device)
        self.head = rand(hq * d, vocab) / math.sqrt(hq * d) * 6.0
        self.table = RotaryFrequencies.create(d, device=device)

    def heads(self, tokens, positions):
        """tokens and positions [...] -> normed, turned q and k, and v."""
        x = self.qkv[tokens]
        q, k = norm_rotary(x[..., :self.hq, :], x[..., self.hq:self.hq + self.hkv, :], positions, self.table, self.wq, self.wk)
        return q, k, x[..., self.hq + self.hkv:, :].contiguous()

    def logits(self, own, other):
        return (own.float() + other.float()).flatten(-2).matmul(self.head)


@pytest.mark.parametrize("hq,hkv,d,beams", [(4, 2, 64, 3), (8, 2, 128, 4)])
def test_beam_search_against_whole_sequences(device, hq, hkv, d, beams):
    """Steps of beam search with static caches; then each surviving row's tokens through the packed operators, all at
    once, which have to give the attention outputs of the last step: both are within u sum p |v| and a rounding of them."""
    gen = torch.Generator().manual_seed(beams)
    requests, vocab, steps = 3, 200, 9
    layer = _Layer(device, hq, hkv, d, vocab, gen)
    rows = requests * beams
    lens = torch.tensor([70, 0, 133, 5], dtype=torch.int32)
    states = Cache(*(torch.randn(4, 140, hkv, d, generator=gen).bfloat16().to(device) for _ in range(2)))
    state_rows = torch.tensor([2, 0, 3], device=device)
    caches = [Cache.create(rows, 16, hkv, d, dtype=torch.bfloat16, device=device) for _ in range(2)]  # the second: no one's, moves along
    lengths = torch.zeros(rows, dtype=torch.int32, device=device)
    tokens = torch.randint(3, vocab, (requests, 1), generator=gen).expand(requests, beams).reshape(rows).to(device)
    scores = torch.zeros(requests, beams, device=device)
    scores[:, 1:] = -math.inf
    finished = torch.zeros(requests, beams, dtype=torch.bool, device=device)
    history = [[t] for t in tokens.tolist()]
    for step in range(steps):
        q, k, v = layer.heads(tokens[:, None], lengths[:, None].long())
        own = attention_with_cache(q, k, v, caches[0], lengths, True)
        caches[1].keys[torch.arange(rows), lengths.long()] = tokens.view(-1, 1, 1).bfloat16()
        lengths += 1
        other = attention_to_states(layer.cross_q[tokens][:, None], states, lens.to(device), state_rows)
        if step == steps - 1:
            break
        logits = layer.logits(own[:, 0], other[:, 0]).view(requests, beams, vocab)
        chosen = select_beams(logits, scores, finished=finished, end_token=1)
        want = O.beam_scores(logits, scores, finished, 1).flatten(1)
        place = (chosen.rows.cpu().long() - beams * torch.arange(requests)[:, None]) * vocab + chosen.tokens.cpu().long()
        best = torch.sort(want, dim=1, descending=True)[0][:, :beams]
        assert ((want.gather(1, place) - best).abs() <= 2.0 ** -18).all() or (best == -math.inf).any()
        reorder_rows(caches, lengths, chosen.rows)
        scores, finished, tokens = chosen.scores, chosen.finished, chosen.tokens.flatten().long()
        history = [history[r] + [t] for r, t in zip(chosen.rows.flatten().tolist(), tokens.tolist())]
    # the second cache holds each row's tokens
    assert caches[1].keys[:, :steps, 0, 0].cpu().tolist() == torch.tensor(history).bfloat16().tolist()
    n = len(history[0])
    all_tokens = torch.tensor(history, device=device).flatten()
    q, k, v = layer.heads(all_tokens, torch.arange(n, device=device).repeat(rows))
    cu = torch.arange(rows + 1, device=device, dtype=torch.int32) * n
    zeros = torch.zeros(rows, dtype=torch.int32, device=device)
    whole, _ = prefixlm_attn_fwd(q, k, v, True, zeros, zeros + n, cu, rows * n, rows, n)
    last = torch.arange(n - 1, rows * n, n)
    p = torch.softmax(torch.einsum("rhd,rkhd->rhk", q.double().cpu()[last],
                                   k.double().cpu().view(rows, n, hkv, d).repeat_interleave(hq // hkv, 2)) / math.sqrt(d), -1)
    size = torch.einsum("rhk,rkhd->rhd", p, v.double().cpu().abs().view(rows, n, hkv, d).repeat_interleave(hq // hkv, 2))
    a, b = own[:, 0].double().cpu(), whole.double().cpu()[last]
    assert ((a - b).abs() <= 2 * (U + MORE) * size + 2.04 * U * b.abs()).all()
    # cross attention of the last tokens, packed
    named = state_rows.tolist()
    cu_q = torch.arange(requests + 1, device=device) * beams
    cu_k = torch.tensor([0] + torch.cumsum(lens[named], 0).tolist(), device=device)
    packed = [torch.cat([t[r, :lens[r]] for r in named]) for t in states]
    b = cross_attention(layer.cross_q[tokens], *packed, cu_q, cu_k).double().cpu()
    size = O.attention_to_states(layer.cross_q[tokens][:, None], *states, lens.tolist(), named, 1 / math.sqrt(d))[1][:, 0]
    assert ((other[:, 0].double().cpu() - b).abs() <= 2 * (U + MORE) * size + 2.04 * U * b.abs()).all()


def test_beams_of_a_paged_cache(device):
    """The same rows through pages: a selection's rows are what fork_rows takes, and every row reads its own history."""
    gen = torch.Generator().manual_seed(11)
    requests, beams, hq, hkv, d, vocab, steps = 2, 4, 4, 2, 64, 90, 70
    layer = _Layer(device, hq, hkv, d, vocab, gen)
    rows = requests * beams
    pool, table = PagedCache.create(40, 1, hkv, d, device=device), PageTable.create(rows, 4, 40, device=device)
    static = Cache.create(rows, steps, hkv, d, dtype=torch.bfloat16, device=device)
    tokens, scores = torch.zeros(rows, dtype=torch.long, device=device), torch.zeros(requests, beams, device=device)
    scores[:, 1:] = -math.inf
    lengths = torch.zeros(rows, dtype=torch.int32, device=device)
    every = torch.arange(rows, dtype=torch.int32, device=device)
    one = torch.ones(rows, dtype=torch.int32, device=device)
    for step in range(steps):
        q, k, v = layer.heads(tokens[:, None], lengths[:, None].long())
        reserve_pages(table, one)
        paged = attention_with_pages(q, k, v, pool, 0, table.pages, table.lengths, True)
        table.lengths.add_(1)
        own = attention_with_cache(q, k, v, static, lengths, True)
        lengths += 1
        # the codes: keys off by 2^-4 of themselves move a score by at most 2^-4 sum |q k| scale, values 2^-4 of p |v|; far within
        # what a row of another history would show
        assert (paged - own).float().abs().mean() < 0.25 * own.float().abs().mean(), step
        chosen = select_beams(layer.logits(own[:, 0], torch.zeros_like(own[:, 0])).view(requests, beams, vocab), scores)
        fork_rows(pool, table, chosen.rows.flatten(), every)
        reorder_rows(static, lengths, chosen.rows)
        assert torch.equal(table.lengths, lengths)
        scores, tokens = chosen.scores - chosen.scores.amax(1, keepdim=True), chosen.tokens.flatten().long()
    assert int(table.missing) == 0


def test_training_step_of_both_attentions(device):
    """Heads normed and turned, then attention over the states; the gradients of the whole by the oracle's formulas."""
    gen = torch.Generator().manual_seed(5)
    hq, hkv, d, pairs = 4, 2, 64, [(40, 70), (25, 0), (3, 129)]
    cu_q, cu_k = [0, 40, 65, 68], [0, 70, 70, 199]
    rand = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, kv, do = rand(68, hq, d).bfloat16().to(device), rand(199, 2 * hkv, d).bfloat16().to(device), rand(68, hq, d).bfloat16().to(device)
    w = (0.5 + torch.rand(d, generator=gen)).to(device)
    pos, table = torch.arange(68, device=device), RotaryFrequencies.create(d, device=device)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    q, _ = norm_rotary(x, None, pos, table, w)
    out = cross_attention(q, kv[:, :hkv], kv[:, hkv:], torch.tensor(cu_q, device=device), torch.tensor(cu_k, device=device))
    dq, dx, dw = torch.autograd.grad(out, (q, x, w), do)
    freq = RotaryFrequencies.inverse_frequencies(d)[0]
    # from the kernel's own dq, as exact input
    (want_x, size_x), (want_w, size_w) = O.norm_rotary_grad(dq, x, w, pos, freq, 1.0, False, 1e-6)
    assert ((dx.cpu().double() - want_x).abs() <= 2.0 ** -18 * size_x + 1.01 * U * want_x.abs()).all()
    assert ((dw.cpu().double() - want_w).abs() <= 2.0 ** -16 * size_w).all()
    want_q, size_q = O.cross_attention(q, kv[:, :hkv], kv[:, hkv:], cu_q, cu_k, 1 / 8, do)[1]
    assert ((dq.cpu().double() - want_q).abs() <= (2.1 * U + MORE) * size_q + 1.02 * U * want_q.abs()).all()


def _every_call(device):
    gen = torch.Generator(device=device).manual_seed(2)
    bf = lambda *s: torch.randn(*s, generator=gen, device=device).bfloat16()  # noqa: E731
    x, k, w = bf(2, 9, 4, 64), bf(2, 9, 2, 64), torch.rand(64, generator=gen, device=device)
    pos, table = torch.arange(9, device=device), RotaryFrequencies.create(32, interleaved=True, device=device)
    q, keys, values = bf(50, 4, 128), bf(70, 2, 128), bf(70, 2, 128)
    cu_q, cu_k = (torch.tensor(c, device=device, dtype=torch.int32) for c in ([0, 20, 50], [0, 33, 70]))
    queries, states = bf(4, 2, 8, 64), Cache(bf(3, 40, 2, 64), bf(3, 40, 2, 64))
    lens, rows = torch.tensor([40, 3, 0], device=device), torch.tensor([1, 0], device=device)
    logits, scores, done = torch.randn(2, 3, 500, generator=gen, device=device), torch.zeros(2, 3, device=device), torch.zeros(2, 3, dtype=torch.bool, device=device)
    done[1, 2] = True

    def norm():
        leaves = [t.detach().requires_grad_(True) for t in (x, k, w, w)]
        out = norm_rotary(leaves[0], leaves[1], pos, table, leaves[2], leaves[3], eps=1e-5)
        return [*out, *torch.autograd.grad(out, leaves, [torch.ones_like(t) for t in out]), norm_rotary(x, None, pos, table)[0]]

    def cross():
        leaves = [t.detach().requires_grad_(True) for t in (q, keys, values)]
        out = cross_attention(*leaves, cu_q, cu_k, softmax_scale=0.1)
        return [out, *torch.autograd.grad(out.sum(), leaves), cross_attention(q, keys, values, cu_q, cu_k)]

    def reorder():
        cache, n = Cache(states.keys.clone(), states.values.clone()), lens.clone()
        reorder_rows(cache, n, torch.tensor([[1, 1, 0]], device=device))
        return [*cache, n]

    return {"norm": norm, "cross": cross, "reorder": reorder,
            "states": lambda: [attention_to_states(queries, states, lens, rows)],
            "select": lambda: [*select_beams(logits, scores, 5, finished=done, end_token=4), *select_beams(logits, scores)[:3]]}


@pytest.mark.parametrize("name", ["norm", "cross", "reorder", "states", "select"])
def test_native_and_general_calls_agree(device, monkeypatch, name):
    native = _every_call(device)[name]()
    monkeypatch.setattr(_capi, "_host", _capi._GeneralPath)
    for a, b in zip(native, _every_call(device)[name]()):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("name", ["norm", "cross", "reorder", "states", "select"])
def test_on_a_side_stream(device, name):
    want = _every_call(device)[name]()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _every_call(device)[name]()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_captured_graphs_take_turns(device):
    """Workspaces of one graph are not another's."""
    calls = _every_call(device)
    names = ["cross", "states", "select", "norm"]
    want = {n: [t.clone() for t in calls[n]()] for n in names}
    graphs = {}
    for n in names:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls[n]()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = calls[n]()
        graphs[n] = (g, held)
    for _ in range(3):
        for n in names:
            graphs[n][0].replay()
        torch.cuda.synchronize()
        for n in names:
            assert all(torch.equal(a, b) for a, b in zip(graphs[n][1], want[n])), n
