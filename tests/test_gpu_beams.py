"""Beam selection and row reordering on the GPU (mimir_amd.beams) against 64 bits.

The kernel's scores: exp2 of an argument with two roundings (of |x - max|, whose weight exp(x - max) outweighs them: the
sum's share is below 2^-24 * 2) and 2^-23 of exp2 itself; a lane's chain of 16 adds, 6 more across lanes, two over waves: 25
roundings.  The sum is off by less than 2^-19 of itself, its logarithm by 2^-19, and the result is rounded once
to fp32.  Choices are compared where neighbours are further apart than twice that."""

import pytest
import torch

from mimir_amd.beams import reorder_rows, select_beams
from mimir_amd.cache import Cache
from oracle import generation_oracle as O

pytestmark = pytest.mark.gpu
OFF = 2.0 ** -19


def _check(logits, scores, count=None, finished=None, end_token=None):
    got = select_beams(logits, scores, count, finished=finished, end_token=end_token)
    count = count or logits.shape[1]
    every = O.beam_scores(logits, scores, finished, end_token).flatten(1)
    best, token, rows, done = O.select_beams(logits, scores, count, finished, end_token)
    vocab, beams = logits.shape[2], logits.shape[1]
    assert got.scores.shape == best.shape and got.tokens.dtype == torch.int32 and got.rows.dtype == torch.int32
    place = (got.rows.cpu().long() - beams * torch.arange(len(best))[:, None]) * vocab + got.tokens.cpu().long()
    assert ((place >= 0) & (place < beams * vocab)).all()
    assert all(len(set(r)) == count for r in place.tolist())
    # each place holds the score that is returned for it, which is that of its rank
    own = every.gather(1, place)
    for want in (own, best):
        finite = want > -float("inf")
        assert ((got.scores.cpu() > -float("inf")) == finite).all()
        off = (got.scores.cpu().double() - want).abs()[finite]
        assert (off <= OFF + 2.0 ** -24 * want.abs()[finite]).all(), off.max()
    # the same choice, but where another lies within twice the error
    srt = torch.sort(every, dim=1, descending=True)[0][:, :count + 1]
    gap = (srt[:, :-1] - srt[:, 1:])
    near = torch.zeros_like(best, dtype=torch.bool)
    close = (gap > 0) & (gap < 2 * OFF)
    near[:, :close.shape[1]] |= close
    near[:, 1:] |= close[:, :count - 1]
    same = (got.tokens.cpu() == token) & (got.rows.cpu() == rows)
    assert (same | near).all()
    if end_token is None:
        assert got.finished is None
    else:
        assert got.finished.dtype == torch.bool and (got.finished.cpu() == done)[~near].all()
    return got


def _logits(gen, requests, beams, vocab, dtype, device):
    x = 2.0 * torch.randn(requests, beams, vocab, generator=gen) + 2.0 * torch.randn(requests, 1, vocab, generator=gen)
    return x.to(dtype).to(device), (-10.0 * torch.rand(requests, beams, generator=gen)).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("requests,beams,vocab,count", [
    (1, 1, 1, 1), (1, 1, 7, 5), (2, 3, 5, 15), (1, 4, 32000, 4), (3, 5, 50257, 10), (2, 8, 16384, 8), (2, 8, 16385, 16), (1, 32, 1000, 64),
    (40, 8, 8191, 8), (33, 16, 4097, 32), (1, 2, 300001, 3), (70, 1, 65537, 1)])
def test_sizes(device, dtype, requests, beams, vocab, count):
    gen = torch.Generator().manual_seed(vocab)
    _check(*_logits(gen, requests, beams, vocab, dtype, device), count)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wide", [False, True])
def test_ties_go_to_the_lowest_place(device, dtype, wide):
    """Equal logits everywhere, in runs, and in equal beams: every piece's list overflows."""
    requests, beams, vocab = (70, 4, 40000) if wide else (2, 4, 40000)
    x = torch.zeros(requests, beams, vocab, dtype=dtype, device=device)
    s = torch.zeros(requests, beams, device=device)
    got = select_beams(x, s, 6)
    assert (got.tokens.cpu() == torch.arange(6)).all()
    assert (got.rows.cpu() == beams * torch.arange(requests)[:, None]).all()
    assert got.scores.unique().numel() == 1
    x[:, :, 100:30000] = 3.0
    x[:, :, 50] = -0.0
    got = select_beams(x, s, 6)
    assert (got.tokens.cpu() == torch.arange(100, 106)).all() and (got.rows.cpu() == beams * torch.arange(requests)[:, None]).all()
    s[:, 2] = 1.0
    x[:, :, 39999] = 5.0
    got = select_beams(x, s, 6)
    assert (got.tokens.cpu() == torch.tensor([39999, 39999, 39999, 39999, 100, 101])).all()
    assert ((got.rows.cpu() - beams * torch.arange(requests)[:, None]) == torch.tensor([2, 0, 1, 3, 2, 2])).all()


def test_negative_zero_is_zero(device):
    x = torch.full((1, 1, 1000), -1.0, device=device)
    x[0, 0, 700], x[0, 0, 300], x[0, 0, 500] = 0.0, -0.0, 0.0
    assert select_beams(x, torch.zeros(1, 1, device=device), 3).tokens.tolist() == [[300, 500, 700]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 33000])
def test_masked_tokens(device, dtype, vocab):
    """Few tokens allowed, none, and fewer than are asked for."""
    gen = torch.Generator().manual_seed(vocab)
    x, s = _logits(gen, 6, 3, vocab, dtype, device)
    allowed = torch.zeros(6, 3, vocab, dtype=torch.bool)
    allowed[0, 0, 7] = allowed[0, 1, vocab - 1] = True                    # two continuations for a count of 8
    allowed[1, :, 5:12] = True
    allowed[2, 1, ::3] = True
    allowed[4] = torch.rand(3, vocab, generator=gen) < 0.5                # row 3: none at all
    allowed[5, 0, 1] = allowed[5, 0, 0] = allowed[5, 2, 2] = True
    x = x.masked_fill(~allowed.to(device), -float("inf"))
    got = _check(x, s, 8)
    assert got.tokens[3].tolist() == list(range(8)) and got.rows[3].tolist() == [9] * 8
    assert got.scores[3].max() == -float("inf")
    assert got.tokens[5, 3:].tolist() == [2, 3, 4, 5, 6] and got.rows[5, 3:].tolist() == [15] * 5  # after beam 0's two


def test_lowest_values_of_the_type(device):
    """Masks of the type's lowest finite value: chosen last, with a finite or infinite score of their own."""
    for dtype in (torch.bfloat16, torch.float32):
        low = torch.finfo(dtype).min
        x = torch.full((1, 2, 4000), low, dtype=dtype, device=device)
        x[0, 0, 3], x[0, 1, 9] = 2.0, 1.0
        got = select_beams(x, torch.tensor([[0.0, -0.5]], device=device), 4)
        assert got.tokens.tolist() == [[3, 9, 0, 1]] and got.rows.tolist() == [[0, 1, 0, 0]]
        assert got.scores[0, :2].tolist() == [0.0, -0.5] and got.scores[0, 2] <= low


def test_broken_logits_and_scores(device):
    inf, nan = float("inf"), float("nan")
    gen = torch.Generator().manual_seed(9)
    for vocab in (60, 20000):
        x, s = _logits(gen, 5, 4, vocab, torch.float32, device)
        x[0, 1, vocab - 1] = nan
        x[1, 2, 3] = inf
        x[2, :, :] = nan
        s[3, 0], s[3, 1], s[3, 2] = nan, inf, -inf
        x[4, 0] = -inf
        got = _check(x, s, 6)
        assert (got.rows[0].cpu() != 1).all() and (got.rows[1].cpu() != 6).all()
        assert (got.rows[3].cpu() == 15).all() and (got.rows[4].cpu() != 16).all()
        assert got.tokens[2].tolist() == list(range(6))


def test_finished_beams(device):
    gen = torch.Generator().manual_seed(4)
    for vocab, end in ((40, 0), (30000, 29999)):
        x, s = _logits(gen, 4, 5, vocab, torch.bfloat16, device)
        done = (torch.rand(4, 5, generator=gen) < 0.5).to(device)
        done[0], done[1] = True, False
        x[done] = float("nan")  # of an ended beam: not read
        s[0, 3] = -float("inf")
        got = _check(x, s, 5, done, end)
        assert got.finished[0].all() and (got.tokens[0, :4] == end).all()
        _check(x, s, 10, done, end)
        _check(x.masked_fill(done[..., None], 0.0), s, 10, None, end)


def test_first_step(device):
    gen = torch.Generator().manual_seed(5)
    x, s = _logits(gen, 3, 4, 20000, torch.bfloat16, device)
    s.zero_()[:, 1:] = -float("inf")
    got = _check(x, s)
    assert (got.rows.cpu() == 4 * torch.arange(3)[:, None]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(device, dtype):
    gen = torch.Generator().manual_seed(6)
    hold = torch.randn(4, 2, 3, 5003, generator=gen).to(dtype).to(device)
    scores = (-torch.rand(3, 2, 2, generator=gen)).to(device)
    _check(hold[:3, 1, :2, 1:5001], scores[:, 1], 4)
    _check(hold[:3, :, 1, 3:4000], scores[..., 0].expand(3, 2), 4)
    _check(hold[:, 0, :, :2].permute(2, 1, 0), scores[0, 0].expand(3, 2).t(), 4)  # no unit stride
    done = torch.zeros(2, 3, dtype=torch.bool, device=device)
    done[0, 1] = True
    _check(hold[:3, :, 0], scores[..., 1], 4, done.t(), 11)


def test_select_captured(device):
    gen = torch.Generator(device=device).manual_seed(7)
    x = torch.randn(3, 4, 20000, device=device, generator=gen)
    s = torch.zeros(3, 4, device=device)
    select_beams(x, s, 8, end_token=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = select_beams(x, s, 8, end_token=3)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device=device, generator=gen))
        s.copy_(-torch.rand(s.shape, device=device, generator=gen))
        want = select_beams(x, s, 8, end_token=3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


# ---------------------------------------------------------------- reordering

def _caches(gen, device, n, rows, length, hkv, d, dtype=torch.bfloat16):
    one = lambda: torch.randn(rows, length, hkv, d, generator=gen).to(dtype).to(device)  # noqa: E731
    return [Cache(one(), one()) for _ in range(n)]


def _check_reorder(caches, lengths, source):
    tensors = [t for c in caches for t in c]
    want, lens = O.reorder_rows(tensors, lengths, source.cpu())
    reorder_rows(caches, lengths, source)
    for i, (t, y) in enumerate(zip(tensors, want)):
        assert torch.equal(t.cpu(), y), i
    assert torch.equal(lengths.cpu(), lens)


@pytest.mark.parametrize("ltype,stype", [(torch.int32, torch.int32), (torch.int64, torch.int64), (torch.int32, torch.int64)])
@pytest.mark.parametrize("requests,beams,layers,length,hkv,d", [
    (1, 1, 1, 10, 1, 64), (1, 2, 1, 1, 1, 8), (3, 4, 2, 100, 2, 64), (2, 5, 1, 777, 4, 128), (5, 8, 1, 33, 8, 128), (2, 13, 3, 40, 1, 24),
    (1, 32, 1, 50, 2, 64), (3, 17, 9, 9, 2, 8)])
def test_reorder(device, ltype, stype, requests, beams, layers, length, hkv, d):
    gen = torch.Generator().manual_seed(length + beams)
    rows = requests * beams
    caches = _caches(gen, device, layers, rows, length, hkv, d)
    lengths = torch.randint(0, length + 1, (rows,), generator=gen).to(ltype).to(device)
    for _ in range(2):  # the second on what the first left
        source = torch.randint(0, beams, (requests, beams), generator=gen) + beams * torch.arange(requests)[:, None]
        _check_reorder(caches, lengths, source.to(stype).to(device))


def test_reorder_swaps_and_keeps(device):
    gen = torch.Generator().manual_seed(1)
    caches = _caches(gen, device, 1, 6, 300, 2, 64)
    lengths = torch.tensor([300, 0, 17, 299, 300, 1], device=device)
    _check_reorder(caches, lengths, torch.tensor([[1, 0, 2], [4, 5, 3]], device=device))
    _check_reorder(caches, lengths, torch.tensor([[0, 1, 2], [3, 4, 5]], device=device))


def test_reorder_leaves_rows_with_sources_elsewhere(device):
    gen = torch.Generator().manual_seed(2)
    caches = _caches(gen, device, 1, 8, 50, 1, 64)
    lengths = torch.tensor([50, 40, -3, 70, 20, 5], device=device)
    source = torch.tensor([[3, 0, 0], [3, 9, -1]], device=device)
    _check_reorder(caches, lengths, source)
    source = torch.tensor([[1 << 32, 2, 1], [(1 << 32) + 3, 3, 3]], device=device)
    _check_reorder(caches, lengths, source)


def test_reorder_layouts(device):
    """Rows of one larger tensor, keys and values side by side in it, another element type, more rows than the lengths have."""
    gen = torch.Generator().manual_seed(3)
    hold = torch.randn(7, 2, 30, 2, 8, generator=gen).to(device)
    lengths = torch.randint(0, 31, (6,), generator=gen).to(device)
    cache = Cache(hold[:, 0], hold[:, 1])
    _check_reorder([cache], lengths, torch.tensor([[2, 1, 0], [3, 3, 3]], device=device))
    reorder_rows(cache, lengths, torch.tensor([[0, 1, 2], [3, 4, 5]], device=device))
    reorder_rows([], lengths, torch.tensor([[0, 0, 0], [3, 4, 5]], device=device))
    assert (lengths[:3] == lengths[0]).all()


def test_reorder_of_large_caches(device):
    """Caches of 2^28 bytes and more, little of which is moved: stored past the caches, read by the next reordering."""
    gen = torch.Generator().manual_seed(6)
    length = (1 << 28) // (2 * 6 * 64 * 2) + 1
    cache = Cache.create(6, length, 1, 64, dtype=torch.bfloat16, device=device)
    for t in cache:
        t[:, :700] = torch.randn(6, 700, 1, 64, generator=gen).to(device)
    lengths = torch.tensor([700, 0, 333, 1, 699, 64], device=device)
    for source in ([[2, 0, 0], [4, 5, 3]], [[1, 2, 0], [5, 5, 4]]):
        source = torch.tensor(source, device=device)
        heads = [t[:, :701].clone() for t in cache]
        want, lens = O.reorder_rows(heads, lengths, source.cpu())
        reorder_rows(cache, lengths, source)
        assert all(torch.equal(t[:, :701].cpu(), y) for t, y in zip(cache, want)) and torch.equal(lengths.cpu(), lens)


def test_reorder_of_many_layers(device):
    """More tensors than one launch takes: nothing has moved where one of the later ones is refused."""
    gen = torch.Generator().manual_seed(5)
    lengths, source = torch.tensor([9, 5, 3, 9], device=device), torch.tensor([[1, 0], [2, 2]], device=device)
    hold = torch.randn(4, 20, 2, 9, 1, 64, generator=gen).to(device)  # all layers' rows side by side
    caches = [Cache(hold[:, i, 0], hold[:, i, 1]) for i in range(20)]
    _check_reorder(caches, lengths.clone(), source)
    caches = _caches(gen, device, 10, 4, 9, 1, 64)
    before = [t.clone() for c in caches for t in c]
    wide = torch.zeros(4, 9 * 64 + 4, device=device, dtype=torch.bfloat16)[:, :9 * 64].view(4, 9, 1, 64)  # rows off 16 bytes
    apart = torch.zeros(2, 4, 9, 1, 64, device=device, dtype=torch.bfloat16)
    flat = torch.zeros(9 * 4 * 64 + 64, device=device, dtype=torch.bfloat16)
    half = Cache(*(flat[n:n + 9 * 4 * 64].view(4, 9, 1, 64) for n in (0, 64)))  # a position apart
    for bad in (caches[0], Cache(apart[0], apart[0]), Cache(wide, apart[1]), half):
        given = lengths.clone()
        with pytest.raises(ValueError):
            reorder_rows([*caches, bad], given, source)
        assert torch.equal(given, lengths) and all(torch.equal(t, y) for t, y in zip((t for c in caches for t in c), before))


def test_reorder_refusals(device):
    from mimir_amd import set_validate_metadata

    cache = Cache.create(4, 10, 2, 64, dtype=torch.bfloat16, device=device)
    lens, src = torch.zeros(4, dtype=torch.int32, device=device), torch.zeros(2, 2, dtype=torch.int32, device=device)
    for caches, lengths, source, error in [
            ([cache, cache], lens, src, ValueError), ([Cache(cache.keys, cache.keys)], lens, src, ValueError),
            ([Cache(cache.keys[:, ::2], cache.values[:, ::2])], lens, src, ValueError), ([cache], lens[:3], src, ValueError),
            ([cache], lens.float(), src, ValueError), ([cache], lens, src.flatten(), ValueError), ([cache], lens, src.float(), ValueError),
            ([Cache(cache.keys, cache.values.float())], lens, src, ValueError),
            ([Cache(cache.keys[..., :3].contiguous(), cache.values[..., :3].contiguous())], lens, src, ValueError),
            ([Cache(cache.keys[:3], cache.values[:3])], lens, src, ValueError),
            ([Cache(cache.keys[:1].expand(4, -1, -1, -1), cache.values)], lens, src, ValueError),
            ([cache], lens.cpu(), src.cpu(), RuntimeError)]:
        with pytest.raises(error):
            reorder_rows(caches, lengths, source)
    set_validate_metadata(True)
    try:
        with pytest.raises(IndexError):
            reorder_rows(cache, lens, src)
        reorder_rows(cache, lens, torch.tensor([[1, 0], [2, 3]], device=device))
    finally:
        set_validate_metadata(False)


def test_reorder_captured(device):
    gen = torch.Generator().manual_seed(8)
    caches = _caches(gen, device, 2, 8, 40, 2, 64)
    lengths = torch.randint(0, 41, (8,), generator=gen).to(device)
    source = torch.arange(8, device=device).view(2, 4).contiguous()
    reorder_rows(caches, lengths, source)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_rows(caches, lengths, source)
    for _ in range(3):
        source.copy_(torch.randint(0, 4, (2, 4), generator=gen) + 4 * torch.arange(2)[:, None])
        tensors = [t for c in caches for t in c]
        want, lens = O.reorder_rows(tensors, lengths, source.cpu())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t.cpu(), y) for t, y in zip(tensors, want)) and torch.equal(lengths.cpu(), lens)


# ---------------------------------------------------------------- logits of any finite size

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("mask", [-1e4, -1e5, -1e9, -1e10, -1e20, -1e30, -1e37])
def test_finite_masks_over_whole_pieces(device, dtype, wide, mask):
    """A piece of a row is at most 16384 tokens from a multiple of them: masked whole at the start, in the middle, up to the end, all
    but a few tokens, and a row of nothing else (where the sums of exp(x - max) are exact: all are 1)."""
    requests, beams, vocab = (70, 4, 50000) if wide else (2, 4, 50000)
    gen = torch.Generator().manual_seed(int(wide))
    x, s = _logits(gen, requests, beams, vocab, dtype, device)
    value = torch.tensor(mask, dtype=dtype)
    x[0, 0, 16384:32768] = value
    x[0, 1, :16384] = value
    x[0, 2, 300:] = value
    x[0, 3, :49990] = value
    x[1] = value
    if wide:
        x[5:, :, 32768:] = value
    got = _check(x, s, 6)
    best = (s[0].double() + torch.log_softmax(x[0].double(), -1).amax(-1)).cpu().max()
    assert (got.scores[0, 0].cpu().double() - best).abs() <= OFF + 2.0 ** -24 * best.abs()
    first = int(s[1].argmax())  # of the row of nothing else: its best beam's first tokens
    assert got.tokens[1].tolist() == list(range(6)) and got.rows[1].tolist() == [beams + first] * 6
    assert torch.isfinite(got.scores).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("top", [1e3, 4095.0, 4097.0, -4095.0, -4097.0, 1e5, 1e6, -1e6, 1e7, -1e8, 1e9, -1e9, 1e20, -1e30])
def test_rows_far_from_zero(device, dtype, wide, top):
    """Logits around `top`, some of them equal to their neighbours by their type's spacing there."""
    requests, beams, vocab = (70, 4, 20000) if wide else (2, 4, 20000)
    gen = torch.Generator().manual_seed(3)
    x, s = _logits(gen, requests, beams, vocab, torch.float32, device)
    x = (x + top).to(dtype)
    x[0, 1] = (x[0, 1].float() - 1e3).to(dtype)  # beams far from each other: their scores are not
    got = _check(x, s, 8)
    assert torch.isfinite(got.scores).all() and (got.scores <= 0).all()


@pytest.mark.parametrize("native", [True, False])
def test_select_refusals(device, monkeypatch, native):
    """The same calls, whether the native host calls are there or not."""
    from mimir_amd import _capi

    if not native:
        monkeypatch.setattr(_capi, "_host", _capi._GeneralPath)
    x, s = torch.zeros(2, 3, 20, device=device), torch.zeros(2, 3, device=device)
    done = torch.zeros(2, 3, dtype=torch.bool, device=device)
    for end in (-1, -2, 20, 1 << 40, -(1 << 40)):
        with pytest.raises(ValueError, match="end_token"):
            select_beams(x, s, end_token=end)
        with pytest.raises(ValueError, match="end_token"):
            select_beams(x, s, finished=done, end_token=end)
    with pytest.raises(ValueError, match="end_token"):
        select_beams(x, s, finished=done)
    for count in (0, -1, 61, 65):
        with pytest.raises(ValueError, match="count"):
            select_beams(x, s, count)
    with pytest.raises(ValueError, match="beams"):
        select_beams(torch.zeros(1, 33, 20, device=device), torch.zeros(1, 33, device=device))
    for scores in (s.double(), s[:1], s[:, :2], s.cpu()):
        with pytest.raises(ValueError, match="scores"):
            select_beams(x, scores)
    for ended in (done.int(), done[:, :2], done.cpu()):
        with pytest.raises(ValueError, match="finished"):
            select_beams(x, s, finished=ended, end_token=0)
    assert select_beams(x, s).finished is None and select_beams(x, s, end_token=0).finished.dtype == torch.bool
