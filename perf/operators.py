"""The measured cases of the 8-bit paged KV cache and the rotary positions beside it.

Each case is one call path of a serving or training program:

* ``rotary``   -- ``rotary`` on the query and key heads of a fused projection, from token
  positions and a frequency table, and (training) the gradients;
* ``attend``   -- ``attention_with_pages``: new keys / values appended to 8-bit pages, one
  power-of-two scale for each page of 64 tokens and head, and the attention over them;
* ``fork``     -- ``fork_rows``: beams or samples that go on from other rows' tokens;
* ``compact``  -- ``compact_pages``: the pages in use moved to the front of the pool;
* ``turnover`` -- ``release_rows`` and ``reserve_pages``: finished conversations leave, new ones
  get their pages.

``run`` computes them with elementary torch operations, or (``own``) by the package's calls.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 64            # tokens of a page
E_MIN = -100         # smallest exponent of a page's scale
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn


def listed():
    return [
        # Serving, a decode step of a small batch at far positions: launch latency.
        dict(name="rotary_decode", kind="rotary", dtype="bf16", batch=8, new=1, hq=16, hkv=4, d=128, rd=128,
             interleaved=False, grad=False, scaling="wavelength", factor=8.0, original=8192, max_pos=60000, pos_seed=1),
        # Training, the headline shape: 8 sequences of 2048, grouped heads, forward and backward.
        dict(name="rotary_train", kind="rotary", dtype="bf16", batch=8, new=2048, hq=16, hkv=4, d=128, rd=128,
             interleaved=False, grad=True, scaling="none", factor=1.0, original=8192, max_pos=0, pos_seed=2),
        # Long-context training: adjacent pairs of half of each head, positions scaled past the original range.
        dict(name="rotary_long", kind="rotary", dtype="bf16", batch=1, new=32768, hq=32, hkv=8, d=128, rd=64,
             interleaved=True, grad=True, scaling="yarn", factor=16.0, original=4096, max_pos=200000, pos_seed=3),
        # Full-precision training, odd lengths and an odd part of the head.
        dict(name="rotary_odd", kind="rotary", dtype="fp32", batch=3, new=683, hq=8, hkv=8, d=64, rd=20,
             interleaved=False, grad=True, scaling="linear", factor=4.0, original=2048, max_pos=5000, pos_seed=4),
        # Serving, one user: a new token against a few hundred cached ones. Launch latency.
        dict(name="attend_single", kind="attend", batch=1, new=1, hq=16, hkv=4, d=128, min_len=700, max_len=700,
             len_seed=5, layers=2, causal=True, ragged=False),
        # Serving, a full batch of conversations of mixed length: the cache read is the work.
        dict(name="attend_wide", kind="attend", batch=64, new=1, hq=16, hkv=4, d=128, min_len=512, max_len=8000,
             len_seed=6, layers=1, causal=True, ragged=False),
        # Serving, a drafted run of tokens checked at once, small heads, some rows idle.
        dict(name="attend_draft", kind="attend", batch=48, new=5, hq=8, hkv=2, d=64, min_len=100, max_len=4000,
             len_seed=7, layers=1, causal=True, ragged=True),
        # Chunked prefill: 512 new tokens per row onto a filled cache.
        dict(name="attend_chunk", kind="attend", batch=8, new=512, hq=16, hkv=4, d=128, min_len=1536, max_len=1536,
             len_seed=8, layers=1, causal=True, ragged=False),
        # Prefixes of odd lengths, each token seeing its whole prefix, padded to the longest.
        dict(name="attend_prefix", kind="attend", batch=5, new=1339, hq=8, hkv=8, d=64, min_len=0, max_len=1000,
             len_seed=9, layers=1, causal=False, ragged=True),
        # Beam search: 32 requests of 8 beams, five of which go on from one of the other three.
        dict(name="fork_beams", kind="fork", rows=256, beams=8, min_len=200, max_len=3000, hkv=4, d=128, layers=4,
             len_seed=10),
        # A pool that is two fifths full, in scattered pages, packed to its front.
        dict(name="compact_pool", kind="compact", rows=64, min_len=64, max_len=3200, hkv=4, d=128, layers=4,
             fill=0.4, len_seed=11),
        # A batch of conversations ends and the next ones are admitted.
        dict(name="turnover_rows", kind="turnover", rows=256, some=40, min_len=10, max_len=8000, len_seed=12),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "rotary", "attend", "attend", "attend", "attend", "fork", "compact", "turnover"])
    seed = rng.randrange(1 << 20)
    if kind == "rotary":
        d = rng.choice([64, 128, 128, 80, 96])
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]), batch=_log(rng, 1, 64), new=_log(rng, 1, 16384),
                    hq=rng.choice([2, 8, 16, 32]), hkv=rng.choice([1, 2, 4, 8]), d=d,
                    rd=rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]), interleaved=rng.random() < 0.5,
                    grad=rng.random() < 0.6, scaling=rng.choice(["none", "linear", "ntk", "wavelength", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 10.0, 32.0]), original=rng.choice([2048, 4096, 8192]),
                    max_pos=_log(rng, 1, 1000000), pos_seed=seed)
        while case["batch"] * case["new"] * (case["hq"] + case["hkv"]) * d > 32768 * 40 * 64:
            case["new"] = (case["new"] + 1) // 2 if case["new"] > 1 else 1
            case["batch"] = max(1, case["batch"] - 1)
        return case
    if kind == "attend":
        hq, hkv, d = rng.choice([(16, 4, 128), (8, 8, 64), (2, 2, 128), (32, 8, 128), (8, 2, 64), (8, 1, 128)])
        shape = rng.choice(["one", "few", "chunk", "long"])
        new = {"one": 1, "few": rng.randint(2, 16), "chunk": _log(rng, 17, 1024), "long": 1}[shape]
        batch = {"one": _log(rng, 1, 100), "few": _log(rng, 1, 64), "chunk": _log(rng, 1, 8), "long": 1}[shape]
        hi = _log(rng, 20000, 131072) if shape == "long" else rng.randint(0, _log(rng, 64, 6000 if shape == "one" else 3000))
        case = dict(kind=kind, batch=batch, new=new, hq=hq, hkv=hkv, d=d, min_len=hi if shape == "long" else rng.randint(0, hi),
                    max_len=hi, len_seed=seed, layers=rng.choice([1, 1, 2]) if batch < 16 else 1, causal=rng.random() < 0.8,
                    ragged=rng.random() < 0.4)
        while case["batch"] > 1 and (work(case)["flops"] > 6e10 or work(case)["bytes"] > 2.9e8):
            case["batch"] //= 2
        while work(case)["flops"] > 6e10:
            case["new"] //= 2
        return case
    hi = _log(rng, 100, 3000)
    pages = dict(min_len=rng.randint(0, hi), max_len=hi, len_seed=seed)
    pool = dict(hkv=rng.choice([2, 4, 8]), d=rng.choice([64, 128]), layers=rng.choice([1, 2, 3]))
    if kind == "fork":
        beams = rng.choice([2, 3, 4, 5, 8])
        return dict(kind=kind, rows=beams * _log(rng, 1, 20), beams=beams, **pages, **pool)
    if kind == "compact":
        case = dict(kind=kind, rows=_log(rng, 1, 60), **pages, **pool, fill=rng.choice([0.3, 0.5, 0.7, 0.9]))
        while len(_pool_plan(case)[2]) * case["layers"] * case["hkv"] * case["d"] > 1 << 23:  # a pool of a GiB
            case["rows"] //= 2
        return case
    rows = _log(rng, 2, 700)
    return dict(kind=kind, rows=rows, some=rng.randint(1, rows), min_len=rng.randint(0, 100), max_len=_log(rng, 100, 10000),
                len_seed=seed)


# ---------------------------------------------------------------- rotary frequencies

def _frequencies(case):
    """The angle per position of each pair (64-bit floats) and the factor on the rotated values."""
    n, base, factor, original = case["rd"], 10000.0, case["factor"], case["original"]
    scaling = case["scaling"] if n > 2 else "none"  # one pair turns at frequency 1 whatever the base
    if scaling == "ntk":  # a larger base: the slowest pair is slowed by the factor
        base *= factor ** (n / (n - 2))
    freq = [base ** (-2.0 * i / n) for i in range(n // 2)]
    if scaling == "linear":
        return [f / factor for f in freq], 1.0
    if scaling == "wavelength":  # pairs of long wavelengths slowed, short ones kept, a blend between
        low, high, out = 1.0, 4.0, []
        for f in freq:
            turns = original * f / (2.0 * math.pi)  # over the original range
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append(keep * f + (1.0 - keep) * f / factor)
        return out, 1.0
    if scaling == "yarn":  # a blend by the pair's index, between the pairs of 32 turns and of one
        at = lambda turns: n * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), n - 1)
        slow = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(n // 2)]
        return [f / factor * s + f * (1.0 - s) for f, s in zip(freq, slow)], 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _positions(case):
    """[batch, new]: each row counts on from a place of its own."""
    rng = random.Random(case["pos_seed"])
    return [[p + i for i in range(case["new"])] for p in (rng.randint(0, case["max_pos"]) for _ in range(case["batch"]))]


# ---------------------------------------------------------------- page tables

def _lengths(case):
    rng = random.Random(case["len_seed"])
    return [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]


def _new_lengths(case):
    """New tokens of each row: all of them, or (ragged) none up to all."""
    rng = random.Random(case["len_seed"] + 1)
    if not case["ragged"]:
        return [case["new"]] * case["batch"]
    return [rng.choice([0, case["new"], rng.randint(0, case["new"]), rng.randint(0, case["new"])]) for _ in range(case["batch"])]


def _attend_table(case):
    """The pages of each row, in scattered order, and the pool's size."""
    need = [-(-(n + m) // PAGE) for n, m in zip(_lengths(case), _new_lengths(case))]
    pages = list(range(sum(need) + 5))
    random.Random(case["len_seed"] + 2).shuffle(pages)
    width = max(need) + 1
    table, at = [], 0
    for n in need:
        table.append(pages[at:at + n] + [-1] * (width - n))
        at += n
    return table, len(pages)


def _row_lengths(case):
    rng = random.Random(case["len_seed"])
    return [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["rows"])]


def _pool_plan(case):
    """Table, lengths, counts and, for fork, sources and destinations, as plain lists."""
    rng = random.Random(case["len_seed"] + 1)
    if case["kind"] == "fork":
        beams = case["beams"]
        lens = [n for n in _row_lengths(case)[:case["rows"] // beams] for _ in range(beams)]
        shared = [rng.randint(0, n // PAGE) for n in lens[::beams] for _ in range(beams)]  # the prompt's pages
    else:
        lens, beams = _row_lengths(case), 1
        shared = [0] * case["rows"]
    need = [-(-n // PAGE) for n in lens]
    total = sum(n - s for n, s in zip(need, shared)) + sum(shared[::beams])
    if case["kind"] == "compact":
        size = max(total + 1, int(total / case["fill"]))
    else:
        size = total + case["rows"] + 3 + (sum(need) if case["kind"] == "turnover" else 0)
    pages = list(range(size))
    rng.shuffle(pages)
    width = max(1, max(need)) + 1
    table, counts, at = [], [0] * size, 0
    for r in range(case["rows"]):
        head = table[r - r % beams][:shared[r]] if r % beams else pages[at:at + shared[r]]
        at += 0 if r % beams else shared[r]
        row = head + pages[at:at + need[r] - shared[r]]
        at += need[r] - shared[r]
        for p in row:
            counts[p] += 1
        table.append(row + [-1] * (width - len(row)))
    src = dst = None
    if case["kind"] == "fork":
        src, dst = [], []
        for r0 in range(0, case["rows"], beams):
            kept = sorted(rng.sample(range(beams), max(1, beams * 3 // 8)))
            for b in range(beams):
                dst.append(r0 + b)
                src.append(r0 + (b if b in kept else rng.choice(kept)))
    if case["kind"] == "turnover":
        src = sorted(rng.sample(range(case["rows"]), case["some"]))
        dst = [0] * case["rows"]
        for r in src:
            dst[r] = rng.randint(case["min_len"], case["max_len"])
    return table, lens, counts, src, dst


# ---------------------------------------------------------------- inputs

def _normal(gen, *shape):
    # projections of normalised activations: near normal, without far tails
    return torch.randn(shape, generator=gen, device=gen.device).clamp_(-5.0, 5.0)


def _exponent(amax):
    """The smallest e >= E_MIN with amax <= 448 * 2^e (448 = 0.875 * 2^9, the largest 8-bit value)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875).int(), torch.full_like(x, E_MIN)).clamp(min=E_MIN)


def _coded(gen, *shape):
    """A pool's worth of 8-bit values and exponents, [pages, layers, heads, a, b] and [pages, layers, heads]."""
    x = _normal(gen, *shape)
    x *= torch.exp(0.7 * torch.randn(shape[:3], generator=gen, device=gen.device))[..., None, None]
    e = _exponent(x.abs().amax((-2, -1)))
    return torch.ldexp(x, -e[..., None, None]).to(F8), e.to(torch.int8)


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    state = dict(case=case)
    if case["kind"] == "rotary":
        b, s, hq, hkv, d = (case[x] for x in ("batch", "new", "hq", "hkv", "d"))
        dtype = DTYPES[case["dtype"]]
        qkv = _normal(gen, b, s, hq + 2 * hkv, d).to(dtype)  # the fused projection: q and k are views of it
        state.update(q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hkv], positions=torch.tensor(_positions(case), device=device))
        if case["grad"]:
            state["q"], state["k"] = (state[x].detach().requires_grad_(True) for x in "qk")
            state.update(dq=_normal(gen, b, s, hq, d).to(dtype), dk=_normal(gen, b, s, hkv, d).to(dtype))
        freq, state["amplitude"] = _frequencies(case)
        state["freq"] = torch.tensor(freq, dtype=torch.float64, device=device)
        # the same as fractions of a turn per position, in units of 2^-64
        state["turns"] = torch.tensor([round(f / (2.0 * math.pi) * 2.0 ** 64) for f in freq], dtype=torch.int64, device=device)
        return state
    if case["kind"] == "attend":
        b, s, hq, hkv, d = (case[x] for x in ("batch", "new", "hq", "hkv", "d"))
        table, size = _attend_table(case)
        bf = lambda *shape: _normal(gen, *shape).to(torch.bfloat16)
        state.update(q=bf(b, s, hq, d), k=1.5 * bf(b, s, hkv, d), v=bf(b, s, hkv, d), table=ints(table),
                     lengths=ints(_lengths(case)), new=ints(_new_lengths(case)) if case["ragged"] else None)
        state["keys"], state["ke"] = _coded(gen, size, case["layers"], hkv, PAGE, d)
        state["values"], state["ve"] = _coded(gen, size, case["layers"], hkv, d, PAGE)
        return state
    table, lens, counts, src, dst = _pool_plan(case)
    state.update(pages=ints(table), lengths=ints(lens), counts=ints(counts), missing=ints([0]))
    if src is not None:
        state.update(src=ints(src), dst=ints(dst))
    if case["kind"] == "turnover":
        state["dst"] += torch.randint(0, 100, state["dst"].shape, generator=gen, device=device, dtype=torch.int32) * (state["dst"] > 0)
    else:
        shape = (len(counts), case["layers"], case["hkv"])
        codes = lambda a, b: torch.randint(0, 127, (*shape, a, b), generator=gen, device=device, dtype=torch.uint8).view(F8)
        exps = lambda: torch.randint(-20, 20, shape, generator=gen, device=device, dtype=torch.int8)
        state.update(keys=codes(PAGE, case["d"]), values=codes(case["d"], PAGE), ke=exps(), ve=exps())
    return state


# ---------------------------------------------------------------- the plain forms

def _turned(x, cos, sin, rd, interleaved):
    """x with the pairs of its first rd columns turned; cos and sin [batch, new, 1, rd / 2]."""
    x = x.float()
    part, rest = x[..., :rd], x[..., rd:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rd // 2], part[..., rd // 2:])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), dim=-1).flatten(-2) if interleaved else torch.cat((u, w), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _rotary(st):
    case = st["case"]
    angle = (st["positions"].double()[..., None] * st["freq"])[:, :, None]
    cos, sin = ((f(angle) * st["amplitude"]).float() for f in (torch.cos, torch.sin))
    turn = lambda x, way: _turned(x, cos, way * sin, case["rd"], case["interleaved"]).to(x.dtype)
    with torch.no_grad():
        out = turn(st["q"], 1.0), turn(st["k"], 1.0)
        return (*out, turn(st["dq"], -1.0), turn(st["dk"], -1.0)) if case["grad"] else out


def _append(st, codes, exps, new_rows, transposed):
    """The new rows [batch, new, heads, d] into the pages of their places, each page under the exponent
    that its old and new tokens need."""
    case, layer = st["case"], st["case"]["layers"] - 1
    raw = codes.view(torch.uint8)
    n, s = st["lengths"].long(), case["new"]
    fresh = st["new"].long() if st["new"] is not None else torch.full_like(n, s)
    touched = (s + PAGE - 1) // PAGE + 1                                      # pages that a row's new tokens may lie in
    index = n[:, None] // PAGE + torch.arange(touched, device=n.device)       # [batch, touched]
    place = index[..., None] * PAGE + torch.arange(PAGE, device=n.device)     # [batch, touched, 64]
    i = place - n[:, None, None]
    is_new, is_old = (i >= 0) & (i < fresh[:, None, None]), i < 0
    page = st["table"].long().gather(1, index.clamp(max=st["table"].shape[1] - 1))
    sel = is_new.any(-1) & (page >= 0) & (index < st["table"].shape[1])
    page, is_new, is_old = page[sel], is_new[sel], is_old[sel]                # of the pages to write
    row = torch.arange(len(n), device=n.device)[:, None].expand_as(sel)[sel]
    x = new_rows[row[:, None], i[sel].clamp(0, s - 1)].float()                # [written, 64, heads, d]
    x = (x * is_new[..., None, None]).transpose(1, 2)                         # [written, heads, 64, d]
    need = _exponent(x.abs().amax((-2, -1)))
    had = exps[page, layer].int()
    e = torch.where(is_old.any(-1)[:, None], torch.maximum(had, need), need)
    held = raw[page, layer].view(F8).float()
    held = held.mT if transposed else held
    moved = torch.ldexp(held, (had - e)[..., None, None])
    got = torch.where(is_new[:, None, :, None], torch.ldexp(x, -e[..., None, None]),
                      torch.where(is_old[:, None, :, None], moved, held)).to(F8)
    raw[page, layer] = (got.mT if transposed else got).contiguous().view(torch.uint8)
    exps[page, layer] = e.to(torch.int8)


def _attend(st):
    case, layer = st["case"], st["case"]["layers"] - 1
    _append(st, st["keys"], st["ke"], st["k"], False)
    _append(st, st["values"], st["ve"], st["v"], True)
    b, s, hq, hkv, d = (case[x] for x in ("batch", "new", "hq", "hkv", "d"))
    n = st["lengths"].long()
    fresh = st["new"].long() if st["new"] is not None else torch.full_like(n, s)
    page = st["table"].long().clamp(min=0)
    read = lambda codes, exps: torch.ldexp(codes.view(torch.uint8)[page, layer].view(F8).float(), exps[page, layer].int()[..., None, None])
    k = read(st["keys"], st["ke"]).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    v = read(st["values"], st["ve"]).permute(0, 2, 1, 4, 3).reshape(b, hkv, -1, d)
    q = st["q"].float().view(b, s, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    scores = torch.matmul(q, k.mT).view(b, hq, s, -1) / math.sqrt(d)
    at, i = torch.arange(k.shape[2], device=n.device), torch.arange(s, device=n.device)
    seen = (at < (n + fresh)[:, None]) & (st["table"] >= 0).repeat_interleave(PAGE, dim=1)
    seen = seen[:, None, :] & (i < fresh[:, None])[..., None]
    if case["causal"]:
        seen = seen & (at <= (n[:, None] + i)[..., None])
    scores = scores.masked_fill(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hkv, -1, k.shape[2]), v).view(b, hq, s, d)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return out.transpose(1, 2).to(torch.bfloat16), st["keys"], st["values"], st["ke"], st["ve"]


def _take_free(counts, wanted):
    """The lowest free page for each wanted place (in the order of the flat mask), -1 past the last; and how many are missing."""
    free = (counts == 0).nonzero().flatten()
    rank = wanted.flatten().long().cumsum(0).view(wanted.shape) - 1
    got = torch.where(wanted & (rank < len(free)), torch.cat((free, free.new_full((1,), -1)))[rank.clamp(0, len(free))], -1)
    counts[got[got >= 0]] = 1
    return got.int(), (wanted.sum() - (got >= 0).sum()).int()


def _pool(st):
    return [st[x].view(torch.uint8) if x in ("keys", "values") else st[x] for x in ("keys", "values", "ke", "ve")]


def _fork(st):
    pages, lengths, counts = st["pages"], st["lengths"], st["counts"]
    moved = st["src"] != st["dst"]
    src, dst = st["src"][moved].long(), st["dst"][moved].long()
    slot = torch.arange(pages.shape[1], device=pages.device)
    old, n = pages[src].long(), lengths[src].long()
    full, part = n // PAGE, n % PAGE > 0
    tail = torch.where(part, old.gather(1, full.clamp(max=len(slot) - 1)[:, None])[:, 0], -1)
    # a source that is itself replaced leaves its last page to the first row that goes on from it
    gone = torch.zeros(len(pages), dtype=torch.bool, device=pages.device)
    gone[dst] = True
    order = torch.arange(len(src), device=pages.device)
    first = torch.full((len(pages),), len(src), device=pages.device).scatter_reduce(0, src, order, "amin")
    heir = part & gone[src] & (first[src] == order) & (tail >= 0) & (counts[tail.clamp(min=0)] == 1)
    count = lambda x, by: counts.index_add_(0, x[x >= 0], torch.full_like(x[x >= 0], by, dtype=torch.int32))
    count(pages[dst].long().flatten(), -1)
    shared = torch.where(slot < full[:, None], old, -1)
    count(shared.flatten(), 1)
    count(torch.where(heir, tail, -1), 1)
    copied = part & ~heir & (tail >= 0)
    new, missing = _take_free(counts, copied)
    st["missing"] += missing
    last = torch.where(heir, tail, new.long())
    lengths[dst] = n.int()
    pages[dst] = torch.where((slot == full[:, None]) & part[:, None], last[:, None], shared).int()
    copied = copied & (new >= 0)
    for x in _pool(st):
        x[new[copied].long()] = x[tail[copied]]
    return [pages, lengths, counts, st["missing"], st["keys"], st["values"], st["ke"], st["ve"]]


def _compact(st):
    pages, counts = st["pages"].clone(), st["counts"].clone()  # the program keeps its table of before
    at = torch.arange(len(counts), device=counts.device)
    held = counts > 0
    used = held.sum()
    src, hole = (held & (at >= used)).nonzero().flatten(), (~held & (at < used)).nonzero().flatten()
    at[src] = hole
    for x in _pool(st):
        x[hole] = x[src]
    counts[hole], counts[src] = counts[src], 0
    pages = torch.where(pages >= 0, at[pages.long().clamp(min=0)].int(), pages)
    return [used.int().view(1), pages, counts, st["keys"], st["values"], st["ke"], st["ve"]]


def _turnover(st):
    pages, lengths, counts = st["pages"], st["lengths"], st["counts"]
    rows = st["src"].long()
    gone = pages[rows].long().flatten()
    gone = gone[gone >= 0]
    counts.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    pages[rows], lengths[rows] = -1, 0
    until = (lengths + st["dst"] + PAGE - 1) // PAGE * (st["dst"] > 0)
    wanted = (torch.arange(pages.shape[1], device=pages.device) < until[:, None]) & (pages < 0)
    got, missing = _take_free(counts, wanted)
    pages.copy_(torch.where(wanted, got, pages))
    st["missing"] += missing
    lengths += st["dst"]
    return [pages, lengths, counts, st["missing"]]


# ---------------------------------------------------------------- the framework's calls

def _own(st):
    from mimir_amd import paged, rotary

    case = st["case"]
    if case["kind"] == "rotary":
        table = rotary.RotaryFrequencies(st["turns"], st["amplitude"], case["interleaved"])
        q, k = rotary.rotary(st["q"], st["k"], st["positions"], table)
        if not case["grad"]:
            return q, k
        return (q, k, *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"])))
    if case["kind"] == "attend":
        cache = paged.PagedCache(st["keys"], st["values"], st["ke"], st["ve"])
        out = paged.attention_with_pages(st["q"], st["k"], st["v"], cache, case["layers"] - 1, st["table"], st["lengths"],
                                         case["causal"], new_lengths=st["new"])
        return out, *cache
    if case["kind"] == "compact":
        table = paged.PageTable(st["pages"].clone(), st["lengths"], st["counts"].clone(), st["missing"])
        cache = paged.PagedCache(st["keys"], st["values"], st["ke"], st["ve"])
        return [paged.compact_pages(cache, table), table.pages, table.counts, *cache]
    table = paged.PageTable(st["pages"], st["lengths"], st["counts"], st["missing"])
    if case["kind"] == "fork":
        cache = paged.PagedCache(st["keys"], st["values"], st["ke"], st["ve"])
        paged.fork_rows(cache, table, st["src"], st["dst"])
        return [*table, *cache]
    paged.release_rows(table, st["src"])
    paged.reserve_pages(table, st["dst"])
    table.lengths.add_(st["dst"])
    return [*table]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _rotary, "attend": _attend, "fork": _fork, "compact": _compact, "turnover": _turnover}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "rotary":
        rows, e = case["batch"] * case["new"], 2 if case["dtype"] == "bf16" else 4
        heads, passes = case["hq"] + case["hkv"], 2 if case["grad"] else 1
        return dict(bytes=passes * (2 * rows * heads * case["d"] * e + 8 * rows) + 4 * case["rd"],
                    flops=passes * rows * (3 * heads * case["rd"] + 10 * case["rd"]))
    if case["kind"] == "attend":
        s, hq, hkv, d = (case[x] for x in ("new", "hq", "hkv", "d"))
        both = list(zip(_lengths(case), _new_lengths(case)))
        cached, new = sum(n for n, m in both if m), sum(m for _, m in both)
        pairs = sum(n * m + (m * (m + 1) // 2 if case["causal"] else m * m) for n, m in both)
        held = 2 * hkv * d  # bytes of a token's key and value
        # cached tokens in, new ones in (bf16) and out (8 bits), q in, the output of all rows
        return dict(bytes=cached * held + new * held * 3 + new * hq * d * 2 + case["batch"] * s * hq * d * 2
                    + 4 * sum(-(-(n + m) // PAGE) * (1 + hkv // 2) for n, m in both), flops=4 * hq * d * pairs)
    table, lens, counts, src, dst = _pool_plan(case)
    slots = 4 * len(table) * len(table[0])
    if case["kind"] == "turnover":
        return dict(bytes=2 * 4 * len(counts) + slots // len(table) * len(src) * 2, flops=len(counts))
    page = case["layers"] * case["hkv"] * (2 * PAGE * case["d"] + 2)
    if case["kind"] == "fork":
        copies = sum(a != b and lens[a] % PAGE > 0 for a, b in zip(src, dst))
        return dict(bytes=2 * copies * page + 2 * slots + 8 * len(counts), flops=len(counts))
    used = sum(c > 0 for c in counts)
    return dict(bytes=2 * page * sum(c > 0 for c in counts[used:]) + 2 * slots + 8 * len(counts), flops=len(counts))


# ---------------------------------------------------------------- 64-bit results

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rotary":
            return _exact_rotary(case, st)
        if case["kind"] == "attend":
            return _exact_attend(case, st)
        if case["kind"] == "turnover":
            return None
        return _exact_pool(case, st)


def _exact_rotary(case, st):
    rd, z = case["rd"], torch.exp(1j * st["positions"].double()[..., None, None] * st["freq"]) * st["amplitude"]

    def turn(x, z):  # pairs as complex numbers
        x = x.double()
        head = x[..., :rd].unflatten(-1, (rd // 2, 2) if case["interleaved"] else (2, rd // 2))
        head = head if case["interleaved"] else head.mT
        y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * z)
        return torch.cat(((y if case["interleaved"] else y.mT).flatten(-2), x[..., rd:]), dim=-1)

    out = turn(st["q"], z), turn(st["k"], z)
    return (*out, turn(st["dq"], z.conj()), turn(st["dk"], z.conj())) if case["grad"] else out


def _exact_page(codes, exps, at, old, new):
    """One page [heads, 64, d] after the rows `new` [m, heads, d] went to its slots at.. over `old` kept ones, as values."""
    held = codes.double()
    need = new.abs().amax((0, 2)) / 448.0
    e = torch.where(need > 0, torch.ceil(torch.log2(need)), torch.full_like(need, E_MIN)).clamp(min=E_MIN)
    e = torch.where(need > torch.exp2(e), e + 1, e)  # a logarithm just below a whole number
    e = torch.where((need <= torch.exp2(e - 1)) & (e > E_MIN), e - 1, e)
    if old:
        e = torch.maximum(e, exps.double())
        held[:, :old] = (held[:, :old] * torch.exp2(exps.double() - e)[:, None, None]).float().to(F8).double()
    held[:, at:at + len(new)] = (new.transpose(0, 1) * torch.exp2(-e)[:, None, None]).float().to(F8).double()
    return held, e


def _exact_attend(case, st):
    layer, s, hq, hkv, d = case["layers"] - 1, case["new"], case["hq"], case["hkv"], case["d"]
    table, _ = _attend_table(case)
    out = torch.zeros(case["batch"], s, hq, d, dtype=torch.float64, device=st["q"].device)
    for b, (n, m) in enumerate(zip(_lengths(case), _new_lengths(case))):
        if m == 0:
            continue
        full, last = n // PAGE, -(-(n + m) // PAGE)
        kv = []
        for codes, exps, new, turned in ((st["keys"], st["ke"], st["k"], False), (st["values"], st["ve"], st["v"], True)):
            pages = torch.tensor(table[b][:last], device=codes.device)
            c = codes.view(torch.uint8)[pages, layer].view(F8).double()
            c = c.mT.contiguous() if turned else c
            e = exps[pages, layer].double()
            for j in range(full, last):
                lo, hi = max(n, j * PAGE), min(n + m, (j + 1) * PAGE)
                c[j], e[j] = _exact_page(c[j], e[j], lo - j * PAGE, max(0, n - j * PAGE), new[b, lo - n:hi - n].double())
            kv.append((c * torch.exp2(e)[..., None, None]).transpose(0, 1).reshape(hkv, -1, d)[:, :n + m])
        k, v = (x.repeat_interleave(hq // hkv, dim=0) for x in kv)
        for a in range(0, m, 256):
            q = st["q"][b, a:min(m, a + 256)].double().transpose(0, 1)
            p = torch.matmul(q, k.mT) / math.sqrt(d)
            if case["causal"]:
                p.masked_fill_(torch.arange(n + m, device=p.device) > n + a + torch.arange(q.shape[1], device=p.device)[:, None], -math.inf)
            out[b, a:a + q.shape[1]] = torch.matmul(torch.softmax(p, dim=-1), v).transpose(0, 1)
    return out, None, None, None, None


def _exact_pool(case, st):
    """The pool's codes after the pages' moves, found one page at a time from plain lists."""
    if st["keys"].numel() > 1 << 30:
        return None
    table, lens, counts, src, dst = _pool_plan(case)
    moves, used = [], sum(c > 0 for c in counts)
    if case["kind"] == "compact":
        holes = iter([p for p in range(used) if counts[p] == 0])
        moves = [(p, next(holes)) for p in range(used, len(counts)) if counts[p] > 0]
    else:  # no survivor is replaced here: every other row frees its pages and copies its source's last one
        pairs = [(a, b) for a, b in zip(src, dst) if a != b]
        for _, b in pairs:
            for p in table[b]:
                counts[p] -= p >= 0
        for a, _ in pairs:
            for p in table[a][:lens[a] // PAGE]:
                counts[p] += 1
        free = iter([p for p, c in enumerate(counts) if c == 0])
        moves = [(table[a][lens[a] // PAGE], next(free)) for a, _ in pairs if lens[a] % PAGE]
    keys, values = st["keys"].float(), st["values"].float()
    for a, b in moves:
        keys[b], values[b] = keys[a], values[a]
    before = 1 if case["kind"] == "compact" else 2
    return [None] * (before + 2) + [keys, values, None, None]
