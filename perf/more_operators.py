"""The measured cases of normed rotary heads, cross attention and beam search.

Each case is one call path of a training or serving program:

* ``norm``    -- ``norm_rotary``: the query and key heads of a fused projection, each normed by its
  root mean square, scaled by a learned weight and turned by its position; (training) the gradients;
* ``cross``   -- ``cross_attention``: packed queries over another packed set of states (an encoder's),
  each sequence with lengths of its own; (training) the gradients;
* ``states``  -- ``attention_to_states``: the decode step of the same, the beams or samples of a
  request over one row of a static cache of states;
* ``select``  -- ``select_beams``: the best continuations over a request's beams and the vocabulary;
* ``reorder`` -- ``reorder_rows``: the cache rows of the chosen beams in their new places.

``run`` computes them with elementary torch operations, or (``own``) by the package's calls.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # Serving, a decode step of a small batch at far positions: launch latency.
        dict(name="norm_decode", kind="norm", dtype="bf16", wtype="bf16", batch=8, new=1, hq=16, hkv=4, d=128, rd=128,
             interleaved=False, grad=False, max_pos=60000, pos_seed=1),
        # Training, the headline shape: 8 sequences of 2048, grouped heads, forward and backward.
        dict(name="norm_train", kind="norm", dtype="bf16", wtype="fp32", batch=8, new=2048, hq=16, hkv=4, d=128, rd=128,
             interleaved=False, grad=True, max_pos=0, pos_seed=2),
        # Full-precision training, odd lengths, adjacent pairs of an odd part of the head.
        dict(name="norm_odd", kind="norm", dtype="fp32", wtype="fp32", batch=3, new=683, hq=8, hkv=8, d=64, rd=20,
             interleaved=True, grad=True, max_pos=5000, pos_seed=4),
        # Training: 8 documents of up to 2048 tokens, each over another text of up to 2048.
        dict(name="cross_train", kind="cross", hq=16, hkv=4, d=128, seqs=8, min_q=1500, max_q=2048, min_k=1024, max_k=2048,
             pad_q=0, pad_k=0, len_seed=5, grad=True),
        # Training with small heads: many short packed documents, some without a query or a state, padded at the end.
        dict(name="cross_ragged", kind="cross", hq=8, hkv=8, d=64, seqs=48, min_q=0, max_q=700, min_k=0, max_k=1300,
             pad_q=77, pad_k=130, len_seed=6, grad=True),
        # Scoring a long document against a long one, forward only.
        dict(name="cross_long", kind="cross", hq=32, hkv=8, d=128, seqs=2, min_q=7000, max_q=8192, min_k=12000, max_k=16384,
             pad_q=0, pad_k=0, len_seed=7, grad=False),
        # Serving, one request of 4 beams against a text of 1500 tokens. Launch latency.
        dict(name="states_single", kind="states", requests=1, pool=2, beams=4, new=1, hq=16, hkv=4, d=128, length=1536,
             min_len=1500, max_len=1500, len_seed=8),
        # Serving, a full batch of requests of 8 beams each: reading the states is the work.
        dict(name="states_wide", kind="states", requests=48, pool=64, beams=8, new=1, hq=16, hkv=4, d=128, length=4096,
             min_len=300, max_len=4096, len_seed=9),
        # The first step of one request (one live beam), two candidates a beam, full-precision logits. Launch latency.
        dict(name="select_first", kind="select", dtype="fp32", requests=1, beams=5, vocab=32000, count=10, first=True, ended=0.0,
             banned=0.0, seed=10),
        # 48 requests of 8 beams over a large vocabulary of odd size, some beams ended, some tokens banned.
        dict(name="select_wide", kind="select", dtype="bf16", requests=48, beams=8, vocab=128257, count=8, first=False, ended=0.1,
             banned=0.01, seed=11),
        # The cache rows of 16 requests of 8 beams, two layers, after a selection.
        dict(name="reorder_wide", kind="reorder", requests=16, beams=8, layers=2, length=1024, min_len=200, max_len=1000, hkv=4,
             d=128, kept=0.4, len_seed=13),
        # The same of one request: launch latency.
        dict(name="reorder_single", kind="reorder", requests=1, beams=4, layers=1, length=512, min_len=333, max_len=333, hkv=2,
             d=64, kept=0.5, len_seed=14),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "cross", "cross", "cross", "states", "states", "select", "select", "reorder"])
    seed = rng.randrange(1 << 20)
    if kind == "norm":
        d = rng.choice([64, 128, 128, 80, 96])
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]), wtype="fp32", batch=_log(rng, 1, 64),
                    new=_log(rng, 1, 8192), hq=rng.choice([2, 8, 16, 32]), hkv=rng.choice([1, 2, 4, 8]), d=d,
                    rd=rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)]), interleaved=rng.random() < 0.5,
                    grad=rng.random() < 0.6, max_pos=_log(rng, 1, 1000000), pos_seed=seed)
        case["wtype"] = rng.choice(["fp32", case["dtype"]])
        while work(case)["bytes"] > 4e8:
            case["new"] = (case["new"] + 1) // 2 if case["new"] > 1 else 1
            case["batch"] = max(1, case["batch"] - 1)
        return case
    heads = rng.choice([(16, 4, 128), (8, 8, 64), (2, 2, 128), (32, 8, 128), (8, 2, 64), (8, 1, 128), (12, 4, 64)])
    if kind == "cross":
        hq, hkv, d = heads
        hi_q, hi_k = _log(rng, 1, 4096), _log(rng, 1, 8192)
        case = dict(kind=kind, hq=hq, hkv=hkv, d=d, seqs=_log(rng, 1, 64), min_q=rng.randint(0, hi_q), max_q=hi_q,
                    min_k=rng.randint(0, hi_k), max_k=hi_k, pad_q=rng.choice([0, 0, rng.randint(1, 300)]),
                    pad_k=rng.choice([0, 0, rng.randint(1, 300)]), len_seed=seed, grad=rng.random() < 0.6)
        while case["seqs"] > 1 and (work(case)["flops"] > 3e11 or work(case)["bytes"] > 4e8):
            case["seqs"] //= 2
        while work(case)["flops"] > 3e11:
            case["min_k"], case["max_k"] = case["min_k"] // 2, case["max_k"] // 2
        return case
    if kind == "states":
        hq, hkv, d = heads
        length = _log(rng, 8, 16384)
        case = dict(kind=kind, requests=_log(rng, 1, 48), beams=rng.choice([1, 1, 2, 4, 5, 8]), new=rng.choice([1, 1, 1, rng.randint(2, 7)]),
                    hq=hq, hkv=hkv, d=d, length=length, min_len=rng.randint(0, length), max_len=length, len_seed=seed)
        while case["requests"] > 1 and case["requests"] * length * hkv * d > 48 * 4096 * 4 * 128:
            case["requests"] //= 2
        case["pool"] = case["requests"] + rng.randint(0, 3)
        return case
    if kind == "select":
        case = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]), requests=_log(rng, 1, 64), beams=rng.choice([1, 2, 3, 4, 5, 8, 16]),
                    vocab=_log(rng, 300, 200000), first=rng.random() < 0.2, ended=rng.choice([0.0, 0.2]),
                    banned=rng.choice([0.0, 0.05]), seed=seed)
        case["count"] = case["beams"] * rng.choice([1, 1, 2])
        while case["requests"] > 1 and case["requests"] * case["beams"] * case["vocab"] > 40000000:
            case["requests"] //= 2
        case["vocab"] = min(case["vocab"], 40000000 // case["beams"])
        if case["dtype"] == "fp32":
            case["vocab"] = max(300, case["vocab"] // 2)
        return case
    length = _log(rng, 64, 2048)
    case = dict(kind=kind, requests=_log(rng, 1, 24), beams=rng.choice([2, 3, 4, 5, 8, 16]), layers=rng.choice([1, 1, 2]), length=length,
                min_len=rng.randint(0, length), max_len=length, hkv=heads[1], d=heads[2], kept=rng.choice([0.3, 0.5, 0.8]), len_seed=seed)
    size = lambda: case["requests"] * case["beams"] * case["layers"] * length * heads[1] * heads[2]
    while case["requests"] > 1 and (work(case)["bytes"] > 3e8 or size() > 1 << 27):
        case["requests"] //= 2
    while case["beams"] > 2 and (work(case)["bytes"] > 3e8 or size() > 1 << 27):
        case["beams"] //= 2
    return case


# ---------------------------------------------------------------- plans, as plain lists

def _frequencies(case):
    return [10000.0 ** (-2.0 * i / case["rd"]) for i in range(case["rd"] // 2)]


def _positions(case):
    """[batch, new]: each row counts on from a place of its own."""
    rng = random.Random(case["pos_seed"])
    return [[p + i for i in range(case["new"])] for p in (rng.randint(0, case["max_pos"]) for _ in range(case["batch"]))]


def _pairs(case):
    """(queries, states) of each sequence."""
    rng = random.Random(case["len_seed"])
    one = lambda lo, hi: rng.choice([lo, hi, rng.randint(lo, hi), rng.randint(lo, hi)])
    return [(one(case["min_q"], case["max_q"]), one(case["min_k"], case["max_k"])) for _ in range(case["seqs"])]


def _state_plan(case):
    """(lengths of the pool's rows, the row of each request)."""
    rng = random.Random(case["len_seed"])
    return [rng.randint(case["min_len"], case["max_len"]) for _ in range(case["pool"])], rng.sample(range(case["pool"]), case["requests"])


def _row_plan(case):
    """(lengths, source row) of each cache row: a share of a request's beams stays, the rest go on from those."""
    rng = random.Random(case["len_seed"])
    w = case["beams"]
    lens, src = [], []
    for r in range(case["requests"]):
        lens += [rng.randint(case["min_len"], case["max_len"])] * w
        kept = sorted(rng.sample(range(w), max(1, round(w * case["kept"]))))
        src += [r * w + (b if b in kept else rng.choice(kept)) for b in range(w)]
    return lens, src


# ---------------------------------------------------------------- inputs

def _normal(gen, *shape):
    # projections of normalised activations: near normal, without far tails
    return torch.randn(shape, generator=gen, device=gen.device).clamp_(-5.0, 5.0)


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device).manual_seed(seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    bf = lambda *shape: _normal(gen, *shape).to(torch.bfloat16)
    state = dict(case=case)
    if case["kind"] == "norm":
        b, s, hq, hkv, d = (case[x] for x in ("batch", "new", "hq", "hkv", "d"))
        dtype, wtype = DTYPES[case["dtype"]], DTYPES[case["wtype"]]
        # the fused projection: q and k are views of it; rows of differing size
        qkv = (_normal(gen, b, s, hq + 2 * hkv, d) * torch.exp(0.7 * _normal(gen, b, s, 1, 1))).to(dtype)
        state.update(q=qkv[:, :, :hq], k=qkv[:, :, hq:hq + hkv], positions=torch.tensor(_positions(case), device=device),
                     qw=(1.0 + 0.2 * _normal(gen, d)).to(wtype), kw=(1.0 + 0.2 * _normal(gen, d)).to(wtype))
        if case["grad"]:
            for x in ("q", "k", "qw", "kw"):
                state[x] = state[x].detach().requires_grad_(True)
            state.update(dq=_normal(gen, b, s, hq, d).to(dtype), dk=_normal(gen, b, s, hkv, d).to(dtype))
        freq = _frequencies(case)
        state["freq"] = torch.tensor(freq, dtype=torch.float64, device=device)
        # the same as fractions of a turn per position, in units of 2^-64
        state["turns"] = torch.tensor([round(f / (2.0 * math.pi) * 2.0 ** 64) for f in freq], dtype=torch.int64, device=device)
    elif case["kind"] == "cross":
        hq, hkv, d = (case[x] for x in ("hq", "hkv", "d"))
        at_q, at_k = [0], [0]
        for n, m in _pairs(case):
            at_q.append(at_q[-1] + n)
            at_k.append(at_k[-1] + m)
        tq, tk = at_q[-1] + case["pad_q"], at_k[-1] + case["pad_k"]
        kv = bf(tk, 2 * hkv, d)  # one projection of the states: keys and values are views of it
        state.update(q=bf(tq, hq, d), k=kv[:, :hkv], v=kv[:, hkv:], cu_q=ints(at_q), cu_k=ints(at_k))
        if case["grad"]:
            for x in ("q", "k", "v"):
                state[x] = state[x].detach().requires_grad_(True)
            state["do"] = bf(tq, hq, d)
    elif case["kind"] == "states":
        hq, hkv, d = (case[x] for x in ("hq", "hkv", "d"))
        lens, rows = _state_plan(case)
        state.update(q=bf(case["requests"] * case["beams"], case["new"], hq, d), keys=bf(case["pool"], case["length"], hkv, d),
                     values=bf(case["pool"], case["length"], hkv, d), lengths=ints(lens), rows=ints(rows))
    elif case["kind"] == "select":
        r, w, v = case["requests"], case["beams"], case["vocab"]
        # a request's beams share what is likely; a few tokens stand out
        logits = 1.5 * _normal(gen, r, w, v) + 1.5 * _normal(gen, r, 1, v)
        logits += 9.0 * (torch.rand(r, 1, v, generator=gen, device=device) < 8.0 / v)
        if case["banned"]:
            logits.masked_fill_(torch.rand(r, w, v, generator=gen, device=device) < case["banned"], -math.inf)
        scores = -12.0 * torch.rand(r, w, generator=gen, device=device)
        if case["first"]:
            scores[:, 1:] = -math.inf
        state.update(logits=logits.to(DTYPES[case["dtype"]]), scores=scores, end=2,
                     finished=torch.rand(r, w, generator=gen, device=device) < case["ended"])
    else:
        lens, src = _row_plan(case)
        shape = (case["requests"] * case["beams"], case["length"], case["hkv"], case["d"])
        state.update(keys=[bf(*shape) for _ in range(case["layers"])], values=[bf(*shape) for _ in range(case["layers"])],
                     lengths=ints(lens), src=ints(src).view(case["requests"], case["beams"]))
    return state


# ---------------------------------------------------------------- the plain forms

def _turned(x, cos, sin, rd, interleaved):
    """x with the pairs of its first rd columns turned; cos and sin [batch, new, 1, rd / 2]."""
    part, rest = x[..., :rd], x[..., rd:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rd // 2], part[..., rd // 2:])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((u, w), dim=-1).flatten(-2) if interleaved else torch.cat((u, w), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _norm(st):
    case = st["case"]
    angle = (st["positions"].double()[..., None] * st["freq"])[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    turn = lambda x, way: _turned(x, cos, way * sin, case["rd"], case["interleaved"])
    outs, grads, wgrads = [], [], []
    with torch.no_grad():
        for x, w, g in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
            xf, wf = x.float(), w.float()
            r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
            n = xf * r
            outs.append(turn(n * wf, 1.0).to(x.dtype))
            if case["grad"]:
                gn = turn(g.float(), -1.0)
                wgrads.append((gn * n).sum((0, 1, 2), dtype=torch.float64).to(w.dtype))
                gw = gn * wf
                grads.append((r * (gw - n * (gw * n).mean(-1, keepdim=True))).to(x.dtype))
    return (*outs, *grads, *wgrads)


def _cross(st):
    case = st["case"]
    g, scale = case["hq"] // case["hkv"], 1.0 / math.sqrt(case["d"])
    q, k, v = st["q"].detach(), st["k"].detach(), st["v"].detach()
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=x.device) if case["grad"] else None for x in (q, k, v))
    i = j = 0
    for n, m in _pairs(case):
        a, b = slice(i, i + n), slice(j, j + m)
        i, j = i + n, j + m
        for h in range(case["hkv"] if n and m else 0):
            heads = slice(h * g, h * g + g)
            kh, vh = k[b, h].float(), v[b, h].float()
            qh = q[a, heads].float().transpose(0, 1)                      # [group, n, d]
            s = torch.matmul(qh, kh.t()) * scale
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            out[a, heads] = torch.matmul(p, vh).transpose(0, 1).to(q.dtype)
            if case["grad"]:
                do = st["do"][a, heads].float().transpose(0, 1)
                dp = torch.matmul(do, vh.t())
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                dq[a, heads] = torch.matmul(ds, kh).transpose(0, 1).to(q.dtype)
                dk[b, h] = torch.matmul(ds.flatten(0, 1).t(), qh.flatten(0, 1)).to(q.dtype)
                dv[b, h] = torch.matmul(p.flatten(0, 1).t(), do.flatten(0, 1)).to(q.dtype)
    return (out, dq, dk, dv) if case["grad"] else out


def _states(st):
    case = st["case"]
    hq, hkv, d, s = (case[x] for x in ("hq", "hkv", "d", "new"))
    rows = st["rows"].long()
    n, m = case["requests"], case["beams"] * s * (hq // hkv)
    k, v = (st[x][rows].float().transpose(1, 2) for x in ("keys", "values"))           # [requests, hkv, length, d]
    q = st["q"].float().view(n, case["beams"], s, hkv, hq // hkv, d).permute(0, 3, 1, 2, 4, 5).reshape(n, hkv, m, d)
    scores = torch.matmul(q, k.mT) / math.sqrt(d)
    seen = torch.arange(case["length"], device=rows.device) < st["lengths"].long()[rows][:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(n, hkv, case["beams"], s, hq // hkv, d).permute(0, 2, 3, 1, 4, 5)
    return out.reshape(st["q"].shape).to(torch.bfloat16)


def _candidates(st):
    """[requests, beams * vocab]: the score of each continuation, in 64 bits: neighbours may lie close."""
    logits, ended = st["logits"].double(), st["finished"][..., None]
    top = logits.amax(-1, keepdim=True)
    log_p = logits - (top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True)))
    end = torch.arange(logits.shape[-1], device=logits.device) == st["end"]
    log_p = torch.where(ended, torch.where(end, 0.0, -math.inf), log_p)
    return (st["scores"].double()[..., None] + log_p).flatten(1)


def _select(st):
    x = _candidates(st)
    x = torch.where(x == -math.inf, torch.full_like(x, -1e300), x)  # -inf: taken
    index = torch.arange(x.shape[1], device=x.device)
    best, at = [], []
    for _ in range(st["case"]["count"]):
        top = x.amax(-1, keepdim=True)
        first = torch.where(x == top, index, x.shape[1]).amin(-1, keepdim=True)
        best.append(torch.where(top == -1e300, -math.inf, top))
        at.append(first)
        x = x.scatter(1, first, -math.inf)
    return _chosen(st, torch.cat(best, 1), torch.cat(at, 1))


def _chosen(st, best, at):
    """(scores, tokens, rows, finished) of the chosen places of the flat candidates."""
    w, v = st["case"]["beams"], st["case"]["vocab"]
    beam, token = at // v, at % v
    rows = beam + w * torch.arange(len(at), device=at.device)[:, None]
    return [best.float(), token.int(), rows.int(), st["finished"].gather(1, beam) | (token == st["end"])]


def _reorder(st):
    src = st["src"].flatten().long()
    n = st["lengths"].long()[src]
    moved = (torch.arange(st["case"]["length"], device=n.device) < n[:, None])[..., None, None]
    for x in (*st["keys"], *st["values"]):
        x.copy_(torch.where(moved, x[src], x))
    st["lengths"].copy_(st["lengths"][src])
    return [*st["keys"], *st["values"], st["lengths"]]


# ---------------------------------------------------------------- the framework's calls

def _own(st):
    from mimir_amd import beams, cross, rotary
    from mimir_amd.cache import Cache

    case = st["case"]
    if case["kind"] == "norm":
        table = rotary.RotaryFrequencies(st["turns"], 1.0, case["interleaved"])
        q, k = rotary.norm_rotary(st["q"], st["k"], st["positions"], table, st["qw"], st["kw"], eps=EPS)
        if not case["grad"]:
            return q, k
        return (q, k, *torch.autograd.grad((q, k), (st["q"], st["k"], st["qw"], st["kw"]), (st["dq"], st["dk"])))
    if case["kind"] == "cross":
        out = cross.cross_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"])
        return (out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["do"])) if case["grad"] else out
    if case["kind"] == "states":
        return cross.attention_to_states(st["q"], Cache(st["keys"], st["values"]), st["lengths"], st["rows"])
    if case["kind"] == "select":
        return list(beams.select_beams(st["logits"], st["scores"], case["count"], finished=st["finished"], end_token=st["end"]))
    beams.reorder_rows([Cache(k, v) for k, v in zip(st["keys"], st["values"])], st["lengths"], st["src"])
    return [*st["keys"], *st["values"], st["lengths"]]


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "cross": _cross, "states": _states, "select": _select, "reorder": _reorder}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "norm":
        rows, e, heads = case["batch"] * case["new"], 2 if case["dtype"] == "bf16" else 4, case["hq"] + case["hkv"]
        passes = 5 if case["grad"] else 2  # read and write; read twice and write
        return dict(bytes=passes * rows * heads * case["d"] * e + 8 * rows * (passes // 2) + 16 * case["d"],
                    flops=(passes // 2) * rows * (heads * (6 * case["d"] + 3 * case["rd"]) + 10 * case["rd"]))
    if case["kind"] == "cross":
        hq, hkv, d = (case[x] for x in ("hq", "hkv", "d"))
        pairs = _pairs(case)
        nq, nk = sum(n for n, _ in pairs) + case["pad_q"], sum(m for _, m in pairs) + case["pad_k"]
        both = sum(n * m for n, m in pairs)
        # q, k, v in and the output out; with gradients q, k, v, the output's gradient in and three out
        held = (2 * nq * hq + 2 * nk * hkv) * 2 * d
        return dict(bytes=held + ((3 * nq * hq + 4 * nk * hkv) * 2 * d if case["grad"] else 0),
                    flops=(14 if case["grad"] else 4) * hq * d * both)
    if case["kind"] == "states":
        lens, rows = _state_plan(case)
        n, q = sum(lens[r] for r in rows), case["beams"] * case["new"] * case["hq"] * case["d"]
        return dict(bytes=4 * n * case["hkv"] * case["d"] + 4 * case["requests"] * q, flops=4 * n * q)
    if case["kind"] == "select":
        n, live = case["requests"] * case["beams"], 1.0 - case["ended"]
        return dict(bytes=int(live * n * case["vocab"] * (2 if case["dtype"] == "bf16" else 4)) + 17 * case["requests"] * case["count"],
                    flops=int(4 * live * n * case["vocab"]))
    lens, src = _row_plan(case)
    moved = [i for i, j in enumerate(src) if i != j]
    tokens = sum(lens[j] for j in {src[i] for i in moved}) + sum(lens[src[i]] for i in moved)
    return dict(bytes=tokens * case["layers"] * 4 * case["hkv"] * case["d"] + 8 * len(src), flops=len(src))


# ---------------------------------------------------------------- 64-bit results

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "cross": _exact_cross, "states": _exact_states, "select": _exact_select,
                "reorder": _exact_reorder}[case["kind"]](case, st)


def _exact_norm(case, st):
    rd, z = case["rd"], torch.exp(1j * st["positions"].double()[..., None, None] * st["freq"])

    def turn(x, z):  # pairs as complex numbers
        head = x[..., :rd].unflatten(-1, (rd // 2, 2) if case["interleaved"] else (2, rd // 2))
        head = head if case["interleaved"] else head.mT
        y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * z)
        return torch.cat(((y if case["interleaved"] else y.mT).flatten(-2), x[..., rd:]), dim=-1)

    out, grads, wgrads = [], [], []
    for x, w, g in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
        x, w, d = x.double(), w.double(), case["d"]
        size = torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / d + EPS)
        out.append(turn(x / size * w, z))
        if case["grad"]:
            g = turn(g.double(), z.conj())
            wgrads.append(torch.einsum("bshd,bshd->d", g, x / size))
            grads.append(g * w / size - x * ((g * w * x).sum(-1, keepdim=True) / (d * size ** 3)))
    return (*out, *grads, *wgrads)


def _exact_cross(case, st):
    q, k, v = (st[x].detach().double() for x in ("q", "k", "v"))
    g = case["hq"] // case["hkv"]
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    at_q, at_k = st["cu_q"].tolist(), st["cu_k"].tolist()
    for a, b, c, e in zip(at_q, at_q[1:], at_k, at_k[1:]):
        for h in range(case["hq"] if b > a and e > c else 0):
            kh, vh = k[c:e, h // g], v[c:e, h // g]
            p = torch.softmax(q[a:b, h] @ kh.t() / math.sqrt(case["d"]), dim=-1)
            out[a:b, h] = p @ vh
            if case["grad"]:
                do = st["do"][a:b, h].double()
                grads[2][c:e, h // g] += p.t() @ do
                ds = p * (do @ vh.t() - (do * out[a:b, h]).sum(-1, keepdim=True)) / math.sqrt(case["d"])
                grads[0][a:b, h] = ds @ kh
                grads[1][c:e, h // g] += ds.t() @ q[a:b, h]
    return (out, *grads) if case["grad"] else out


def _exact_states(case, st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    lens, rows = _state_plan(case)
    g, w = case["hq"] // case["hkv"], case["beams"]
    for i, r in enumerate(rows):
        for h in range(case["hq"] if lens[r] else 0):
            k, v = (st[x][r, :lens[r], h // g].double() for x in ("keys", "values"))
            q = st["q"][i * w:(i + 1) * w, :, h].double()
            out[i * w:(i + 1) * w, :, h] = torch.softmax(q @ k.t() / math.sqrt(case["d"]), dim=-1) @ v
    return out


def _exact_select(case, st):
    best, at = [], []
    for i in range(case["requests"]):
        log_p = torch.log_softmax(st["logits"][i].double(), dim=-1)
        for b in st["finished"][i].nonzero().flatten().tolist():
            log_p[b] = -math.inf
            log_p[b, st["end"]] = 0.0
        x, order = torch.sort((st["scores"][i].double()[:, None] + log_p).flatten(), descending=True, stable=True)
        best.append(x[:case["count"]])
        at.append(order[:case["count"]])
    _, *rest = _chosen(st, torch.stack(best), torch.stack(at))
    return [torch.stack(best), *rest]


def _exact_reorder(case, st):
    lens, src = _row_plan(case)
    out = []
    for x in (*st["keys"], *st["values"]):
        y = x.float()
        for i, j in enumerate(src):
            y[i, :lens[j]] = x[j, :lens[j]].float()
        out.append(y)
    return [*out, torch.tensor([lens[j] for j in src], dtype=torch.int32, device=st["lengths"].device)]
