"""Plain 64-bit forms of normed rotary heads, cross attention, beam selection and row reordering, for tests.

Each is written from its definition with loops over sequences, heads and rows, and returns next to its results the
sizes (sums of magnitudes) that rounding errors are measured against."""

import math

import torch


def _f64(t):
    return t.detach().cpu().double()


# ---------------------------------------------------------------- normed rotary heads

def _pairs(x, rd, interleaved):
    """The turned columns of x [..., d] as (first, second) of each pair."""
    return (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., :rd // 2], x[..., rd // 2:rd])


def _unpairs(x, a, b, rd, interleaved):
    x = x.clone()
    first, second = _pairs(x, rd, interleaved)  # views
    first.copy_(a)
    second.copy_(b)
    return x


def turn(x, angle, amplitude, interleaved):
    """x [tokens, heads, d] in 64 bits turned by angle [tokens, pairs]."""
    rd = 2 * angle.shape[-1]
    a, b = _pairs(x, rd, interleaved)
    c, s = (amplitude * f(angle)[:, None] for f in (torch.cos, torch.sin))
    return _unpairs(x, a * c - b * s, b * c + a * s, rd, interleaved)


def pair_size(x, angle, amplitude, interleaved):
    """|a| + |b| of each turned pair, times the amplitude; |x| of the other columns."""
    rd = 2 * angle.shape[-1]
    a, b = _pairs(x.abs(), rd, interleaved)
    both = (a + b) * abs(amplitude)
    return _unpairs(x.abs(), both, both, rd, interleaved)


def norm_rotary(x, w, positions, freq, amplitude, interleaved, eps):
    """(y, size) for x [tokens, heads, d], w [d] or None."""
    x, angle = _f64(x), positions.cpu().double()[:, None] * torch.tensor(freq, dtype=torch.float64)
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else _f64(w)
    n = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    return turn(n, angle, amplitude, interleaved), pair_size(n, angle, amplitude, interleaved)


def norm_rotary_grad(dy, x, w, positions, freq, amplitude, interleaved, eps):
    """((dx, size), (dw, size))."""
    dy, x, angle = _f64(dy), _f64(x), positions.cpu().double()[:, None] * torch.tensor(freq, dtype=torch.float64)
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else _f64(w)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    g, size = turn(dy, -angle, amplitude, interleaved), pair_size(dy, angle, amplitude, interleaved)
    dx = r * (w * g - x * r * r * (w * g * x).mean(-1, keepdim=True))
    dx_size = r * (w.abs() * size + x.abs() * r * r * (w.abs() * size * x.abs()).mean(-1, keepdim=True))
    return (dx, dx_size), ((r * g * x).sum((0, 1)), (r * size * x.abs()).sum((0, 1)))


# ---------------------------------------------------------------- cross attention

def cross_attention(q, k, v, cu_q, cu_k, scale, dout=None):
    """out, and with dout (dq, dk, dv), each with its size: packed q [tq, hq, d] over k, v [tk, hkv, d].

    Sizes: of out sum_j p |v|; of the gradients the same products with magnitudes, |dS| taken as
    p (|dO| |V|^T + |delta|) with delta of magnitudes."""
    q, k, v = _f64(q), _f64(k), _f64(v)
    group = q.shape[1] // k.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    sizes = [torch.zeros_like(t) for t in (q, k, v)]
    for a, b, c, e in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if b <= a or e <= c:
            continue
        for h in range(q.shape[1]):
            qh, kh, vh = q[a:b, h], k[c:e, h // group], v[c:e, h // group]
            p = torch.softmax(qh @ kh.t() * scale, dim=-1)
            out[a:b, h], size[a:b, h] = p @ vh, p @ vh.abs()
            if dout is None:
                continue
            do = _f64(dout)[a:b, h]
            delta = (do * out[a:b, h]).sum(-1, keepdim=True)
            ds = p * (do @ vh.t() - delta) * scale
            ds_size = p * (do.abs() @ vh.abs().t() + (do.abs() * size[a:b, h]).sum(-1, keepdim=True)) * scale
            grads[0][a:b, h], sizes[0][a:b, h] = ds @ kh, ds_size @ kh.abs()
            grads[1][c:e, h // group] += ds.t() @ qh
            sizes[1][c:e, h // group] += ds_size.t() @ qh.abs()
            grads[2][c:e, h // group] += p.t() @ do
            sizes[2][c:e, h // group] += p.t() @ do.abs()
    return ((out, size),) if dout is None else ((out, size), *zip(grads, sizes))


def attention_to_states(q, keys, values, lengths, rows, scale):
    """(out, size) for q [batch, s, hq, d] over rows of keys / values [pool, length, hkv, d]: batch row i reads
    the states of row rows[i // (batch // len(rows))]."""
    batch, s, hq, d = q.shape
    beams = batch // len(rows)
    group = hq // keys.shape[2]
    out, size = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for i in range(batch):
        r = int(rows[i // beams])
        if not 0 <= r < keys.shape[0]:
            continue
        n = min(max(int(lengths[r]), 0), keys.shape[1])
        for h in range(hq if n else 0):
            k, v = _f64(keys[r, :n, h // group]), _f64(values[r, :n, h // group])
            p = torch.softmax(_f64(q[i, :, h]) @ k.t() * scale, dim=-1)
            out[i, :, h], size[i, :, h] = p @ v, p @ v.abs()
    return out, size


# ---------------------------------------------------------------- beams

def beam_scores(logits, scores, finished=None, end_token=None):
    """[requests, beams, vocab] 64-bit scores of all continuations; -inf where there is none."""
    x = _f64(logits)
    s = _f64(scores)
    log_p = torch.log_softmax(x, dim=-1)
    lost = ~torch.isfinite(torch.logsumexp(x, dim=-1))  # NaN or +inf among the logits, or nothing finite
    out = torch.where(lost[..., None] | ~torch.isfinite(s)[..., None], -math.inf, s[..., None] + log_p)
    if finished is not None:
        for r, w in finished.cpu().nonzero().tolist():
            out[r, w] = -math.inf
            out[r, w, end_token] = s[r, w] if math.isfinite(s[r, w]) else -math.inf
    return out


def select_beams(logits, scores, count, finished=None, end_token=None):
    """(scores, tokens, rows, finished): the best `count` continuations, ties to the lowest beam, then token."""
    every = beam_scores(logits, scores, finished, end_token)
    requests, beams, vocab = every.shape
    best, order = torch.sort(every.flatten(1), dim=1, descending=True, stable=True)
    best, order = best[:, :count], order[:, :count]
    beam, token = order // vocab, order % vocab
    done = None
    if end_token is not None:
        done = token == end_token
        if finished is not None:
            done = done | finished.cpu().gather(1, beam)
    return best, token, beam + beams * torch.arange(requests)[:, None], done


def reorder_rows(tensors, lengths, source):
    """(new tensors, new lengths): row i takes the first lengths[source[i]] positions of row source[i], if that is in its group."""
    w = source.shape[1]
    out, lens = [t.detach().cpu().clone() for t in tensors], lengths.cpu().clone()
    for i, j in enumerate(source.flatten().tolist()):
        if j == i or j // w != i // w or j < 0:
            continue
        n = min(max(int(lengths[j]), 0), tensors[0].shape[1])
        for t, y in zip(tensors, out):
            y[i, :n] = t[j, :n].detach().cpu()
        lens[i] = lengths[j]
    return out, lens
