"""CPU restatement, in 64 bits and one token at a time, of the paged 8-bit cache
(mimir_amd.paged), of its pages' bookkeeping and of rotary positions (mimir_amd.rotary).
Test infrastructure only; written from the definitions, without torch's 8-bit casts."""

from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 64
E_MIN = -100


def _e4m3_values():
    """The value of each code: sign, 4 exponent bits (bias 7), 3 fraction bits; the last code of each sign is NaN."""
    out = []
    for code in range(256):
        e, f = code >> 3 & 15, code & 7
        x = math.ldexp(f, -9) if e == 0 else math.ldexp(8 + f, e - 10)
        out.append((-x if code & 128 else x) if code & 127 != 127 else math.nan)
    return np.array(out)


VALUES = _e4m3_values()
_POS = VALUES[:127]
_MID = (_POS[1:] + _POS[:-1]) / 2


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest codes of values within +-448, ties to the even code; NaN for NaN and infinities."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    lower = np.searchsorted(_MID, a, side="left")     # codes whose upper midpoint lies below a
    tie = (lower < 126) & (a == _MID[np.minimum(lower, 125)])
    code = lower + (tie & (lower % 2 == 1))
    code = np.where(np.isfinite(x), code, 127)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def exponent(amax: float) -> int:
    """The smallest e >= E_MIN with amax <= 448 * 2^e."""
    e = E_MIN
    while amax > math.ldexp(448.0, e):
        e += 1
    return e


class Cache:
    """Codes as uint8 arrays: keys [pages, layers, heads, 64, d], values [pages, layers, heads, d, 64]."""

    def __init__(self, keys, values, ke, ve):
        raw = lambda t: t.detach().cpu().view(torch.uint8).numpy().copy()  # noqa: E731
        self.keys, self.values, self.ke, self.ve = raw(keys), raw(values), ke.cpu().numpy().copy(), ve.cpu().numpy().copy()

    def _append(self, codes, exps, slots, new, held):
        """codes [tokens 64, d] and exps (a one-element view) of one page and head."""
        finite = np.abs(new[np.isfinite(new)])
        e = exponent(finite.max() if finite.size else 0.0)
        if held > 0:
            old = int(exps)
            e = max(e, old)
            if e > old:
                codes[:held] = encode(VALUES[codes[:held]] * 2.0 ** (old - e))
        codes[slots] = encode(new * 2.0 ** -e)
        return e

    def attend(self, q, k, v, layer, table, lengths, causal, rows=None, new=None, scale=None):
        """Appends, then the output in 64 bits and how far a kernel may be from it, element by element.

        A kernel may hold queries as two 8-bit halves hi + lo 2^-4 under a power of two of each row and 32 columns (two
        runs of 16, 32 apart), and probabilities as bf16.  With |x| at most 2^8.8, hi is off by at most 2^-4 of x, lo by
        2^-4 of that rest, 2^-8 of x together, which bf16 elements do not need (their bits end there), or by half the
        smallest code step, 2^-10, times 2^-4.  The largest of the 32 lies above 224 = 2^7.8 under its power of two, so
        that is 2^-14 / 2^7.8 < 2^-21 of it.  Rounding to bf16 is off by at most 2^-8.

        So a score is off by at most s = (d + 8) 2^-24 sum |q k| (its fp32 sums and the exponent's argument) + 2^-21
        (the exponential's own approximation) + 2^-21 sum max |q| sum |k| over the 32s; an output by (2 s + 2^-8) sum p |v| / sum p
        (the sum of the probabilities moves by s as well), by (n / 32 + 64) 2^-24 of that for the fp32 sums over n
        tokens (partial sums of 32 tokens a product, joined), and by its own rounding, 2^-8 of it."""
        q, k, v = (x.detach().cpu().double().numpy() for x in (q, k, v))
        B, S, hq, d = q.shape
        hkv = k.shape[2]
        out, tol = np.zeros(q.shape), np.zeros(q.shape)
        scale = 1 / math.sqrt(d) if scale is None else scale
        pages, width = self.keys.shape[0], table.shape[1]
        table, lengths = table.cpu().numpy(), lengths.cpu().numpy()
        rows = np.arange(B) if rows is None else rows.cpu().numpy()
        new = np.full(B, S) if new is None else new.cpu().numpy()
        row_ok = [0 <= rows[b] < len(table) and lengths[b] >= 0 and new[b] > 0 for b in range(B)]
        new = np.minimum(new, S)
        ok = lambda p: 0 <= p < pages  # noqa: E731
        for b in range(B):
            if not row_ok[b]:
                continue
            n, m = int(min(lengths[b], width * PAGE)), int(new[b])
            for i in range(n // PAGE, min(width, -(-(n + m) // PAGE))):
                page = int(table[rows[b], i])
                if not ok(page):
                    continue
                lo, hi = max(n, i * PAGE), min(n + m, (i + 1) * PAGE)
                if lo >= hi:
                    continue
                slots = slice(lo - i * PAGE, hi - i * PAGE)
                for h in range(hkv):
                    self.ke[page, layer, h] = self._append(self.keys[page, layer, h], self.ke[page, layer, h], slots,
                                                           k[b, lo - n:hi - n, h], lo - i * PAGE)
                    self.ve[page, layer, h] = self._append(self.values[page, layer, h].T, self.ve[page, layer, h], slots,
                                                           v[b, lo - n:hi - n, h], lo - i * PAGE)
        for b in range(B):
            if not row_ok[b]:
                continue
            n, m = int(min(lengths[b], width * PAGE)), int(new[b])
            kv = min(n + m, width * PAGE)
            held = [int(table[rows[b], i]) for i in range(-(-kv // PAGE))]
            there = np.repeat([ok(p) for p in held], PAGE)[:kv]
            at = [p if ok(p) else 0 for p in held]
            for h in range(hkv):
                kk = (VALUES[self.keys[at, layer, h]] * 2.0 ** self.ke[at, layer, h].astype(float)[:, None, None]).reshape(-1, d)[:kv]
                vv = (VALUES[self.values[at, layer, h]] * 2.0 ** self.ve[at, layer, h].astype(float)[:, None, None]).transpose(0, 2, 1).reshape(-1, d)[:kv]
                for i in range(m):
                    see = there & (np.arange(kv) <= (n + i if causal else kv))
                    if not see.any():
                        continue
                    qq = q[b, i, h * (hq // hkv):(h + 1) * (hq // hkv)]
                    ks, vs = kk[see], vv[see]
                    s = qq @ ks.T * scale
                    with np.errstate(invalid="ignore", over="ignore"):
                        p = np.exp(s - s.max(1, keepdims=True))
                        total = p.sum(1, keepdims=True)
                        o = (p @ vs) / total
                        spread = (p @ np.abs(vs)) / total
                        off = (d + 8) * 2.0 ** -24 * (np.abs(qq) @ np.abs(ks).T * scale).max(1, keepdims=True) + 2.0 ** -21
                        blocks = lambda x: np.abs(x).reshape(len(x), d // 64, 2, 2, 16)  # noqa: E731
                        rest = np.einsum("qsb,ksb->qk", blocks(qq).max((2, 4)), blocks(ks).sum((2, 4)))
                        off = off + 2.0 ** -21 * scale * rest.max(1, keepdims=True)
                        slack = (2 * off + 2.0 ** -8 + (kv / 32 + 64) * 2.0 ** -24) * spread
                    out[b, i, h * (hq // hkv):(h + 1) * (hq // hkv)] = o
                    tol[b, i, h * (hq // hkv):(h + 1) * (hq // hkv)] = slack + 2.0 ** -8 * (np.abs(o) + slack)
        return out, tol

    def move(self, moves):
        """Pages (from, to), all read before any is written."""
        for x in (self.keys, self.values, self.ke, self.ve):
            held = [x[a].copy() for a, _ in moves]
            for (_, to), y in zip(moves, held):
                x[to] = y


class Table:
    """pages as lists, lengths, counts, missing; every call as its definition reads."""

    def __init__(self, pages, lengths, counts, missing):
        self.pages, self.lengths, self.counts = pages.tolist(), lengths.tolist(), counts.tolist()
        self.missing = int(missing[0])

    def ok(self, p):
        return 0 <= p < len(self.counts)

    def free(self):
        for p, c in enumerate(self.counts):
            if c == 0:
                self.counts[p] = 1
                return p
        self.missing += 1
        return -1

    def release(self, rows):
        for r in rows:
            if not 0 <= r < len(self.pages):
                continue
            for p in self.pages[r]:
                if self.ok(p):
                    self.counts[p] -= 1
            self.pages[r] = [-1] * len(self.pages[r])
            self.lengths[r] = 0

    def reserve(self, new):
        for r, m in enumerate(new):
            if m <= 0:
                continue
            for i in range(min(len(self.pages[r]), -(-(max(self.lengths[r], 0) + m) // PAGE))):
                if not self.ok(self.pages[r][i]):
                    self.pages[r][i] = self.free()

    def fork(self, src, dst):
        """Returns the pages to copy, (from, to)."""
        n = len(self.pages)
        last = {d: s for s, d in zip(src, dst) if 0 <= s < n and 0 <= d < n}
        at = {d: i for i, (s, d) in enumerate(zip(src, dst)) if 0 <= s < n and 0 <= d < n}
        kept = sorted((at[d], s, d) for d, s in last.items() if s != d)
        before, lengths, plan = [list(p) for p in self.pages], list(self.lengths), []
        for _, s, d in kept:
            full, tail = max(lengths[s], 0) // PAGE, -1
            if lengths[s] > 0 and lengths[s] % PAGE and full < len(before[s]):
                tail = before[s][full]
            plan.append((d, [p if i < full and self.ok(p) else -1 for i, p in enumerate(before[s])], lengths[s], full, tail))
        for d, row, *_ in plan:
            for p in before[d]:
                if self.ok(p):
                    self.counts[p] -= 1
            for p in row:
                if p >= 0:
                    self.counts[p] += 1
        copies = []
        for d, row, length, full, tail in plan:
            if self.ok(tail) and self.counts[tail] == 0:  # given back by all: the first to go on from it
                row[full], self.counts[tail] = tail, 1
            elif self.ok(tail):
                copies.append((tail, row, full))
            self.pages[d], self.lengths[d] = row, length
        moves = []
        for tail, row, full in copies:
            row[full] = self.free()
            if row[full] >= 0:
                moves.append((tail, row[full]))
        assert not {a for a, _ in moves} & {b for _, b in moves}, moves
        return moves

    def compact(self):
        """Returns (used, moves)."""
        used = sum(c > 0 for c in self.counts)
        holes = [p for p in range(used) if self.counts[p] <= 0]
        late = [p for p in range(used, len(self.counts)) if self.counts[p] > 0]
        to = dict(zip(late, holes))
        for a, b in to.items():
            self.counts[b], self.counts[a] = self.counts[a], 0
        self.pages = [[to.get(p, p) for p in row] for row in self.pages]
        return used, list(to.items())


def rotary(x, positions, freq, amplitude, interleaved, inverse=False):
    """x [tokens, heads, d] turned by positions [tokens] * freq, as complex numbers in 64 bits, and the
    sum |a| + |b| of each column's pair (0 past the turned ones)."""
    x = x.detach().cpu().double()
    n = len(freq)
    angle = positions.cpu().double()[:, None, None] * torch.tensor(freq, dtype=torch.float64)
    z = torch.polar(torch.full_like(angle, amplitude), -angle if inverse else angle)
    head = x[..., :2 * n].unflatten(-1, (n, 2) if interleaved else (2, n))
    head = head if interleaved else head.mT
    y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * z)
    size = (head.abs().sum(-1, keepdim=True) * abs(amplitude)).expand_as(y)
    flat = lambda t: (t if interleaved else t.mT).flatten(-2)  # noqa: E731
    return torch.cat((flat(y), x[..., 2 * n:]), -1), torch.cat((flat(size), torch.zeros_like(x[..., 2 * n:])), -1)
