"""Rotary positions from token positions: either pair layout, part of the head, scaled ranges.

``mimir_amd.rope`` rotates by ready cos / sin tables in the rotate-half layout
(src/mimir/model/layers.py:24-40).  :func:`rotary` takes the positions themselves (int32 or
int64, restarting per document, or far along in a decode) and a table of frequencies
(:class:`RotaryFrequencies`): no [tokens, head_dim] tables are built or read, queries and
keys are turned in one launch, and the gradient is the inverse turn.

Frequencies are fractions of a turn per position in units of 2^-64, so that the 64-bit
product with a position wraps at whole turns: for the given ``turns`` the range reduction is
exact at any position.  The rest, within an eighth of a turn, is then rounded to fp32: 2^-28 of
a turn at most.  ``create`` forms its table in 64-bit floats, off by up to 3 * 2^-53 of a
frequency, which far positions multiply: of the fastest pair that stays below 2^-28 of a turn up to
position 7e7.  float32 and bfloat16; no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _capi
from . import prefixlm as P

_DTYPES = {torch.float32: _capi.DTYPE_FLOAT32, torch.bfloat16: _capi.DTYPE_BFLOAT16}
SCALINGS = ("none", "linear", "ntk", "wavelength", "yarn")


class RotaryFrequencies(NamedTuple):
    """``turns`` int64 [rotary_dim / 2] on the device (turn per position of each pair, in units
    of 2^-64), the ``amplitude`` of the turned columns, and the pair layout: pair i is columns
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if ``interleaved``."""
    turns: Tensor
    amplitude: float = 1.0
    interleaved: bool = False

    @staticmethod
    def inverse_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                            original_positions: int = 8192, low_turns: float = 1.0, high_turns: float = 4.0,
                            slow_turns: float = 1.0, fast_turns: float = 32.0):
        """(angle per position of each pair, amplitude), in 64-bit floats, on the host:

        * ``"none"``: base^(-2 i / rotary_dim);
        * ``"linear"``: all divided by ``factor``;
        * ``"ntk"``: base * factor^(n / (n - 2)) for the base, n = rotary_dim: the fastest pair keeps
          its frequency, the slowest is divided by ``factor``;
        * ``"wavelength"``: by the turns t that a pair makes in ``original_positions``: divided by ``factor``
          below ``low_turns``, kept above ``high_turns``, between them mixed by (t - low) / (high - low);
        * ``"yarn"``: mixed by the pair's index, linearly from the (rounded down) one of ``fast_turns``,
          kept, to the (rounded up) one of ``slow_turns``, divided; amplitude 0.1 ln(factor) + 1, and
          1 for a factor below 1.
        """
        n = int(rotary_dim)
        if n < 2 or n % 2:
            raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
        if not base > 1.0 or not factor > 0.0 or not original_positions > 0:
            raise ValueError("base must be over 1, factor and original_positions positive, got "
                             f"{base}, {factor}, {original_positions}")
        base, factor = float(base), float(factor)
        if scaling == "ntk":
            if n == 2:
                raise ValueError("ntk scaling needs a rotary_dim over 2: a single pair does not depend on the base")
            base *= factor ** (n / (n - 2))
        freq = [base ** (-2.0 * i / n) for i in range(n // 2)]
        if scaling == "linear":
            return [f / factor for f in freq], 1.0
        if scaling == "wavelength":
            if not high_turns > low_turns:
                raise ValueError(f"high_turns must exceed low_turns, got {high_turns} and {low_turns}")
            keep = [min(1.0, max(0.0, (original_positions * f / (2.0 * math.pi) - low_turns) / (high_turns - low_turns)))
                    for f in freq]
            return [k * f + (1.0 - k) * f / factor for k, f in zip(keep, freq)], 1.0
        if scaling == "yarn":
            if not fast_turns > slow_turns > 0.0:
                raise ValueError(f"fast_turns must exceed slow_turns, both positive, got {fast_turns} and {slow_turns}")

            def index(turns):  # of the (real-valued) pair that makes so many turns in the original range
                return n * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

            low, high = max(math.floor(index(fast_turns)), 0), min(math.ceil(index(slow_turns)), n - 1)
            slow = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(n // 2)]
            return [f / factor * s + f * (1.0 - s) for s, f in zip(slow, freq)], 0.1 * math.log(max(factor, 1.0)) + 1.0
        return freq, 1.0

    @classmethod
    def create(cls, rotary_dim: int, *, interleaved: bool = False, amplitude: Optional[float] = None, device=None,
               **scaling) -> "RotaryFrequencies":
        """The table for ``rotary_dim`` columns; keywords as of :meth:`inverse_frequencies`.
        ``amplitude`` replaces the scaling's own."""
        freq, own = cls.inverse_frequencies(rotary_dim, **scaling)
        units = [round(f / (2.0 * math.pi) * 2.0 ** 64) % (1 << 64) for f in freq]
        turns = torch.tensor([u - (1 << 64) if u >= 1 << 63 else u for u in units], dtype=torch.int64, device=device)
        return cls(turns, own if amplitude is None else float(amplitude), bool(interleaved))


def _operand(name: str, t: Tensor, like: Tensor) -> Tensor:
    if t.dim() not in (3, 4):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] or [batch, tokens, heads, head_dim], "
                         f"got shape {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"rotary positions support float32 and bfloat16 tensors only, got {t.dtype}")
    if t is not like and (t.dtype != like.dtype or t.device != like.device or t.shape[:-2] != like.shape[:-2]
                          or t.shape[-1] != like.shape[-1]):
        raise ValueError(f"query and key must agree but for their heads, got {tuple(like.shape)} {like.dtype} on "
                         f"{like.device} and {tuple(t.shape)} {t.dtype} on {t.device}")
    return t


def _check(query: Tensor, key: Optional[Tensor], positions: Tensor, frequencies: RotaryFrequencies) -> Tensor:
    _operand("query", query, query)
    if key is not None:
        _operand("key", key, query)
    P._check_device_tensor("query", query)
    turns = frequencies.turns
    if turns.dtype != torch.int64 or turns.dim() != 1 or not turns.is_contiguous() or turns.device != query.device:
        raise ValueError("frequencies.turns must be a contiguous int64 vector on the query's device, got "
                         f"{tuple(turns.shape)} {turns.dtype} on {turns.device}")
    if not 1 <= turns.shape[0] <= query.shape[-1] // 2:
        raise ValueError(f"{turns.shape[0]} frequencies for a head_dim of {query.shape[-1]}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    lead = query.shape[:-2]
    try:
        return positions.to(query.device).expand(lead)
    except RuntimeError:
        raise ValueError(f"positions {tuple(positions.shape)} do not fit tokens {tuple(lead)}") from None


def _turn(query, key, positions, frequencies, inverse: bool, inplace: bool = False):
    """Checked operands -> turned query and key (None without one)."""
    if inplace:
        if key is not None and key.numel() > 0 and key.data_ptr() == query.data_ptr():
            raise ValueError("an in-place query and key need memory of their own: the same tensor would be turned twice")
        for name, t in (("query", query), ("key", key)):
            if t is not None and (t.stride(-1) != 1 or any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride()))):
                raise ValueError(f"an in-place {name} needs a unit head_dim stride and memory of its own for every row")
        q, k, qo, ko = query, key, query, key
    else:
        q, k = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (query, key))
        qo, ko = (None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key))
    four = lambda t: (0, *t.stride()[:2]) if t.dim() == 3 else t.stride()[:3]  # noqa: E731
    none = (0, 0, 0)
    pos = positions.stride()
    lead = query.shape[:-2]
    p = _capi.RotaryParams(
        q.data_ptr(), None if k is None else k.data_ptr(), qo.data_ptr(), None if ko is None else ko.data_ptr(),
        frequencies.turns.data_ptr(), positions.data_ptr(),
        *four(q), *(none if k is None else four(k)), *four(qo), *(none if ko is None else four(ko)),
        *((0, *pos) if len(lead) == 1 else pos),
        1 if len(lead) == 1 else lead[0], lead[-1], query.shape[-2], 0 if key is None else key.shape[-2], query.shape[-1],
        2 * frequencies.turns.shape[0], int(bool(frequencies.interleaved)), _DTYPES[query.dtype], int(inverse),
        int(positions.dtype == torch.int64), float(frequencies.amplitude))
    lib = _capi.load()
    with torch.cuda.device(query.device):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_rotary(ctypes.byref(p), P._stream(query.device)))
    for t in (query, key) if inplace else ():
        if t is not None and not t.is_inference():  # what autograd has saved of it is no longer what it was
            torch.autograd.graph.increment_version(t)
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, turns, amplitude, interleaved, inverse):
        ctx.save_for_backward(positions, turns)
        ctx.save_for_forward(positions, turns)
        ctx.meta = (amplitude, interleaved, inverse, key is not None)
        return _turn(query, key, positions, RotaryFrequencies(turns, amplitude, interleaved), inverse)

    @staticmethod
    def backward(ctx, dquery, dkey):
        positions, turns = ctx.saved_tensors
        amplitude, interleaved, inverse, has_key = ctx.meta
        # the inverse turn, itself differentiable
        dquery, dkey = _Rotary.apply(dquery, dkey if has_key else None, positions, turns, amplitude, interleaved, not inverse)
        return dquery, dkey, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tquery, tkey, *_):
        positions, turns = ctx.saved_tensors
        amplitude, interleaved, inverse, _ = ctx.meta
        # the turn is linear: a tangent turns like its tensor
        turned = iter(())
        given = [t for t in (tquery, tkey) if t is not None]
        if given:
            turned = iter(_Rotary.apply(given[0], given[1] if len(given) > 1 else None, positions, turns, amplitude, interleaved, inverse))
        return tuple(None if t is None else next(turned) for t in (tquery, tkey))


def _has_tangent(t: Optional[Tensor]) -> bool:
    return t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None


def rotary(query: Tensor, key: Optional[Tensor], positions: Tensor, frequencies: RotaryFrequencies, *,
           inverse: bool = False, inplace: bool = False):
    """Turn the pairs of ``query`` [..., tokens, Hq, D] and ``key`` [..., tokens, Hkv, D] (or None) by
    ``positions`` ([tokens] or [batch, tokens], or what broadcasts to them) times ``frequencies``.

    Returns ``(query, key)``, new tensors, or the given ones written in place (``inplace``; not
    for tensors that need a gradient, nor where an element to turn lies in both or twice in one).
    The first ``2 * len(frequencies.turns)`` columns of a head are turned, the others passed on.
    fp32 arithmetic, one rounding.  ``inverse`` turns the other way, which is also the gradient; in
    forward mode tangents are turned like their tensors.  Any strides with a unit one on head_dim are
    read in place, so that the heads of a fused projection need no copy.
    """
    if query.is_cuda:
        res = _capi.host().rotary(query, key, positions, *frequencies, inverse, inplace, P._stream(query.device))
        if res is not None:
            return res
    positions = _check(query, key, positions, frequencies)
    grad = torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))
    grad = grad or _has_tangent(query) or _has_tangent(key)
    if inplace:
        if grad:
            raise ValueError("an in-place rotary has no gradient: leave inplace off")
        return _turn(query, key, positions, frequencies, inverse, True)
    if grad:
        return _Rotary.apply(query, key, positions, frequencies.turns, frequencies.amplitude, frequencies.interleaved,
                             inverse)
    return _turn(query, key, positions, frequencies, inverse)


# ---------------------------------------------------------------- heads normed and turned

def _norm_weight(name: str, w: Optional[Tensor], like: Tensor) -> Optional[Tensor]:
    if w is None:
        return None
    if w.dtype not in (torch.float32, like.dtype):
        raise TypeError(f"{name} must be float32 or of the heads' type {like.dtype}, got {w.dtype}")
    if w.shape != like.shape[-1:] or w.device != like.device:
        raise ValueError(f"{name} must be [{like.shape[-1]}] on {like.device}, got {tuple(w.shape)} on {w.device}")
    return w.contiguous()


def _norm_params(query, key, positions, frequencies, query_weight, key_weight, eps, outputs, grads=(None, None)):
    """The C struct of checked operands with unit head_dim strides, their outputs and (backward) gradients."""
    weight = query_weight if query_weight is not None else key_weight
    lead = query.shape[:-2]
    four = lambda t: (0, 0, 0) if t is None else (0, *t.stride()[:2]) if t.dim() == 3 else t.stride()[:3]  # noqa: E731
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    pos = positions.stride()
    return _capi.NormRotaryParams(
        query.data_ptr(), ptr(key), *map(ptr, outputs), *map(ptr, grads), ptr(query_weight), ptr(key_weight), None, None,
        frequencies.turns.data_ptr(), positions.data_ptr(),
        *four(query), *four(key), *four(outputs[0]), *four(outputs[1]), *four(grads[0]), *four(grads[1]),
        *((0, *pos) if len(lead) == 1 else pos),
        1 if len(lead) == 1 else lead[0], lead[-1], query.shape[-2], 0 if key is None else key.shape[-2], query.shape[-1],
        2 * frequencies.turns.shape[0], int(bool(frequencies.interleaved)), _DTYPES[query.dtype],
        _DTYPES[query.dtype if weight is None else weight.dtype], int(positions.dtype == torch.int64),
        float(frequencies.amplitude), eps, None, 0)


def _launch_norm(entry: str, device, p) -> None:
    lib = _capi.load()
    with torch.cuda.device(device):
        _capi.raise_for_status(lib, getattr(lib, entry)(ctypes.byref(p), P._stream(device)))


def _unit(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.stride(-1) == 1 else t.contiguous()


def _norm_forward(query, key, positions, frequencies, query_weight, key_weight, eps):
    query, key = _unit(query), _unit(key)
    out = tuple(None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key))
    _launch_norm("mimir_prefixlm_norm_rotary", query.device,
                 _norm_params(query, key, positions, frequencies, query_weight, key_weight, eps, out))
    return out


def _gradient(t: Optional[Tensor]) -> Optional[Tensor]:
    """A head takes at most 64 lanes of 2 accesses, so past 128 columns they must be wide: a gradient, whose layout
    is not the caller's choice, is copied where its rows do not allow that."""
    if t is None:
        return None
    columns = 1
    while t.shape[-1] > 128 * columns:
        columns *= 2
    if t.stride(-1) != 1 or t.data_ptr() % (columns * t.element_size()) or any(
            n > 1 and s % columns for n, s in zip(t.shape[:-1], t.stride())):
        t = P._own_copy(t)
    return t


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, turns, amplitude, interleaved, eps):
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, turns)
        ctx.meta = (amplitude, interleaved, eps)
        return _norm_forward(query, key, positions, RotaryFrequencies(turns, amplitude, interleaved), query_weight, key_weight, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dquery, dkey):
        query, key, query_weight, key_weight, positions, turns = ctx.saved_tensors
        amplitude, interleaved, eps = ctx.meta
        query, key = _unit(query), _unit(key)
        dquery, dkey = _gradient(dquery), _gradient(dkey if key is not None else None)
        out = tuple(None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key))
        p = _norm_params(query, key, positions, RotaryFrequencies(turns, amplitude, interleaved), query_weight, key_weight, eps,
                         out, (dquery, dkey))
        weights = [torch.empty_like(w) if w is not None and needed else None
                   for w, needed in zip((query_weight, key_weight), ctx.needs_input_grad[2:4])]
        p.dq_weight, p.dk_weight = (None if w is None else w.data_ptr() for w in weights)
        p.workspace_bytes = _capi.load().mimir_prefixlm_norm_rotary_workspace_bytes(ctypes.byref(p))
        workspace = torch.empty(p.workspace_bytes // 4, dtype=torch.float32, device=query.device)
        p.workspace = workspace.data_ptr()
        _launch_norm("mimir_prefixlm_norm_rotary_bwd", query.device, p)
        return (*out, *weights, None, None, None, None, None)


def norm_rotary(query: Tensor, key: Optional[Tensor], positions: Tensor, frequencies: RotaryFrequencies,
                query_weight: Optional[Tensor] = None, key_weight: Optional[Tensor] = None, *, eps: float = 1e-6):
    """Norm each head of ``query`` [..., tokens, Hq, D] and ``key`` [..., tokens, Hkv, D] (or None) by its root
    mean square, scale it by a learned weight [D] (or None) and turn it as :func:`rotary` does, in one pass:
    ``turn(x / sqrt(mean(x^2) + eps) * weight)`` with the mean over all of the head.

    Returns ``(query, key)``, new tensors; gradients for the heads and the weights, which are float32 or of the
    heads' type, both the same.  fp32 arithmetic, one rounding; the weights' gradients are summed in a fixed order,
    across workgroups in 64 bits.  Positions, frequencies and strides as for :func:`rotary`.
    """
    if query.is_cuda:
        res = _capi.host().norm_rotary(query, key, positions, *frequencies, query_weight, key_weight, eps, P._stream(query.device))
        if res is not None:
            return res
    positions = _check(query, key, positions, frequencies)
    if query.shape[-1] % 2:
        raise ValueError(f"head_dim must be even, got {query.shape[-1]}")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if key is None and key_weight is not None:
        raise ValueError("a key_weight needs a key")
    if query_weight is not None and key_weight is not None and query_weight.dtype != key_weight.dtype:
        raise TypeError(f"query_weight and key_weight must be of one type, got {query_weight.dtype} and {key_weight.dtype}")
    query_weight, key_weight = _norm_weight("query_weight", query_weight, query), _norm_weight("key_weight", key_weight, query)
    given = (query, key, query_weight, key_weight)
    if any(map(_has_tangent, given)):
        raise NotImplementedError("norm_rotary has no forward-mode derivative")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
        return _NormRotary.apply(*given, positions, frequencies.turns, frequencies.amplitude, frequencies.interleaved, eps)
    return _norm_forward(query, key, positions, frequencies, query_weight, key_weight, eps)
