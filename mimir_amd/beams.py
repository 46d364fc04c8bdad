"""Beam search on the device: the best continuations, and the caches' rows in their order.

* :func:`select_beams`: of each request's beams and the vocabulary, the continuations with the
  highest summed log-probability, from the logits as the model leaves them.
* :func:`reorder_rows`: rows of static caches (:class:`mimir_amd.cache.Cache`, all layers in one call) take
  the state of the chosen beams, in place.  Paged caches do that without copying whole rows:
  ``mimir_amd.paged.fork_rows(cache, table, selection.rows.flatten(), all_rows)``.

A request's ``W`` beams are neighbouring rows of the batch, row ``r * W + w``.  Both calls only enqueue work on
the current stream, so a step of beam search can be captured in a HIP graph.  No CPU fallback.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Sequence, Union

import torch
from torch import Tensor

from . import _capi
from . import prefixlm as P
from .cache import Cache

MAX_BEAMS = 32
MAX_COUNT = 64
_DTYPES = {torch.float32: _capi.DTYPE_FLOAT32, torch.bfloat16: _capi.DTYPE_BFLOAT16}


class BeamSelection(NamedTuple):
    """Best first.  ``rows`` are rows of the batch (request * W + beam): what :func:`reorder_rows` and
    ``mimir_amd.paged.fork_rows`` take as sources."""
    scores: Tensor              # float32 [requests, count]
    tokens: Tensor              # int32 [requests, count]
    rows: Tensor                # int32 [requests, count]
    finished: Optional[Tensor]  # bool [requests, count]; None without an end_token


def select_beams(logits: Tensor, scores: Tensor, count: Optional[int] = None, *, finished: Optional[Tensor] = None,
                 end_token: Optional[int] = None) -> BeamSelection:
    """The ``count`` (default: W) best continuations of each request by
    ``scores[r, w] + log_softmax(logits[r, w])[token]``, ties to the lowest beam, then token.

    ``logits`` [requests, W, vocab] bfloat16 or float32, ``scores`` float32 [requests, W] (-inf for a beam that is not
    in use, as all but the first at the first step).  A beam that is ``finished`` (bool [requests, W]) goes on with
    ``end_token`` alone, at its score, and its logits are not read.  Tokens with logit -inf are never chosen, nor is
    a beam whose logits hold NaN or +inf; where fewer than ``count`` continuations are left, the rest have score -inf.
    Sums of exponentials are fp32, the rest is 64 bits and rounded once: a beam's scores are all off by the same,
    less than 2^-19, so beams whose scores lie closer than twice that may change places.  Not differentiable.  W up to 32, ``count`` up to 64.
    """
    if logits.is_cuda and logits.dim() == 3:
        end = -1 if end_token is None else None if end_token == -1 else end_token  # (a given -1 is refused below)
        out = _capi.host().select(logits, scores, logits.shape[1] if count is None else count, finished, end, P._stream(logits.device))
        if out is not None:
            return BeamSelection(*out)
    if logits.dim() != 3:
        raise ValueError(f"logits must be [requests, beams, vocab], got shape {tuple(logits.shape)}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"beam selection supports float32 and bfloat16 logits only, got {logits.dtype}")
    P._check_device_tensor("logits", logits)
    requests, beams, vocab = logits.shape
    count = beams if count is None else int(count)
    if not 1 <= beams <= MAX_BEAMS or not 1 <= count <= min(MAX_COUNT, beams * vocab):
        raise ValueError(f"count {count} of {beams} beams and {vocab} tokens: at most {MAX_BEAMS} beams and a count from 1 to {MAX_COUNT}")
    if scores.dtype != torch.float32 or scores.shape != (requests, beams) or scores.device != logits.device:
        raise ValueError(f"scores must be float32 [{requests}, {beams}] on {logits.device}, got {tuple(scores.shape)} {scores.dtype} on "
                         f"{scores.device}")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != (requests, beams) or finished.device != logits.device:
            raise ValueError(f"finished must be bool [{requests}, {beams}] on {logits.device}, got {tuple(finished.shape)} {finished.dtype} on "
                             f"{finished.device}")
        if end_token is None:
            raise ValueError("finished beams need an end_token")
    if end_token is not None and not 0 <= int(end_token) < vocab:
        raise ValueError(f"end_token {end_token} is not one of {vocab} tokens")
    if logits.stride(-1) != 1 and vocab > 1:
        logits = logits.contiguous()
    device = logits.device
    out = BeamSelection(torch.empty((requests, count), dtype=torch.float32, device=device),
                        torch.empty((requests, count), dtype=torch.int32, device=device),
                        torch.empty((requests, count), dtype=torch.int32, device=device),
                        None if end_token is None else torch.empty((requests, count), dtype=torch.bool, device=device))
    p = _capi.BeamSelectParams(
        logits.data_ptr(), scores.data_ptr(), None if finished is None else finished.data_ptr(),
        out.scores.data_ptr(), out.tokens.data_ptr(), out.rows.data_ptr(), None if out.finished is None else out.finished.data_ptr(),
        *logits.stride()[:2], *scores.stride(), *((0, 0) if finished is None else finished.stride()),
        requests, beams, vocab, count, -1 if end_token is None else int(end_token), _DTYPES[logits.dtype], None, 0)
    lib = _capi.load()
    p.workspace_bytes = lib.mimir_prefixlm_beam_select_workspace_bytes(ctypes.byref(p))
    workspace = torch.empty(max(p.workspace_bytes, 16), dtype=torch.uint8, device=device)
    p.workspace = workspace.data_ptr()
    with torch.cuda.device(device):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_beam_select(ctypes.byref(p), P._stream(device)))
    return out


def _cache_rows(name: str, t: Tensor, like: Tensor) -> None:
    if t.dim() < 2 or t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"all caches must be alike, [rows, positions, ...] of one type on one device, got {tuple(like.shape)} {like.dtype} "
                         f"on {like.device} and {name} {tuple(t.shape)} {t.dtype} on {t.device}")
    row = t[0:1]
    if (t.shape[0] > 0 and not row.is_contiguous()) or (t.shape[0] > 1 and t.stride(0) < row.numel()):
        raise ValueError(f"the rows of {name} must be contiguous and apart")


def _check_all(tensors, rows: int) -> None:
    """What one launch refuses of its tensors, for all of several: nothing runs before a refusal."""
    spans = []
    for t in tensors:
        row, step = t[0].numel() * t.element_size(), t.stride(0) * t.element_size()
        if t.data_ptr() % 16 or step % 16:
            raise ValueError("cache rows must be aligned to 16 bytes")
        spans.append((t.data_ptr(), row, step))
    spans.sort()
    for i, (a, row, step) in enumerate(spans):
        for b, _, other in spans[i + 1:]:
            if b >= a + (rows - 1) * step + row:
                break
            # rows of equal stride: the one at or before the other's first, and the next
            at, off = divmod(b - a, step)
            if step != other or off < row or (step - off < row and at + 1 < rows):
                raise ValueError("cache tensors must not share memory, and lie in each other's gaps with one stride only")


def reorder_rows(caches: Union[Cache, Sequence[Cache]], lengths: Tensor, source: Tensor) -> None:
    """Give row ``i`` of every cache the state of row ``source.flatten()[i]``, in place, as all were before the call:
    the first ``lengths[source[i]]`` positions of its keys and values, and in ``lengths`` (int32 or int64) its length.

    ``source`` int32 or int64 [requests, W] holds rows of the batch, each from its own request's W rows (as
    ``BeamSelection.rows`` with a count of W); a row whose source lies elsewhere stays as it is (with
    ``mimir_amd.set_validate_metadata(True)``: IndexError).  Rows that stay and positions past a length are not
    touched.  ``lengths`` has one entry per row of ``source``; caches may have more rows.  W up to 32.
    """
    caches = [caches] if isinstance(caches, Cache) else list(caches)
    if lengths.is_cuda and not P._validate_metadata and _capi.host().reorder(caches, lengths, source, P._stream(lengths.device)):
        return
    if source.dim() != 2 or source.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"source must be int32 or int64 [requests, beams], got {tuple(source.shape)} {source.dtype}")
    rows, group = source.numel(), source.shape[1]
    if not 1 <= group <= MAX_BEAMS:
        raise ValueError(f"1 to {MAX_BEAMS} beams a request, got {group}")
    if lengths.shape != (rows,) or lengths.dtype not in (torch.int32, torch.int64) or (rows > 1 and lengths.stride(0) != 1):
        raise ValueError(f"lengths must be a contiguous int32 or int64 [{rows}], got {tuple(lengths.shape)} {lengths.dtype}")
    P._check_device_tensor("lengths", lengths)
    tensors = [t for c in caches for t in (c.keys, c.values)]
    for i, t in enumerate(tensors):
        _cache_rows(f"cache {i // 2}", t, tensors[0])
    if tensors and (tensors[0].device != lengths.device or tensors[0].shape[0] < rows):
        raise ValueError(f"caches of {tensors[0].shape[0]} rows on {tensors[0].device} for {rows} rows on {lengths.device}")
    source = source.to(lengths.device).contiguous()
    if P._validate_metadata and rows:
        start = torch.arange(0, rows, group, device=source.device)[:, None]
        if bool(((source < start) | (source >= start + group)).any()):
            raise IndexError("a source row lies outside its request's rows")
    p = _capi.ReorderParams()
    p.lengths, p.source = lengths.data_ptr(), source.data_ptr()
    p.position_bytes, p.max_length = 16, 0
    if tensors:
        t = tensors[0]
        p.max_length = t.shape[1]
        p.position_bytes = t.element_size()
        for n in t.shape[2:]:
            p.position_bytes *= n
    p.rows, p.group = rows, group
    p.index_int64, p.source_int64 = int(lengths.dtype == torch.int64), int(source.dtype == torch.int64)
    lib = _capi.load()
    step = _capi.REORDER_TENSORS
    if len(tensors) > step and rows > 0 and tensors[0].shape[1] > 0:
        _check_all(tensors, rows)
    with torch.cuda.device(lengths.device):
        for i in range(0, max(len(tensors), 1), step):
            part = tensors[i:i + step]
            p.count, p.update_lengths = len(part), int(i + step >= len(tensors))
            for j, t in enumerate(part):
                p.data[j], p.stride[j] = t.data_ptr(), t.stride(0) * t.element_size() if rows > 1 else 0
            _capi.raise_for_status(lib, lib.mimir_prefixlm_reorder_rows(ctypes.byref(p), P._stream(lengths.device)))
    for t in (*tensors, lengths):
        if not t.is_inference():  # what autograd has saved of it is no longer what it was
            torch.autograd.graph.increment_version(t)
