"""Attention to states of another length: cross attention, for training and for serving.

``flash_attn_varlen_prefixlm`` attends a sequence's own tokens.  Here the queries attend another set of
states (an encoder's, another document's), each sequence with lengths of its own and every query seeing
all of its sequence's states:

* :func:`cross_attention`: packed queries over packed states, with gradients;
* :func:`attention_to_states`: the decode step, few queries per request over rows of a static cache of states
  (:class:`mimir_amd.cache.Cache`), a request's beams sharing one reading of them.

bf16, head_dim 64 or 128, grouped heads read in place; every call only enqueues work on the current stream and can
be captured in a HIP graph.  There is no CPU fallback.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
from torch import Tensor

from . import _capi
from . import prefixlm as P
from .cache import Cache


_MAX_STRIDE = 1 << 22  # elements: the kernels address a tile's 128 rows in 31 bits


def _rows(t: Tensor) -> Tensor:
    """Rows of tokens as the kernels read them; copied where they lie otherwise, or too far apart (the last tokens of long
    sequences, one of each)."""
    t = P._kernel_layout(t)
    return t if t.stride(0) < _MAX_STRIDE else P._own_copy(t)


def _scale(softmax_scale: Optional[float], d: int) -> float:
    return 1.0 / math.sqrt(max(d, 1)) if softmax_scale is None else float(softmax_scale)


def _check_heads(query: Tensor, key: Tensor, value: Tensor, tail: int) -> None:
    """dtypes, devices and the [.., heads, head_dim] tails."""
    if query.dtype != torch.bfloat16 or key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError(f"cross attention supports bfloat16 tensors only, got {query.dtype}, {key.dtype} and {value.dtype}")
    if key.shape != value.shape or key.shape[-1] != query.shape[-1]:
        raise ValueError(f"incompatible query / key / value shapes {tuple(query.shape)}, {tuple(key.shape)}, {tuple(value.shape)}")
    if query.shape[-2] == 0 or key.shape[-2] == 0 or query.shape[-2] % key.shape[-2]:
        raise ValueError(f"Query heads {query.shape[-2]} must be divisible by key/value heads {key.shape[-2]}.")
    P._check_device_tensor("query", query)
    if key.device != query.device or value.device != query.device:
        raise ValueError(f"query, key and value must be on one device, got {query.device}, {key.device} and {value.device}")


# ---------------------------------------------------------------- packed sequences

def _params(query, key, value, out, out_lo, lse2, cu_q, cu_k, scale, backward=(None, None, None, None)):
    p = _capi.CrossParams()
    p.q, p.k, p.v, p.out, p.out_lo, p.lse2 = (None if t is None else t.data_ptr() for t in (query, key, value, out, out_lo, lse2))
    p.cu_seqlens_q, p.cu_seqlens_k = cu_q.data_ptr(), cu_k.data_ptr()
    for name, t in zip(("q", "k", "v", "out", "dout", "dq", "dk", "dv"), (query, key, value, out, *backward)):
        if t is not None:
            setattr(p, name, t.data_ptr())
            setattr(p, name + "_stride_token", max(t.stride(0), t.shape[2]))  # (of a single row it may be anything)
            setattr(p, name + "_stride_head", t.stride(1) if t.shape[1] > 1 else 0)
    p.total_q, p.num_q_heads, p.head_dim = query.shape
    p.total_k, p.num_kv_heads = key.shape[:2]
    p.numseqs = cu_q.shape[0] - 1
    p.dtype, p.softmax_scale = _capi.DTYPE_BFLOAT16, scale
    return p


def _launch(entry: str, p, backward: bool, device) -> None:
    lib = _capi.load()
    p.workspace_bytes = lib.mimir_prefixlm_cross_workspace_bytes(ctypes.byref(p), int(backward))
    workspace = torch.empty(p.workspace_bytes, dtype=torch.uint8, device=device)
    p.workspace = workspace.data_ptr()
    with torch.cuda.device(device):
        _capi.raise_for_status(lib, getattr(lib, entry)(ctypes.byref(p), P._stream(device)))


def _forward(query, key, value, cu_q, cu_k, scale, keep: bool):
    query, key, value = map(_rows, (query, key, value))
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    out_lo = torch.empty_like(out) if keep else None
    lse2 = torch.empty((query.shape[1], query.shape[0]), dtype=torch.float32, device=query.device) if keep else None
    _launch("mimir_prefixlm_cross_fwd", _params(query, key, value, out, out_lo, lse2, cu_q, cu_k, scale), False, query.device)
    return out, out_lo, lse2


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, cu_q, cu_k, scale):
        out, out_lo, lse2 = _forward(query, key, value, cu_q, cu_k, scale, True)
        ctx.save_for_backward(query, key, value, out, out_lo, lse2, cu_q, cu_k)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        query, key, value, out, out_lo, lse2, cu_q, cu_k = ctx.saved_tensors
        query, key, value, dout = map(_rows, (query, key, value, dout))
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (query, key, value)]
        _launch("mimir_prefixlm_cross_bwd", _params(query, key, value, out, out_lo, lse2, cu_q, cu_k, ctx.scale, (dout, *grads)), True,
                query.device)
        return (*grads, None, None, None)


def _lengths_list(name: str, t: Tensor, device, total: int) -> Tensor:
    if t.dim() != 1 or t.shape[0] < 1 or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be a vector of int32 or int64, one longer than there are sequences, got {tuple(t.shape)} {t.dtype}")
    if P._validate_metadata:
        steps = t.tolist()
        if steps[0] < 0 or steps[-1] > total or any(b < a for a, b in zip(steps, steps[1:])):
            raise ValueError(f"{name} must not decrease and stay within [0, {total}], got {steps}")
    return t.to(device=device, dtype=torch.int32).contiguous()


def cross_attention(query: Tensor, key: Tensor, value: Tensor, cu_seqlens_q: Tensor, cu_seqlens_k: Tensor, *,
                    softmax_scale: Optional[float] = None) -> Tensor:
    """Queries [total_q, Hq, D] over states key / value [total_k, Hkv, D]: those of sequence s, rows ``cu_seqlens_q[s]``
    up to ``cu_seqlens_q[s + 1]``, attend rows ``cu_seqlens_k[s]`` up to ``cu_seqlens_k[s + 1]``, all of them.

    Returns [total_q, Hq, D], with gradients for query, key and value.  A sequence may have no queries or no states
    (its output is then 0); rows before the first or behind the last sequence give 0 and get zero gradients.  Both lists
    (int32 or int64 [numseqs + 1]) must not decrease and stay within the rows there are (checked with
    ``mimir_amd.set_validate_metadata(True)``).  The backward computes all three gradients, whichever are needed.  ``softmax_scale``
    is positive, 1 / sqrt(D) by default.  P and dS are rounded to bf16 for their products, sums are fp32; results do not
    depend on timing.  For the backward the output's low half is kept (bf16, as large as the output): the sums
    rowsum(dO * O) that dS is the difference to would carry the output's rounding without it.
    """
    if query.is_cuda and query.dim() == 3 and not P._validate_metadata:
        out = _capi.host().cross_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, _scale(softmax_scale, query.shape[2]),
                                           P._stream(query.device))
        if out is not None:
            return out
    if query.dim() != 3 or key.dim() != 3 or value.dim() != 3:
        raise ValueError("query, key and value must be [tokens, heads, head_dim]")
    _check_heads(query, key, value, 3)
    cu_q = _lengths_list("cu_seqlens_q", cu_seqlens_q, query.device, query.shape[0])
    cu_k = _lengths_list("cu_seqlens_k", cu_seqlens_k, query.device, key.shape[0])
    if cu_q.shape != cu_k.shape:
        raise ValueError(f"cu_seqlens_q and cu_seqlens_k are of {cu_q.shape[0] - 1} and {cu_k.shape[0] - 1} sequences")
    scale = _scale(softmax_scale, query.shape[2])
    if any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in (query, key, value)):
        raise NotImplementedError("cross_attention has no forward-mode derivative")
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        return _CrossAttention.apply(query, key, value, cu_q, cu_k, scale)
    return _forward(query, key, value, cu_q, cu_k, scale, False)[0]


# ---------------------------------------------------------------- rows of a cache of states

def attention_to_states(query: Tensor, states: Cache, state_lengths: Tensor, state_rows: Optional[Tensor] = None, *,
                        softmax_scale: Optional[float] = None) -> Tensor:
    """Queries [B, S, Hq, D] over rows of ``states`` (keys / values [rows, positions, Hkv, D]), of which row r holds
    ``state_lengths[r]`` (int32 or int64 [rows], clamped to the positions there are).

    ``state_rows`` (int32 or int64 [requests]; default: row i of the cache for request i) names each request's row.
    B is a multiple of the number of requests: each has B / requests neighbouring batch rows (its beams or samples),
    and every query sees all states of its request.  A request whose row lies outside the cache, or is empty, gets 0 (with
    ``mimir_amd.set_validate_metadata(True)`` the first is an IndexError).  Returns [B, S, Hq, D]; not differentiable.
    """
    if query.is_cuda and query.dim() == 4 and not P._validate_metadata:
        out = _capi.host().states(query, *states, state_lengths, state_rows, _scale(softmax_scale, query.shape[3]), P._stream(query.device))
        if out is not None:
            return out
    if query.dim() != 4 or states.keys.dim() != 4 or states.values.dim() != 4:
        raise ValueError("query must be [batch, tokens, heads, head_dim], states [rows, positions, heads, head_dim]")
    _check_heads(query, states.keys, states.values, 4)
    B, S, hq, d = query.shape
    pool, length, hkv, _ = states.keys.shape
    if torch.is_grad_enabled() and (query.requires_grad or states.keys.requires_grad or states.values.requires_grad):
        raise ValueError("attention_to_states has no gradient: use cross_attention")
    for name, t, n in (("state_lengths", state_lengths, pool), ("state_rows", state_rows, None)):
        if t is not None and (t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or t.device != query.device
                              or (n is not None and t.shape[0] != n)):
            raise ValueError(f"{name} must be int32 or int64 [{'requests' if n is None else n}] on {query.device}, got {tuple(t.shape)} {t.dtype} "
                             f"on {t.device}")
    requests = pool if state_rows is None else state_rows.shape[0]
    if (B > 0 and requests == 0) or (requests and B % requests):
        raise ValueError(f"a batch of {B} rows for {requests} requests")
    for name, t in (("keys", states.keys), ("values", states.values)):
        if t.stride(-1) != 1 or t.data_ptr() % 16 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in range(3)):
            raise ValueError(f"the cached {name} need a unit head_dim stride and 16-byte aligned rows")
        if length > 1 and t.stride(1) < d:
            raise ValueError(f"the cached {name} need a position stride of at least head_dim, got {t.stride(1)}")
    if P._validate_metadata and state_rows is not None and requests:
        if bool(((state_rows < 0) | (state_rows >= pool)).any()):
            raise IndexError(f"state_rows must lie in [0, {pool})")
    out = torch.empty((B, S, hq, d), dtype=query.dtype, device=query.device)
    if B == 0 or S == 0:
        return out
    # all tokens of a request in a row: [B * S, Hq, D], a token's heads no nearer than the head_dim (one expanded to many is copied)
    # and no further than the kernels reach
    token = query.stride(1 if S > 1 else 0)
    if query.stride(-1) != 1 or query.data_ptr() % 16 or (B > 1 and S > 1 and query.stride(0) != S * token) or (B * S > 1 and not d <= token < _MAX_STRIDE) or any(
            query.shape[i] > 1 and query.stride(i) % 8 for i in range(3)):
        query = P._own_copy(query)
    state_lengths = state_lengths.contiguous()
    state_rows = None if state_rows is None else state_rows.contiguous()
    step = lambda t, i, least=0: max(t.stride(i), least) if t.shape[i] > 1 else least  # noqa: E731
    q_token = max(query.stride(1 if S > 1 else 0), d) if B * S > 1 else d
    p = _capi.StatesParams(
        query.data_ptr(), states.keys.data_ptr(), states.values.data_ptr(), out.data_ptr(), state_lengths.data_ptr(),
        None if state_rows is None else state_rows.data_ptr(), q_token, step(query, 2),
        *(x for t in states[:2] for x in (step(t, 0), step(t, 1, d), step(t, 2))), hq * d, d,
        requests, B // requests * S, pool, length, hq, hkv, d, _capi.DTYPE_BFLOAT16, int(state_lengths.dtype == torch.int64),
        int(state_rows is not None and state_rows.dtype == torch.int64), _scale(softmax_scale, d), None, 0)
    lib = _capi.load()
    p.workspace_bytes = lib.mimir_prefixlm_states_workspace_bytes(ctypes.byref(p))
    workspace = torch.empty(p.workspace_bytes, dtype=torch.uint8, device=query.device)
    p.workspace = workspace.data_ptr()
    with torch.cuda.device(query.device):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_states_attn(ctypes.byref(p), P._stream(query.device)))
    return out
