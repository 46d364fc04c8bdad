"""Cross attention without a GPU: the oracle's gradients against differences, and the refusals of the C ABI."""

import ctypes

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.cache import Cache
from mimir_amd.cross import attention_to_states, cross_attention
from oracle import generation_oracle as O


def test_oracle_gradients_against_differences():
    gen = torch.Generator().manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    q, k, v, do = rand(6, 4, 3), rand(7, 2, 3), rand(7, 2, 3), rand(6, 4, 3)
    args = ([0, 2, 2, 5], [1, 4, 4, 6], 0.7)
    f = lambda q, k, v: (O.cross_attention(q, k, v, *args)[0][0] * do).sum()  # noqa: E731
    grads = [g for g, _ in O.cross_attention(q, k, v, *args, do)[1:]]
    h = 1e-6  # of smooth functions of order 1: h^2 and 2^-53 / h are both below 1e-9
    for i, (t, grad) in enumerate(zip((q, k, v), grads)):
        for at in range(t.numel()):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[at] = h
            up, down = ([x + s * step.view(x.shape) if j == i else x for j, x in enumerate((q, k, v))] for s in (1.0, -1.0))
            assert abs((f(*up) - f(*down)) / (2 * h) - grad.flatten()[at]) < 1e-7


def test_cpu_tensors_are_refused():
    x, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4])
    with pytest.raises(RuntimeError, match="ROCm"):
        cross_attention(x, x, x, cu, cu)
    with pytest.raises(RuntimeError, match="ROCm"):
        attention_to_states(x[None], Cache(x[None], x[None]), torch.tensor([4]))


def _cross(**kw):
    p = _capi.CrossParams()
    values = dict(q=4096, k=8192, v=12288, out=16384, out_lo=4096, lse2=4096, cu_seqlens_q=64, cu_seqlens_k=64, dout=4096, dq=4096, dk=4096, dv=4096, total_q=4, total_k=5,
                  numseqs=1, num_q_heads=2, num_kv_heads=1, head_dim=64, dtype=_capi.DTYPE_BFLOAT16, softmax_scale=0.125, workspace=256, workspace_bytes=1 << 20)
    for t in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        values[t + "_stride_token"], values[t + "_stride_head"] = 128, 64
    for name, value in {**values, **kw}.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("kw,error", [
    (dict(dtype=0), TypeError), (dict(head_dim=96), ValueError), (dict(num_q_heads=3, num_kv_heads=2), ValueError), (dict(num_kv_heads=0), ValueError),
    (dict(total_q=-1), ValueError), (dict(numseqs=-1), ValueError), (dict(softmax_scale=0.0), ValueError), (dict(softmax_scale=float("nan")), ValueError),
    (dict(q=None), ValueError), (dict(k=8200), ValueError), (dict(v_stride_token=132), ValueError), (dict(q_stride_token=32), ValueError),
    (dict(k_stride_token=1 << 22), ValueError), (dict(out_stride_head=-64), ValueError), (dict(cu_seqlens_k=None), ValueError),
    (dict(total_q=0x40000000), ValueError), (dict(workspace=None), ValueError), (dict(workspace=264), ValueError), (dict(workspace_bytes=31), ValueError)])
def test_c_cross_refusals(kw, error, backward):
    lib = _capi.load()
    entry = lib.mimir_prefixlm_cross_bwd if backward else lib.mimir_prefixlm_cross_fwd
    with pytest.raises(error):
        _capi.raise_for_status(lib, entry(ctypes.byref(_cross(**kw)), None))


@pytest.mark.parametrize("kw", [dict(lse2=None), dict(out_lo=None), dict(out_lo=4104), dict(dout=None), dict(dv=None), dict(dk=4104)])
def test_c_backward_refusals(kw):
    lib = _capi.load()
    with pytest.raises(ValueError):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_cross_bwd(ctypes.byref(_cross(**kw)), None))


@pytest.mark.parametrize("backward,kw", [(False, dict(total_q=1, numseqs=1 << 24)), (False, dict(total_q=0x3fffffff, numseqs=1 << 23)),
                                         (True, dict(total_q=0, numseqs=1 << 23)), (True, dict(numseqs=0x7fffffff))])
def test_c_launches_of_2_to_the_32_threads_are_refused(backward, kw):
    lib = _capi.load()
    p = _cross(**{**kw, "workspace_bytes": 1 << 40})
    with pytest.raises(ValueError, match="too many"):
        _capi.raise_for_status(lib, (lib.mimir_prefixlm_cross_bwd if backward else lib.mimir_prefixlm_cross_fwd)(ctypes.byref(p), None))


def test_c_states_launches_of_2_to_the_32_threads_are_refused():
    lib = _capi.load()
    p = _states(requests=1 << 23, seq_tokens=130, num_q_heads=1, workspace_bytes=1 << 40)
    with pytest.raises(ValueError, match="too many"):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_states_attn(ctypes.byref(p), None))


def test_cross_workspace():
    lib = _capi.load()
    size = lambda b, **kw: lib.mimir_prefixlm_cross_workspace_bytes(ctypes.byref(_cross(**kw)), b)  # noqa: E731
    # lists of ceil(total / 128) + numseqs entries of 16 bytes, and (backward) fp32 [Hq, total_q], in steps of 256 bytes
    assert size(0, total_q=1000, numseqs=3) == 256
    assert size(0, total_q=20000, numseqs=30) == (157 + 30) * 16 + 80  # rounded up to 256
    assert size(1, total_q=1000, total_k=20000, numseqs=3) == 256 + 2560 + 2 * 1000 * 4 + 192
    assert size(1, total_q=0, total_k=0) == 0


def _states(**kw):
    p = _capi.StatesParams()
    values = dict(q=4096, keys=4096, values=4096, out=4096, lengths=64, rows=64, q_stride_token=128, q_stride_head=64, k_stride_row=1280, k_stride_token=128,
                  k_stride_head=64, v_stride_row=1280, v_stride_token=128, v_stride_head=64, out_stride_token=128, out_stride_head=64, requests=2, seq_tokens=3,
                  cache_rows=4, cache_len=10, num_q_heads=2, num_kv_heads=1, head_dim=64, dtype=_capi.DTYPE_BFLOAT16, softmax_scale=0.125, workspace=256,
                  workspace_bytes=1 << 24)
    for name, value in {**values, **kw}.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("kw,error", [
    (dict(dtype=0), TypeError), (dict(head_dim=32), ValueError), (dict(num_q_heads=3, num_kv_heads=2), ValueError), (dict(num_q_heads=0), ValueError),
    (dict(requests=-1), ValueError), (dict(cache_len=-1), ValueError), (dict(softmax_scale=-1.0), ValueError), (dict(q=None), ValueError),
    (dict(lengths=None), ValueError), (dict(values=None), ValueError), (dict(keys=4104), ValueError), (dict(k_stride_token=60), ValueError),
    (dict(k_stride_token=56), ValueError), (dict(v_stride_row=-1280), ValueError), (dict(out_stride_token=1 << 22), ValueError),
    (dict(requests=0x7fffffff), ValueError), (dict(workspace=None), ValueError), (dict(workspace=128), ValueError), (dict(workspace_bytes=100), ValueError)])
def test_c_states_refusals(kw, error):
    lib = _capi.load()
    with pytest.raises(error):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_states_attn(ctypes.byref(_states(**kw)), None))


def test_calls_without_work():
    lib = _capi.load()
    assert lib.mimir_prefixlm_cross_fwd(ctypes.byref(_cross(total_q=0, q=None)), None) == _capi.OK
    assert lib.mimir_prefixlm_cross_bwd(ctypes.byref(_cross(total_q=0, total_k=0)), None) == _capi.OK
    assert lib.mimir_prefixlm_states_attn(ctypes.byref(_states(requests=0)), None) == _capi.OK


def test_structs_match_the_header():
    from tests.test_capi import _c_layout

    for cls, name in ((_capi.CrossParams, "MimirCrossParams"), (_capi.StatesParams, "MimirStatesParams")):
        fields = [f[0] for f in cls._fields_]
        size, offsets = _c_layout(name, fields)
        assert ctypes.sizeof(cls) == size
        assert [getattr(cls, f).offset for f in fields] == offsets
