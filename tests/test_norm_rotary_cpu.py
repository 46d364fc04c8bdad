"""norm_rotary without a GPU: the oracle's gradient against differences, and the refusals."""

import ctypes

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.rotary import RotaryFrequencies, norm_rotary
from oracle import generation_oracle as O


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rd", [8, 4])
def test_oracle_gradient_against_differences(interleaved, rd):
    gen = torch.Generator().manual_seed(rd)
    x, dy = (torch.randn(3, 2, 8, generator=gen, dtype=torch.float64) for _ in range(2))
    w = torch.rand(8, generator=gen, dtype=torch.float64) + 0.5
    args = (torch.tensor([0, 5, 900]), [1.0, 0.3, 0.1, 0.01][:rd // 2], 1.25, interleaved, 1e-3)
    f = lambda x, w: (O.norm_rotary(x, w, *args)[0] * dy).sum()  # noqa: E731
    (dx, _), (dw, _) = O.norm_rotary_grad(dy, x, w, *args)
    h = 1e-6  # of a smooth function of order 1: h^2 and 2^-53 / h are both below 1e-9
    for t, grad in ((x, dx), (w, dw)):
        for i in range(t.numel()):
            step = torch.zeros(t.numel(), dtype=torch.float64)
            step[i] = h
            step = step.view(t.shape)
            up, down = ((f(x + s * step, w) if t is x else f(x, w + s * step)) for s in (1.0, -1.0))
            assert abs((up - down) / (2 * h) - grad.flatten()[i]) < 1e-7


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm"):
        norm_rotary(torch.zeros(3, 2, 8), None, torch.arange(3), RotaryFrequencies.create(8, device="cpu"))


def _params(**kw):
    p = _capi.NormRotaryParams()
    values = dict(q=4096, q_out=8192, dq=12288, turns=64, positions=64, batch=1, seqlen=1, num_q_heads=1, num_kv_heads=0, head_dim=64,
                  rotary_dim=64, dtype=_capi.DTYPE_FLOAT32, weight_dtype=_capi.DTYPE_FLOAT32, amplitude=1.0, eps=1e-6,
                  q_stride_token=64, q_stride_head=64, q_out_stride_token=64, q_out_stride_head=64, dq_stride_token=64, dq_stride_head=64)
    for name, value in {**values, **kw}.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("kw,error", [
    (dict(dtype=7), TypeError), (dict(dtype=_capi.DTYPE_FLOAT32, weight_dtype=_capi.DTYPE_BFLOAT16), TypeError),
    (dict(batch=-1), ValueError), (dict(num_q_heads=0), ValueError), (dict(head_dim=63), ValueError), (dict(rotary_dim=66), ValueError),
    (dict(rotary_dim=3), ValueError), (dict(eps=-1.0), ValueError), (dict(eps=float("inf")), ValueError), (dict(amplitude=float("nan")), ValueError),
    (dict(q=None), ValueError), (dict(turns=None), ValueError), (dict(num_kv_heads=2), ValueError), (dict(q=4097), ValueError),
    (dict(q_out=4096), ValueError), (dict(q_out=4096 + 128), ValueError), (dict(seqlen=2, q_out_stride_token=32), ValueError),
    (dict(head_dim=256, rotary_dim=2, q_stride_token=257, seqlen=2), ValueError)])
def test_c_refusals(kw, error, bwd):
    lib = _capi.load()
    entry = lib.mimir_prefixlm_norm_rotary_bwd if bwd else lib.mimir_prefixlm_norm_rotary
    with pytest.raises(error):
        _capi.raise_for_status(lib, entry(ctypes.byref(_params(**kw)), None))


def test_c_refusals_of_the_gradient():
    lib = _capi.load()
    run = lambda p: _capi.raise_for_status(lib, lib.mimir_prefixlm_norm_rotary_bwd(ctypes.byref(p), None))  # noqa: E731
    with pytest.raises(ValueError, match="NULL"):
        run(_params(dq=None))
    with pytest.raises(ValueError, match="memory of their own"):
        run(_params(dq=8192))
    p = _params(dq_weight=64)
    need = lib.mimir_prefixlm_norm_rotary_workspace_bytes(ctypes.byref(p))
    assert need >= 2 * 64 * 4
    p.workspace, p.workspace_bytes = 1 << 20, need - 1
    with pytest.raises(ValueError, match="workspace"):
        run(p)
    p.workspace, p.workspace_bytes = None, need
    with pytest.raises(ValueError, match="workspace"):
        run(p)
    assert lib.mimir_prefixlm_norm_rotary_workspace_bytes(ctypes.byref(_params())) == 0


def test_struct_matches_the_header():
    """Offsets as gcc lays the header's struct out."""
    from tests.test_capi import _c_layout

    fields = [f[0] for f in _capi.NormRotaryParams._fields_]
    size, offsets = _c_layout("MimirNormRotaryParams", fields)
    assert ctypes.sizeof(_capi.NormRotaryParams) == size
    assert [getattr(_capi.NormRotaryParams, f).offset for f in fields] == offsets


def _status(p, bwd):
    lib = _capi.load()
    entry = lib.mimir_prefixlm_norm_rotary_bwd if bwd else lib.mimir_prefixlm_norm_rotary
    return entry(ctypes.byref(p), None), lib.mimir_prefixlm_last_error().decode()


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("kw", [dict(q_stride_head=1), dict(q_stride_batch=3), dict(q_stride_token=1, q_out_stride_batch=1, q_out_stride_head=3),
                                dict(dq_stride_token=5, dq_stride_head=1), dict(seqlen=1, k_stride_head=1, dk_stride_batch=1, num_kv_heads=1)])
@pytest.mark.skipif(torch.cuda.is_available(), reason="what is not refused would be launched, on addresses that are none")
def test_strides_of_one_entry_refuse_nothing(kw, bwd):
    """256 columns need accesses of two: strides of dims of one entry (here all) do not stand in their way.  Past all
    refusals there is no device here."""
    at = dict(head_dim=256, rotary_dim=256, q=1 << 20, q_out=2 << 20, dq=3 << 20, k=4 << 20, k_out=5 << 20, dk=6 << 20)
    for t in ("q", "q_out", "dq", "k", "k_out", "dk"):
        at[t + "_stride_token"] = at[t + "_stride_head"] = at[t + "_stride_batch"] = 256
    status, message = _status(_params(**{**at, **kw}), bwd)
    assert "columns at a time" not in message and status == _capi.ERR_HIP
    status, message = _status(_params(**{**at, **kw, "num_q_heads": 2, "q_stride_head": 257}), bwd)
    assert "columns at a time" in message
