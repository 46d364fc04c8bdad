"""Operands that torch calls contiguous but that do not start on 16 bytes, or have odd strides on dims of one entry,
are copied to where the kernels can read them."""

import pytest
import torch

from mimir_amd import cache, paged
from mimir_amd import prefixlm as P


def _projection(B, S, extra, at, heads=2, d=64, dtype=torch.bfloat16):
    """Heads of a fused projection with a few more columns, from column ``at`` on."""
    x = torch.arange(B * S * (heads * d + extra), dtype=torch.float32).to(dtype).view(B, S, heads * d + extra)
    return x[..., at:at + heads * d].unflatten(-1, (heads, d))


@pytest.mark.parametrize("B,S", [(1, 1), (1, 3), (2, 1), (2, 3)])
@pytest.mark.parametrize("extra,at", [(4, 4), (4, 0), (3, 1), (8, 8), (8, 0), (16, 2)])
def test_rows_of_the_cached_attention(monkeypatch, B, S, extra, at):
    monkeypatch.setattr(P, "_check_device_tensor", lambda name, t: None)
    t = _projection(B, S, extra, at)
    for got, strides in ((paged._rows4(t), paged._strides), (cache._rows4("query", t), lambda x: x.stride()[:3])):
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and got.stride(-1) == 1 and not any(s % 8 for s in strides(got))
    if at % 8 == 0 and (B == S == 1 or extra % 8 == 0):
        assert paged._rows4(t).data_ptr() == t.data_ptr()  # read in place


@pytest.mark.parametrize("T", [1, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_the_operator(T, dtype):
    flat = torch.arange(T * 2 * 64 + 8, dtype=torch.float32).to(dtype)
    for at in range(8):
        t = flat[at:at + T * 2 * 64].view(T, 2, 64)
        got = P._kernel_layout(t)
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0
        assert (got.data_ptr() == t.data_ptr()) == (t.data_ptr() % 16 == 0)
    odd = flat[:T * 128].as_strided((T, 2, 64), (129 if T == 1 else 128, 64, 1))
    got = P._kernel_layout(odd)
    assert torch.equal(got, odd) and got.stride(0) % 8 == 0


def test_rope_tables():
    flat = torch.arange(3 * 64 + 4, dtype=torch.float32)
    for at in range(4):
        t = flat[at:at + 3 * 64].view(3, 64)
        got = P.rope_rows(t, 3, 64, t.device, "cos")
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and (got.data_ptr() == t.data_ptr()) == (at == 0)
