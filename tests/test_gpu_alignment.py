"""Calls whose operands torch calls contiguous, off their 16 bytes or with odd strides on dims of one entry, against
the same calls on aligned copies."""

import pytest
import torch

import mimir_amd
from mimir_amd.cache import Cache, attention_with_cache
from mimir_amd.paged import PagedCache, PageTable, attention_with_pages, reserve_pages

pytestmark = pytest.mark.gpu


def _heads(device, B, S, width, at, heads, d, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, width, generator=gen).bfloat16().to(device)
    return x[..., at:at + heads * d].unflatten(-1, (heads, d))


@pytest.mark.parametrize("B,S", [(1, 1), (2, 1), (1, 70), (2, 70)])
@pytest.mark.parametrize("q_at,k_at", [(0, 4), (8, 0), (2, 1)])
def test_cached_attention(device, B, S, q_at, k_at):
    d, hq, hkv = 64, 4, 2
    q = _heads(device, B, S, hq * d + 12, q_at, hq, d, 1)
    k, v = _heads(device, B, S, hkv * d + 5, k_at, hkv, d, 2), _heads(device, B, S, hkv * d + 5, 0, hkv, d, 3)
    lens = torch.full((B,), 30, dtype=torch.int32, device=device)
    for causal in (True, False):
        got = []
        for copy in (False, True):
            ops = [t.clone(memory_format=torch.contiguous_format) if copy else t for t in (q, k, v)]
            paged, table = PagedCache.create(2 * 4, 1, hkv, d, device=device), PageTable.create(B, 2, 2 * 4, device=device)
            reserve_pages(table, lens + S)
            bf16 = Cache.create(B, 128, hkv, d, dtype=torch.bfloat16, device=device)
            got.append((attention_with_pages(*ops, paged, 0, table.pages, lens, causal), paged.keys.view(torch.uint8),
                        attention_with_cache(*ops, bf16, lens, causal), bf16.keys, bf16.values))
        for a, b in zip(*got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 37])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_operator(device, T, dtype):
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    n = T * 2 * 64
    flat = [torch.randn(n + 8, device=device).to(dtype) for _ in range(3)]
    for at in (1, 2, 4):
        grads = []
        for copy in (False, True):
            ops = [x[at + i:at + i + n].view(T, 2, 64) for i, x in enumerate(flat)]
            ops = [(x.clone(memory_format=torch.contiguous_format) if copy else x.detach()).requires_grad_(True) for x in ops]
            out = mimir_amd.flash_attn_varlen_prefixlm(*ops, False, ints(T // 2), ints(T - T // 2), ints(0, T), T, 1, T // 2, T - T // 2, T)
            grads.append((out, *torch.autograd.grad(out.float().sum(), ops)))
        for a, b in zip(*grads):
            assert torch.equal(a, b)


def test_row_numbers_past_32_bits_beside_narrow_lengths(device):
    """They name no row: zeros, and nothing is written."""
    q, k = torch.randn(2, 1, 4, 64, device=device).bfloat16(), torch.randn(2, 1, 2, 64, device=device).bfloat16()
    lens = torch.tensor([3, 5], dtype=torch.int32, device=device)
    far = torch.tensor([1 << 32, 1], device=device)
    paged, table = PagedCache.create(4, 1, 2, 64, device=device), PageTable.create(2, 1, 4, device=device)
    reserve_pages(table, lens + 1)
    out = attention_with_pages(q, k, k, paged, 0, table.pages, lens, True, far)
    assert not out[0].any() and out[1].any() and not paged.keys[0].view(torch.uint8).any() and paged.keys[1].view(torch.uint8).any()
    new = torch.tensor([1, (1 << 32) + 1], device=device)  # more than the call's one token: that one
    assert torch.equal(attention_with_pages(q, k, k, paged, 0, table.pages, lens, True, far, new_lengths=new), out)
    bf16 = Cache.create(2, 16, 2, 64, dtype=torch.bfloat16, device=device)
    out = attention_with_cache(q, k, k, bf16, lens, True, far)
    assert not out[0].any() and out[1].any() and not bf16.keys[0].any()
