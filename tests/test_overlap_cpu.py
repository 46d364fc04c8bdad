"""In-place rotary positions refuse memory whose elements would be turned twice: the overlap of strided
regions (csrc/strided_overlap.h) against sets of addresses, and the calls that use it."""

import ctypes
import os
import random
import subprocess
from pathlib import Path

import pytest
import torch

from mimir_amd import _capi
from test_paged_host_cpu import bound  # noqa: F401 (a fixture)
from test_rotary_cpu import _params

HEADER = Path(__file__).resolve().parents[1] / "mimir_amd" / "csrc" / "strided_overlap.h"
PROGRAM = f'#include "{HEADER}"\n' + r"""
using mimir::Region;
static Region region(const int64_t* x) { return {(const void*)x[0], x[1], {x[2], x[3], x[4]}, {x[5], x[6], x[7]}}; }
extern "C" int itself(const int64_t* a) { return mimir::overlaps_itself(region(a)); }
extern "C" int each_other(const int64_t* a, const int64_t* b) { return mimir::overlap_each_other(region(a), region(b)); }
"""


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    so = tmp_path_factory.mktemp("overlap") / "overlap.so"
    subprocess.run([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-shared", "-fPIC", "-x", "c++", "-", "-o", str(so)], input=PROGRAM,
                   text=True, check=True)
    lib = ctypes.CDLL(str(so))
    pack = lambda r: (ctypes.c_int64 * 8)(*r)  # noqa: E731
    return lambda a: bool(lib.itself(pack(a))), lambda a, b: bool(lib.each_other(pack(a), pack(b)))


def _bytes(r):
    base, run, n, s = r[0], r[1], r[2:5], r[5:8]
    return [base + i * s[0] + j * s[1] + k * s[2] + e for i in range(n[0]) for j in range(n[1]) for k in range(n[2]) for e in range(run)]


def test_overlap_is_exact(overlap):
    itself, each_other = overlap
    rng = random.Random(0)
    seen = set()
    for _ in range(6000):
        def region():
            n = [rng.choice([0, 1, 2, 3, 4]) if rng.random() < 0.9 else rng.randint(1, 7) for _ in range(3)]
            s = [rng.choice([0, 2, 4, 6, 8, 12, 24, 30, 48, 64, 96, -8, -24]) for _ in range(3)]
            return [1000 + 2 * rng.randint(0, 60), rng.choice([2, 4, 6, 8, 16]), *n, *s]

        a, b = region(), region()
        if rng.random() < 0.5:
            b[5:] = a[5:]  # views of one tensor
        x, y = _bytes(a), _bytes(b)
        assert itself(a) == (len(set(x)) < len(x)), a
        assert each_other(a, b) == bool(set(x) & set(y)), (a, b)
        seen.add((len(set(x)) < len(x), bool(set(x) & set(y))))
    assert len(seen) == 4


def test_overlap_of_large_regions(overlap):
    itself, each_other = overlap
    at = 1 << 40
    for b, s, h, d in ((8, 32768, 40, 256), (1, 1 << 20, 1, 128), (512, 1, 64, 256)):
        fused = 2 * h * d
        q, k = [at, d, b, s, h, s * fused, fused, d], [at + h * d, d, b, s, h, s * fused, fused, d]
        assert not itself(q) and not each_other(q, k)                                  # heads side by side
        q[7] = k[7] = 2 * d
        k[0] = at + d
        assert not itself(q) and not each_other(q, k)                                  # heads in turn
        k[0] = at + d - 2
        assert each_other(q, k)
        q, k = [at, d, b, s, h, s * fused, d, s * d], [at + h * s * d, d, b, s, h, s * fused, d, s * d]
        assert not itself(q) and not each_other(q, k)                                  # heads in front of tokens
        assert each_other(q, [k[0] - 2, *k[1:]])


CASES = [
    (lambda x: (x[:, :3], x[:, 2:]), True),               # one head in both
    (lambda x: (x[:, :2], x[:, 2:]), False),              # a fused projection's heads
    (lambda x: (x[:, ::2], x[:, 1::2]), False),           # heads in turn
    (lambda x: (x[:, ::2], x[:, 2:]), True),
    (lambda x: (x[:4], x[1:]), True),                     # the same tokens, one apart
    (lambda x: (x[:, :2, :8], x[:, :2, 8:]), False),      # halves of the same heads
    (lambda x: (x[:, :2, :8], x[:, :2, 4:12]), True),
    (lambda x: (x[:, 3:], x[:, :3]), False),
    (lambda x: (torch.as_strided(x, (5, 3, 8), (16, 4, 1)), None), True),  # heads that lie in each other
    (lambda x: (torch.as_strided(x, (5, 3, 8), (8, 16, 1)), None), True),  # and tokens in heads
    (lambda x: (torch.as_strided(x, (5, 3, 8), (8, 40, 1)), None), False),
]


@pytest.mark.parametrize("case,turned_twice", CASES)
def test_in_place_views_of_one_tensor(bound, case, turned_twice):  # noqa: F811
    host, stub = bound
    calls = ctypes.c_int.in_dll(stub, "stub_calls")
    q, k = case(torch.ones(5, 4, 16))
    pos, turns = torch.arange(q.shape[0]), torch.zeros(q.shape[-1] // 2, dtype=torch.int64)
    calls.value, version = 0, q._version
    out = host.rotary(q, k, pos, turns, 1.0, False, False, True, 0)
    assert (out is None) == turned_twice and calls.value == (not turned_twice)
    assert q._version == version + (not turned_twice) * (1 if k is None else 2)
    assert host.rotary(q, k, pos, turns, 1.0, False, False, False, 0) is not None  # into new tensors it is served


def test_only_the_turned_columns_count_in_place(bound):  # noqa: F811
    host, _ = bound
    x, pos = torch.ones(5, 4, 16), torch.arange(5)
    call = lambda n: host.rotary(x[:, :, :8], x[:, :, 4:12], pos, torch.zeros(n, dtype=torch.int64), 1.0, False, False, True, 0)  # noqa: E731
    assert call(2) is not None and call(3) is None and call(4) is None


@pytest.mark.parametrize("kw", [
    dict(),                                                  # heads of stride 0
    dict(q_stride_head=64, q_out_stride_head=64, k=4096 + 64 * 2, k_out=4096 + 64 * 2),  # the key is query head 1
    dict(q_stride_head=32, q_out_stride_head=32, k=1 << 20, k_out=1 << 20),
    dict(q_stride_head=64, q_out_stride_head=64, q_out=4096 + 2 * 8, k=1 << 20, k_out=1 << 21),  # the output is the input moved on
    dict(q_stride_head=64, q_out_stride_head=64, q_out=1 << 20, k=1 << 21, k_out=4096 + 2 * 64),  # the key's output is a query head
    dict(q_stride_head=64, q_out_stride_head=128, k=1 << 20, k_out=1 << 20),
])
def test_c_abi_refuses_overlapping_outputs(kw):
    lib = _capi.load()
    with pytest.raises(ValueError, match="memory of their own"):
        _capi.raise_for_status(lib, lib.mimir_prefixlm_rotary(ctypes.byref(_params(**kw)), None))
