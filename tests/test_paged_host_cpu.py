"""The native host calls of rotary positions and the paged cache, bound to a stub of the C ABI, on CPU
tensors: what each does with a status of the launch, what it passes on, and what it leaves to the
general path."""

import ctypes
import importlib.machinery
import importlib.util
import os
import shutil
import subprocess

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.paged import PagedCache, PageTable
from test_host_calls_cpu import INCLUDE, STUB

MORE = r"""
extern "C" {
int stub_heads = 0, stub_inverse = 0, stub_null_k = 0;
int mimir_prefixlm_rotary(const MimirRotaryParams* p, void*) {  // x + 1 turned one way, x - 1 the other
  stub_heads = p->num_q_heads + p->num_kv_heads;
  stub_inverse = p->inverse;
  for (int part = 0; part < 2; ++part) {
    const float* x = (const float*)(part ? p->k : p->q);
    float* y = (float*)(part ? p->k_out : p->q_out);
    if (x == nullptr) continue;
    for (int i = 0; i < p->seqlen; ++i)
      for (int h = 0; h < (part ? p->num_kv_heads : p->num_q_heads); ++h)
        for (int d = 0; d < p->head_dim; ++d)
          y[i * (part ? p->k_out_stride_token : p->q_out_stride_token) + h * (part ? p->k_out_stride_head : p->q_out_stride_head) + d] =
              x[i * (part ? p->k_stride_token : p->q_stride_token) + h * (part ? p->k_stride_head : p->q_stride_head) + d] * (p->inverse ? 3 : 2);
  }
  return launched();
}
int mimir_prefixlm_paged_attn(const MimirPagedAttnParams*, void*) { return launched(); }
size_t mimir_prefixlm_paged_attn_workspace_bytes(const MimirPagedAttnParams*) { return 64; }
size_t mimir_prefixlm_pages_workspace_bytes(const MimirPagesParams*, int32_t) { return 64; }
int mimir_prefixlm_pages_fork(const MimirPagesParams*, const int32_t*, const int32_t*, int32_t, void*) { return launched(); }
int mimir_prefixlm_pages_compact(const MimirPagesParams*, int32_t*, void*) { return launched(); }
int mimir_prefixlm_pages_release(const MimirPagesParams*, const int32_t*, int32_t, void*) { return launched(); }
int mimir_prefixlm_pages_reserve(const MimirPagesParams*, const int32_t*, void*) { return launched(); }
}
"""


@pytest.fixture(scope="module")
def bound(tmp_path_factory):
    if not _capi.HOST_PATH.exists():
        from mimir_amd.build import build

        build(verbose=False)
    tmp = tmp_path_factory.mktemp("host")
    assert str(INCLUDE) in STUB
    subprocess.run([os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-x", "c++", "-", "-o", str(tmp / "stub.so")],
                   input=STUB + MORE, text=True, check=True)
    copy = shutil.copy(_capi.HOST_PATH, tmp / "_host_calls.so")
    loader = importlib.machinery.ExtensionFileLoader("_host_calls", str(copy))
    host = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host_calls", loader))
    loader.exec_module(host)
    host.bind(str(tmp / "stub.so"), "cpu")
    host.streams(lambda device: 0)
    return host, ctypes.CDLL(str(tmp / "stub.so"))


def _state():
    cache = PagedCache.create(4, 2, 2, 64, device="cpu")
    table = PageTable.create(3, 2, 4, device="cpu")
    q, k = torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16)
    ints = torch.zeros(3, dtype=torch.int32)
    return cache, table, q, k, ints


def _calls(host):
    cache, table, q, k, ints = _state()
    x, pos, turns = torch.ones(5, 2, 8), torch.arange(5), torch.zeros(4, dtype=torch.int64)
    return {
        "rotary": lambda: host.rotary(x, None, pos, turns, 1.0, False, False, False, 0),
        "paged_attn": lambda: host.paged_attn(q, k, k, cache, 1, table.pages, ints, True, None, ints, 0.125, 0),
        "fork": lambda: host.pages("fork", table, cache, ints, ints, 0),
        "compact": lambda: host.pages("compact", table, cache, None, None, 0),
        "release": lambda: host.pages("release", table, None, ints[:2], None, 0),
        "reserve": lambda: host.pages("reserve", table, None, ints, None, 0),
    }


@pytest.mark.parametrize("name", ["rotary", "paged_attn", "fork", "compact", "release", "reserve"])
def test_status_of_the_launch(bound, name):
    host, stub = bound
    status, calls = (ctypes.c_int.in_dll(stub, x) for x in ("stub_status", "stub_calls"))
    call = _calls(host)[name]
    calls.value, status.value = 0, _capi.OK
    assert call() is not None and calls.value == 1
    try:
        for refused in (_capi.ERR_INVALID_ARGUMENT, _capi.ERR_UNSUPPORTED_DTYPE, _capi.ERR_UNSUPPORTED_SHAPE):
            calls.value, status.value = 0, refused
            assert call() is None and calls.value == 1  # left to the general path, which raises
        calls.value, status.value = 0, _capi.ERR_HIP
        with pytest.raises(RuntimeError, match="stub launch failed"):
            call()
        assert calls.value == 1
    finally:
        status.value = _capi.OK


def test_rotary_gradients(bound):
    host, stub = bound
    x = torch.randn(5, 3, 8, requires_grad=True)
    k = torch.randn(5, 1, 8, requires_grad=True)
    pos, turns = torch.arange(5), torch.zeros(4, dtype=torch.int64)
    a, b = host.rotary(x, k, pos, turns, 1.0, False, False, False, 0)
    assert torch.equal(a, 2 * x) and torch.equal(b, 2 * k) and a.requires_grad
    dx, dk = torch.autograd.grad((a, b), (x, k), (torch.ones_like(a), torch.ones_like(b)), retain_graph=True)
    assert (dx == 3).all() and (dk == 3).all() and ctypes.c_int.in_dll(stub, "stub_inverse").value == 1
    assert ctypes.c_int.in_dll(stub, "stub_heads").value == 4
    dk, = torch.autograd.grad(b.sum(), k, retain_graph=True)  # one side alone
    assert (dk == 3).all() and ctypes.c_int.in_dll(stub, "stub_heads").value == 1
    w = torch.randn(5, 3, 8, requires_grad=True)
    dx, = torch.autograd.grad((a * w).sum(), x, create_graph=True)
    assert (torch.autograd.grad(dx.sum(), w)[0] == 2).all()  # the gradient of the turn back is the turn
    a, b = host.rotary(x, k.detach(), pos, turns, 1.0, False, False, False, 0)
    dx, = torch.autograd.grad(a.sum() + b.sum(), x)
    assert (dx == 3).all() and ctypes.c_int.in_dll(stub, "stub_heads").value == 3
    with torch.no_grad():
        assert not host.rotary(x, k, pos, turns, 1.0, False, False, False, 0)[0].requires_grad


def test_left_to_the_general_path(bound):
    host, stub = bound
    calls = ctypes.c_int.in_dll(stub, "stub_calls")
    cache, table, q, k, ints = _state()
    x, pos, turns = torch.ones(5, 2, 8), torch.arange(5), torch.zeros(4, dtype=torch.int64)
    calls.value = 0
    rotary = lambda q=x, k=None, pos=pos, turns=turns, inplace=False: host.rotary(q, k, pos, turns, 1.0, False, False, inplace, 0)  # noqa: E731
    for kw in (dict(q=x.double()), dict(q=x[0]), dict(q=x[:0]), dict(k=x[:3]), dict(k=x.bfloat16()), dict(pos=pos.float()), dict(pos=pos[:3]),
               dict(turns=turns.int()), dict(turns=torch.zeros(5, dtype=torch.int64)), dict(q=x.transpose(1, 2)), dict(pos=pos[None]),
               dict(q=x.clone().requires_grad_(True), inplace=True), dict(q=x[:, :1].expand(5, 2, 8), inplace=True)):
        assert rotary(**kw) is None, kw
    attn = lambda q=q, k=k, cache=cache, layer=0, pages=table.pages, lens=ints, new=None, rows=None: host.paged_attn(  # noqa: E731
        q, k, k, cache, layer, pages, lens, True, rows, new, 0.125, 0)
    for kw in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:0]), dict(k=k[:2]), dict(layer=2), dict(layer=-1), dict(pages=table.pages.long()),
               dict(lens=ints.float()), dict(lens=ints[:2]), dict(new=ints.long()), dict(rows=ints[:1]),
               dict(cache=cache._replace(keys=cache.keys.view(torch.uint8))), dict(cache=cache._replace(values=cache.values[:2])),
               dict(cache=cache._replace(keys=cache.keys.transpose(1, 2))), dict(cache=PagedCache.create(4, 1, 3, 64, device="cpu"))):
        assert attn(**kw) is None, kw
    pages = lambda call, table=table, cache=cache, a=ints, b=None: host.pages(call, table, cache, a, b, 0)  # noqa: E731
    for args in (("other",), ("fork",), ("fork", table, cache, ints, ints[:2]), ("release", table, None, ints.long()), ("release", table, None, ints[:0]),
                 ("reserve", table, None, ints[:2]), ("reserve", table._replace(pages=table.pages.t()), None),
                 ("compact", table, PagedCache.create(5, 1, 1, 64, device="cpu"), None),
                 ("release", table._replace(lengths=ints[:2]), None), ("release", table._replace(counts=ints.long()), None)):
        assert pages(*args) is None, args[0]
    assert calls.value == 0


def test_one_tensor_in_place_as_query_and_key(bound):
    host, _ = bound
    x, pos, turns = torch.ones(5, 2, 8), torch.arange(5), torch.zeros(4, dtype=torch.int64)
    assert host.rotary(x, x, pos, turns, 1.0, False, False, True, 0) is None
    assert host.rotary(x, x[:, :1], pos, turns, 1.0, False, False, True, 0) is None
    assert host.rotary(x[:, :1], x[:, 1:], pos, turns, 1.0, False, False, True, 0) is not None  # a fused projection's heads
    assert host.rotary(x, x, pos, turns, 1.0, False, False, False, 0) is not None


def test_in_place_is_seen_by_autograd(bound):
    host, _ = bound
    pos, turns = torch.arange(5), torch.zeros(4, dtype=torch.int64)
    x = torch.ones(5, 2, 8, requires_grad=True) * 1
    y = (x * x).sum()
    with torch.no_grad():
        assert host.rotary(x, None, pos, turns, 1.0, False, False, True, 0) is not None
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    with torch.inference_mode():
        z = torch.ones(5, 2, 8)
        assert host.rotary(z, z.clone(), pos, turns, 1.0, False, False, True, 0) is not None


def test_tangents_take_the_general_path(bound):
    import torch.autograd.forward_ad as fwd

    host, stub = bound
    x, pos, turns = torch.ones(5, 2, 8), torch.arange(5), torch.zeros(4, dtype=torch.int64)
    with fwd.dual_level():
        d = fwd.make_dual(x, x)
        ctypes.c_int.in_dll(stub, "stub_calls").value = 0
        for q, k in ((d, None), (d, x), (x, d), (d, d)):
            for inplace in (False, True):
                assert host.rotary(q, k, pos, turns, 1.0, False, False, inplace, 0) is None
        assert ctypes.c_int.in_dll(stub, "stub_calls").value == 0
        assert host.rotary(x, None, pos, turns, 1.0, False, False, False, 0) is not None


def test_a_failed_launch_under_autograd_is_not_run_again(bound):
    host, stub = bound
    status, calls = (ctypes.c_int.in_dll(stub, x) for x in ("stub_status", "stub_calls"))
    x, pos, turns = torch.ones(5, 2, 8, requires_grad=True), torch.arange(5), torch.zeros(4, dtype=torch.int64)
    call = lambda: host.rotary(x, None, pos, turns, 1.0, False, False, False, 0)  # noqa: E731
    out, _ = call()
    try:
        calls.value, status.value = 0, _capi.ERR_HIP
        with pytest.raises(RuntimeError, match="stub launch failed"):
            call()
        assert calls.value == 1
        with pytest.raises(RuntimeError, match="stub launch failed"):
            out.sum().backward()
        assert calls.value == 2
        status.value = _capi.ERR_UNSUPPORTED_SHAPE  # nothing launched: the general path raises it
        assert call() is None
    finally:
        status.value = _capi.OK


def test_launches_release_the_interpreter(tmp_path):
    source = (STUB + MORE).replace("static int launched() {", "int PyGILState_Check(void);\nint stub_locked = 0;\n"
                                   "static int launched() { stub_locked += PyGILState_Check();")
    subprocess.run([os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-x", "c++", "-", "-o", str(tmp_path / "stub.so")],
                   input=source, text=True, check=True)
    copy = shutil.copy(_capi.HOST_PATH, tmp_path / "_host_calls.so")
    loader = importlib.machinery.ExtensionFileLoader("_host_calls", str(copy))
    host = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host_calls", loader))
    loader.exec_module(host)
    host.bind(str(tmp_path / "stub.so"), "cpu")
    host.streams(lambda device: 0)
    stub = ctypes.CDLL(str(tmp_path / "stub.so"))
    calls, locked = (ctypes.c_int.in_dll(stub, x) for x in ("stub_calls", "stub_locked"))
    for name, call in _calls(host).items():
        assert call() is not None and locked.value == 0, name
    x = torch.ones(5, 2, 8, requires_grad=True)
    y, _ = host.rotary(x, None, torch.arange(5), torch.zeros(4, dtype=torch.int64), 1.0, False, False, False, 0)
    y.sum().backward()
    assert locked.value == 0 and calls.value == 8
