"""The native host calls of normed rotary heads, cross attention and beam search, bound to a stub of the C ABI,
on CPU tensors: statuses of the launch, gradients, and what is left to the general path."""

import ctypes
import importlib.machinery
import importlib.util
import os
import shutil
import subprocess

import pytest
import torch

from mimir_amd import _capi
from mimir_amd.cache import Cache
from test_host_calls_cpu import INCLUDE, STUB

MORE = r"""
extern "C" {
int stub_wants = 0, stub_null = 0;
size_t mimir_prefixlm_norm_rotary_workspace_bytes(const MimirNormRotaryParams*) { return 64; }
int mimir_prefixlm_norm_rotary(const MimirNormRotaryParams* p, void*) {
  for (int i = 0; i < p->seqlen * p->head_dim; ++i) ((float*)p->q_out)[i] = 2 * ((const float*)p->q)[i];
  return launched();
}
int mimir_prefixlm_norm_rotary_bwd(const MimirNormRotaryParams* p, void*) {  // what is asked for, as numbers
  stub_wants = (p->dq_weight != nullptr) + 2 * (p->dk_weight != nullptr) + 4 * (p->k != nullptr) + 8 * (p->workspace != nullptr);
  for (int i = 0; i < p->seqlen * p->head_dim; ++i) ((float*)p->q_out)[i] = 3 * ((const float*)p->dq)[i];
  if (p->k_out != nullptr)
    for (int i = 0; i < p->seqlen * p->head_dim; ++i) ((float*)p->k_out)[i] = 5 * ((const float*)p->dk)[i];
  for (int i = 0; i < p->head_dim; ++i) {
    if (p->dq_weight != nullptr) ((float*)p->dq_weight)[i] = 7;
    if (p->dk_weight != nullptr) ((float*)p->dk_weight)[i] = 11;
  }
  return launched();
}
size_t mimir_prefixlm_cross_workspace_bytes(const MimirCrossParams*, int32_t backward) { return backward ? 512 : 256; }
int mimir_prefixlm_cross_fwd(const MimirCrossParams* p, void*) {
  stub_null = p->lse2 == nullptr;
  for (int i = 0; i < p->total_q * p->num_q_heads * p->head_dim; ++i) ((uint16_t*)p->out)[i] = 0x3f80;  // 1
  return launched();
}
int mimir_prefixlm_cross_bwd(const MimirCrossParams* p, void*) {
  stub_wants = p->workspace_bytes == 512 && p->lse2 != nullptr && p->out_lo != nullptr;
  for (int i = 0; i < p->total_q * p->num_q_heads * p->head_dim; ++i) ((uint16_t*)p->dq)[i] = ((const uint16_t*)p->dout)[i];
  for (int i = 0; i < p->total_k * p->num_kv_heads * p->head_dim; ++i) ((uint16_t*)p->dk)[i] = 0x4000, ((uint16_t*)p->dv)[i] = 0x4040;  // 2, 3
  return launched();
}
size_t mimir_prefixlm_states_workspace_bytes(const MimirStatesParams*) { return 256; }
int mimir_prefixlm_states_attn(const MimirStatesParams* p, void*) { stub_wants = p->seq_tokens; return launched(); }
size_t mimir_prefixlm_beam_select_workspace_bytes(const MimirBeamSelectParams*) { return 256; }
int mimir_prefixlm_beam_select(const MimirBeamSelectParams* p, void*) { stub_wants = p->count; return launched(); }
int mimir_prefixlm_reorder_rows(const MimirReorderParams* p, void*) { stub_wants = p->count; return launched(); }
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


def _aligned(*shape):
    """bf16 in memory that starts on 16 bytes."""
    n = 1
    for s in shape:
        n *= s
    hold = torch.zeros(n + 8, dtype=torch.bfloat16)
    at = (16 - hold.data_ptr() % 16) % 16 // 2
    return hold[at:at + n].view(shape)


def _norm(host, q, k=None, qw=None, kw=None, eps=1e-6, pos=None, turns=None):
    pos = torch.arange(q.shape[0]) if pos is None else pos
    turns = torch.zeros(4, dtype=torch.int64) if turns is None else turns
    return host.norm_rotary(q, k, pos, turns, 1.0, False, qw, kw, eps, 0)


def _calls(host):
    x = torch.ones(5, 1, 8)
    q, k, cu = _aligned(6, 2, 64), _aligned(7, 1, 64), torch.tensor([0, 6], dtype=torch.int32)
    q4, states = _aligned(4, 1, 2, 64), Cache(_aligned(2, 9, 1, 64), _aligned(2, 9, 1, 64))
    ints, source = torch.zeros(2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    return {
        "norm_rotary": lambda: _norm(host, x),
        "cross_attention": lambda: host.cross_attention(q, k, k, cu, cu, 0.125, 0),
        "states": lambda: host.states(q4, *states, ints, None, 0.125, 0),
        "select": lambda: host.select(torch.zeros(2, 3, 9), torch.zeros(2, 3), 4, None, -1, 0),
        "reorder": lambda: host.reorder([states], ints, source, 0),
    }


@pytest.mark.parametrize("name", ["norm_rotary", "cross_attention", "states", "select", "reorder"])
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


def test_a_failed_launch_under_autograd_is_not_run_again(bound):
    host, stub = bound
    status, calls = (ctypes.c_int.in_dll(stub, x) for x in ("stub_status", "stub_calls"))
    x = torch.ones(5, 1, 8, requires_grad=True)
    q, k, cu = _aligned(6, 2, 64).requires_grad_(True), _aligned(7, 1, 64), torch.tensor([0, 6], dtype=torch.int32)
    try:
        for call in (lambda: _norm(host, x)[0], lambda: host.cross_attention(q, k, k, cu, cu, 0.125, 0)):
            calls.value, status.value = 0, _capi.ERR_HIP
            with pytest.raises(RuntimeError, match="stub launch failed"):
                call()
            assert calls.value == 1
            status.value = _capi.ERR_UNSUPPORTED_SHAPE
            assert _none_or_raises(call)
            status.value = _capi.OK
            out = call()
            status.value = _capi.ERR_HIP
            with pytest.raises(RuntimeError, match="stub launch failed"):
                out.sum().backward()
    finally:
        status.value = _capi.OK


def _none_or_raises(call):
    try:
        return call() is None
    except TypeError:  # the [0] of a call that is left to the general path
        return True


@pytest.mark.parametrize("with_key", [False, True])
@pytest.mark.parametrize("weights", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_norm_rotary_gradients(bound, with_key, weights):
    host, stub = bound
    wants = ctypes.c_int.in_dll(stub, "stub_wants")
    if weights[1] and not with_key:
        return
    x, k = torch.randn(5, 1, 8, requires_grad=True), torch.randn(5, 1, 8, requires_grad=True) if with_key else None
    qw, kw = (torch.ones(8, requires_grad=True) if w else None for w in weights)
    y, z = _norm(host, x, k, qw, kw)
    assert torch.equal(y, 2 * x) and (z is None) == (k is None)
    g = torch.randn(5, 1, 8)
    leaves = [t for t in (x, k, qw, kw) if t is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad([t for t in (y, z) if t is not None], leaves, [g, 2 * g][:1 + with_key])))
    assert wants.value == weights[0] + 2 * weights[1] + 4 * with_key + 8
    assert torch.equal(got[id(x)], 3 * g)
    if with_key:
        assert torch.equal(got[id(k)], 10 * g)
    if weights[0]:
        assert (got[id(qw)] == 7).all()
    if weights[1]:
        assert (got[id(kw)] == 11).all()


def test_norm_rotary_weight_that_needs_no_gradient(bound):
    host, stub = bound
    wants = ctypes.c_int.in_dll(stub, "stub_wants")
    x, k, kw = torch.randn(5, 1, 8), torch.randn(5, 1, 8, requires_grad=True), torch.ones(8, requires_grad=True)
    y, z = _norm(host, x, k, torch.ones(8), kw)
    (y.sum() + z.sum()).backward()
    assert wants.value == 2 + 4 + 8 and (kw.grad == 11).all() and (k.grad == 5).all() and x.grad is None
    # one output unused: zeros come for it
    x.requires_grad_(True)
    y, z = _norm(host, x, k.detach(), None, kw.detach())
    gx, = torch.autograd.grad(y.sum(), x)
    assert (gx == 3).all()


def test_cross_gradients(bound):
    host, stub = bound
    wants, null = (ctypes.c_int.in_dll(stub, x) for x in ("stub_wants", "stub_null"))
    q, k, v = _aligned(6, 2, 64).requires_grad_(True), _aligned(7, 1, 64), _aligned(7, 1, 64).requires_grad_(True)
    cu = torch.tensor([0, 6], dtype=torch.int32)
    with torch.no_grad():
        host.cross_attention(q, k, v, cu, cu, 0.125, 0)
    assert null.value == 1  # a forward alone keeps nothing
    out = host.cross_attention(q, k, v, cu, cu, 0.125, 0)
    assert null.value == 0 and (out == 1).all()
    dq, dv = torch.autograd.grad(out.sum(), (q, v))  # an expanded gradient
    assert wants.value == 1 and (dq == 1).all() and (dv == 3).all()


def test_differentiable_once_only(bound):
    host, _ = bound
    x = torch.randn(5, 1, 8, requires_grad=True)
    g, = torch.autograd.grad(_norm(host, x)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="norm_rotary is differentiable once only"):
        g.sum().backward()
    q, k, cu = _aligned(6, 2, 64).requires_grad_(True), _aligned(7, 1, 64), torch.tensor([0, 6], dtype=torch.int32)
    g, = torch.autograd.grad(host.cross_attention(q, k, k, cu, cu, 0.125, 0).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="cross_attention is differentiable once only"):
        g.float().sum().backward()


def test_left_to_the_general_path(bound):
    host, stub = bound
    calls = ctypes.c_int.in_dll(stub, "stub_calls")
    calls.value = 0
    x, w = torch.ones(5, 1, 8), torch.ones(8)
    assert _norm(host, x.half()) is None and _norm(host, x[0]) is None and _norm(host, x.transpose(0, 2)) is None
    assert _norm(host, x[:0]) is None and _norm(host, x, x[:, :, :4]) is None and _norm(host, x, None, w[:4]) is None
    assert _norm(host, x, None, w.double()) is None and _norm(host, x, None, None, w) is None and _norm(host, x, x, w, w.bfloat16()) is None
    assert _norm(host, x, None, w.expand(2, 8)) is None and _norm(host, x, eps=-1.0) is None and _norm(host, x, eps=float("nan")) is None
    assert _norm(host, x, eps="1") is None and _norm(host, x, pos=torch.arange(5.0)) is None and _norm(host, x, turns=torch.zeros(5, dtype=torch.int64)) is None
    with torch.autograd.forward_ad.dual_level():
        assert _norm(host, torch.autograd.forward_ad.make_dual(x, x)) is None
    q, k, cu = _aligned(6, 2, 64), _aligned(7, 1, 64), torch.tensor([0, 6], dtype=torch.int32)
    cross = lambda q=q, k=k, v=k, a=cu, b=cu, s=0.125: host.cross_attention(q, k, v, a, b, s, 0)  # noqa: E731
    assert cross(q=q.float()) is None and cross(q=q[:0]) is None and cross(k=k[:0], v=k[:0]) is None and cross(v=k[:3]) is None
    assert cross(a=cu.long()) is None and cross(b=cu[:1]) is None and cross(a=cu[:1], b=cu[:1]) is None and cross(q=q[..., :32]) is None
    assert cross(q=q.transpose(1, 2)) is None and cross(s="x") is None and cross(k=k.expand(7, 1, 64).float()) is None
    q4, keys, ints = _aligned(4, 1, 2, 64), _aligned(2, 9, 1, 64), torch.zeros(2, dtype=torch.int32)
    states = lambda q=q4, k=keys, v=keys, n=ints, rows=None: host.states(q, k, v, n, rows, 0.125, 0)  # noqa: E731
    assert states(q=q4.float()) is None and states(n=ints[:1]) is None and states(n=ints.float()) is None and states(rows=ints[:0]) is None
    assert states(q=q4[:3]) is None and states(v=keys[:, :3]) is None and states(q=q4.clone().requires_grad_(True)) is None
    assert states(q=_aligned(4, 6, 2, 64)[:, :3]) is None  # a request's tokens not in a row
    x, s, done = torch.zeros(2, 3, 9), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)
    select = lambda x=x, s=s, n=4, done=None, end=-1: host.select(x, s, n, done, end, 0)  # noqa: E731
    assert select(x=x.half()) is None and select(x=x[0]) is None and select(x=x.transpose(1, 2)) is None and select(s=s.double()) is None
    assert select(n=0) is None and select(n=28) is None and select(n=2.0) is None and select(n=None) is None and select(end=9) is None
    assert select(done=done) is None and select(done=done.int(), end=0) is None and select(s=s[:1]) is None and select(x=x[:0], s=s[:0]) is None
    caches, source = [Cache(keys, keys.clone())], torch.zeros(1, 2, dtype=torch.int32)
    reorder = lambda c=caches, n=ints, s=source: host.reorder(c, n, s, 0)  # noqa: E731
    assert reorder(c=[]) is None and reorder(c=caches * 9) is None and reorder(c=[keys]) is None and reorder(n=ints[:1]) is None
    assert reorder(s=source.flatten()) is None and reorder(s=source.float()) is None and reorder(n=ints.float()) is None
    assert reorder(c=[Cache(keys, keys[:, :3])]) is None and reorder(c=[Cache(keys[..., ::2], keys[..., ::2])]) is None
    assert reorder(s=torch.zeros(1, 33, dtype=torch.int32), n=torch.zeros(33, dtype=torch.int32)) is None
    assert calls.value == 0


def test_reordered_caches_are_seen_by_autograd(bound):
    host, _ = bound
    cache, ints, source = Cache(_aligned(2, 9, 1, 64), _aligned(2, 9, 1, 64)), torch.zeros(2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    before = [t._version for t in (*cache, ints)]
    assert host.reorder([cache], ints, source, 0) is True
    assert [t._version for t in (*cache, ints)] == [v + 1 for v in before]
    with torch.inference_mode():
        assert host.reorder([Cache(cache.keys.clone(), cache.values.clone())], ints.clone(), source, 0) is True


def test_a_library_without_the_calls(bound, tmp_path):
    """Bound to a stub that lacks them: every call is left to the general path."""
    subprocess.run([os.environ.get("CXX", "g++"), "-shared", "-fPIC", "-x", "c++", "-", "-o", str(tmp_path / "old.so")], input=STUB, text=True, check=True)
    copy = shutil.copy(_capi.HOST_PATH, tmp_path / "_host_calls.so")
    loader = importlib.machinery.ExtensionFileLoader("_host_calls", str(copy))
    host = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host_calls", loader))
    loader.exec_module(host)
    host.bind(str(tmp_path / "old.so"), "cpu")
    for name, call in _calls(host).items():
        assert call() is None, name
