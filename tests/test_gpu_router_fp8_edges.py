"""Corners of the router and FP8 operators: tensors that are not stored as they read, derivatives that are not there, padded batches, rows that are asked for very
often, outputs with the longest rows."""
import ctypes as C
import math

import pytest
import torch

import sm120fp4_b200 as pkg
import sm120fp4_b200._lib as L

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
fwd = torch.autograd.forward_ad


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def same(a, b):
    return torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, b.view(torch.uint8) if b.dtype == FP8 else b)


@pytest.fixture(params=["native", "general"])
def path(request, monkeypatch):
    """Both host sides: the extension, and the path beside it."""
    if request.param == "general":
        monkeypatch.setattr(L, "_host", L.NO_HOST)
    return request.param


# ---------------------------------------------------------------------------------------------------- derivatives that are not there

def test_forward_mode_is_refused(path):
    """Outputs without a tangent would read as a derivative of zero."""
    x = randn(6, 16)
    ids = pkg.top_k_gate(x, 2)[1]
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: pkg.top_k_gate(dual, 2), lambda: pkg.top_k_gate(dual, 2, renormalize=False), lambda: pkg.balance_loss(dual, ids)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(pkg.top_k_gate(x, 2)[1], ids)      # plain tensors as ever
    for call in (lambda t: pkg.top_k_gate(t, 2)[0], lambda t: pkg.balance_loss(t, ids)[0]):
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))


def test_an_error_in_a_gradient_reaches_the_caller():
    """The library says no inside a backward pass, on a thread of the autograd engine: an exception like any other."""
    h, host, no = L.lib(), L.host(), C.CFUNCTYPE(C.c_int, *L.SIGNATURES["b200moe_gate_backward"][1])(lambda *args: L.ERR_ARG)
    functions = L.host_functions(h)
    x = randn(5, 16, seed=1).requires_grad_(True)
    w = pkg.top_k_gate(x, 3)[0]
    assert host.top_k_gate(x, 3, True) is not None
    try:
        host.bind_ops(*(C.cast(no, C.c_void_p).value if f is h.b200moe_gate_backward else C.cast(f, C.c_void_p).value for f in functions))
        with pytest.raises(RuntimeError, match=r"top_k_gate backward: bad argument.*\(-1\)"):
            w.sum().backward()
    finally:
        host.bind_ops(*(C.cast(f, C.c_void_p).value for f in functions))
    pkg.top_k_gate(x, 3)[0].sum().backward()
    assert x.grad is not None


# ---------------------------------------------------------------------------------------------------- tensors that are not stored as they read

# ---------------------------------------------------------------------------------------------------- rows outside every run

def best_us(fn, n=7):
    """Shortest of n calls, in microseconds on the device."""
    times = []
    for _ in range(n):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return min(times)
