"""What the router and FP8 operators refuse, without a GPU: wrong types and shapes in Python, wrong arguments at the C ABI (nothing is launched)."""
import pytest
import torch


def test_python_refusals():
    import sm120fp4_b200 as pkg
    x = torch.zeros(4, 8)
    long = torch.zeros(1, 2).expand((1 << 30) + 1, 2)      # (one row of memory)
    for fn in (lambda t: pkg.top_k_gate(t, 1), lambda t: pkg.balance_loss(t, torch.zeros(4, 2, dtype=torch.int32)), pkg.quantize_fp8, pkg.quantize_fp8_weight):
        with pytest.raises(ValueError):
            fn(long)
    with pytest.raises(ValueError):
        pkg.top_k_gate(torch.zeros(8), 2)
    with pytest.raises(TypeError):
        pkg.top_k_gate(torch.zeros(4, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        pkg.top_k_gate(torch.zeros(4, 513), 2)
    with pytest.raises(RuntimeError):
        pkg.top_k_gate(x, 2)
    with pytest.raises(TypeError):
        pkg.balance_loss(torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        pkg.balance_loss(x, torch.zeros(4, 2, dtype=torch.int32))
    for fn in (pkg.quantize_fp8, pkg.quantize_fp8_weight):
        with pytest.raises(ValueError):
            fn(torch.zeros(4, 0))
        with pytest.raises(ValueError):
            fn(torch.zeros(4))
        with pytest.raises(TypeError):
            fn(torch.zeros(4, 8, dtype=torch.int8))
        with pytest.raises(RuntimeError):
            fn(x)


def codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_matmul_refusals():
    import sm120fp4_b200 as pkg
    a, sa, w, sw = codes(4, 256), torch.zeros(4, 2), codes(32, 256), torch.zeros(1, 2)
    with pytest.raises(RuntimeError):
        pkg.matmul_fp8(a, sa, w, sw)
    with pytest.raises(TypeError):
        pkg.matmul_fp8(a.view(torch.uint8), sa, w, sw)
    with pytest.raises(ValueError):
        pkg.matmul_fp8(a, sa, codes(32, 128), sw)
    with pytest.raises(ValueError):
        pkg.matmul_fp8(a, torch.zeros(4, 1), w, sw)
    with pytest.raises(ValueError):
        pkg.matmul_fp8(a, sa, w, torch.zeros(32, 2))
    with pytest.raises(TypeError):
        pkg.matmul_fp8(a, sa.half(), w, sw)
    with pytest.raises(ValueError):
        pkg.matmul_fp8(codes(4, 264)[:, :250], sa, codes(32, 256)[:, :250], sw)      # rows of 264 bytes: the second starts on 8
    with pytest.raises(ValueError):
        pkg.matmul_fp8(codes(4, 272)[:, 8:264], sa, w, sw)                            # rows of a begin on 8
    with pytest.raises(ValueError):
        pkg.matmul_fp8(codes(256, 4).t(), sa, w, sw)
    we, swe, experts, offsets = codes(3, 32, 256), torch.zeros(3, 1, 2), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        pkg.matmul_fp8_experts(a, sa, we, swe, experts, offsets)
    with pytest.raises(TypeError):
        pkg.matmul_fp8_experts(a, sa, we, swe, experts.long(), offsets)
    with pytest.raises(ValueError):
        pkg.matmul_fp8_experts(a, sa, we, swe, experts, offsets[:2])
    with pytest.raises(ValueError):
        pkg.matmul_fp8_experts(a, sa, codes(3, 64, 256)[:, :32], swe, experts, offsets)      # matrices that do not follow one another
    with pytest.raises(ValueError):
        pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets)


def test_c_abi_refusals():
    import sm120fp4_b200._lib as L
    h = L.lib()
    p = 4096      # an aligned address that is never read: every call below is refused or has nothing to do
    assert h.b200moe_gate(None, 0, 8, 4, 8, 2, 1, p, p, None) == L.ERR_ARG
    assert h.b200moe_gate(p, 3, 8, 4, 8, 2, 1, p, p, None) == L.ERR_ARG
    assert h.b200moe_gate(p, 0, 8, 4, 8, 9, 1, p, p, None) == L.ERR_ARG
    assert h.b200moe_gate(p, 0, 7, 4, 8, 2, 1, p, p, None) == L.ERR_ARG
    assert h.b200moe_gate(p, 0, 600, 4, 600, 2, 1, p, p, None) == L.ERR_LIMIT
    assert h.b200moe_gate(p, 0, 64, 4, 64, 17, 1, p, p, None) == L.ERR_LIMIT
    assert h.b200moe_gate(p + 1, 0, 8, 4, 8, 2, 1, p, p, None) == L.ERR_ARG
    assert h.b200moe_gate(None, 0, 8, 0, 8, 2, 1, None, None, None) == 0
    assert h.b200moe_gate(p, 0, 8, (1 << 30) + 1, 8, 2, 1, p, p, None) == L.ERR_LIMIT
    assert h.b200moe_quantize_fp8(p, 0, 16, (1 << 30) + 1, None, (1 << 30) + 1, 16, p, 16, p, None, 0, None) == L.ERR_LIMIT
    assert h.b200moe_quantize_fp8_blocks(p, 0, 1, 65535 * 128 + 1, 16, p, 16, p, None) == L.ERR_LIMIT
    assert h.b200moe_matmul_fp8(p, 16, p, p, 16, p, (1 << 30) + 1, 4, 16, p, 0, 4, None) == L.ERR_LIMIT
    assert h.b200moe_matmul_fp8_experts(p, 16, p, 4, p, 16, p, 1 << 20, p, p, 1, 1 << 11, 16, p, 0, 1 << 11, 0, None) == L.ERR_LIMIT      # rows of all experts beyond 2^31
    assert h.b200moe_gate_backward(p, p, p, None, 0, 8, 4, 8, 2, 0, p, None) == L.ERR_ARG
    assert h.b200moe_balance_workspace_bytes(-1, 8) == L.ERR_ARG and h.b200moe_balance_workspace_bytes(1, 513) == L.ERR_LIMIT
    assert h.b200moe_balance_workspace_bytes(1000, 64) > 0
    assert h.b200moe_balance_loss(p, 0, 8, 4, 8, p, 2, p, p, p, p, 3, None) == L.ERR_WORKSPACE
    assert h.b200moe_balance_loss(p, 0, 8, 4, 8, p, 33, p, p, p, p, 1 << 20, None) == L.ERR_LIMIT
    assert h.b200moe_balance_loss(p, 0, 8, 4, 8, None, 2, p, p, p, p, 1 << 20, None) == L.ERR_ARG
    assert h.b200moe_balance_backward(p, p, 0, 8, 4, 8, p, 2, p, None, p, None) == L.ERR_ARG
    assert h.b200moe_quantize_fp8(p, 0, 16, 4, None, 5, 16, p, 16, p, None, 0, None) == L.ERR_ARG      # rows without a source
    assert h.b200moe_quantize_fp8(p, 0, 16, 4, None, 4, 0, p, 16, p, None, 0, None) == L.ERR_ARG
    assert h.b200moe_quantize_fp8(p, 0, 16, 4, None, 4, 16, p, 15, p, None, 0, None) == L.ERR_ARG
    assert h.b200moe_quantize_fp8(None, 0, 16, 0, None, 0, 16, None, 16, None, None, 0, None) == 0
    assert h.b200moe_quantize_fp8_workspace_bytes(10, 20, 16) == 0 and h.b200moe_quantize_fp8_workspace_bytes(4096, 32768, 2048) == 4 * (4096 + 32768)
    assert h.b200moe_quantize_fp8(p, 0, 2048, 4096, p, 32768, 2048, p, 2048, p, None, 0, None) == L.ERR_WORKSPACE
    assert h.b200moe_quantize_fp8_blocks(p, 0, 1, 4, 16, None, 16, p, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8(p, 16, p, p, 16, p, 4, 4, 17, p, 0, 4, None) == L.ERR_ARG      # rows shorter than K
    assert h.b200moe_matmul_fp8(p, 24, p, p, 32, p, 4, 4, 16, p, 0, 4, None) == L.ERR_ARG      # rows that do not start on 16 bytes
    assert h.b200moe_matmul_fp8(p + 8, 16, p, p, 16, p, 4, 4, 16, p, 0, 4, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8(p, 16, p, p, 16, p, 4, 4, 16, p, 0, 3, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8(p, 16, p, p, 16, p, 4, 4, 16, p, 3, 4, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8(p, 16, p, p, 16, p, 0, 4, 16, p, 0, 4, None) == 0
    assert h.b200moe_matmul_fp8_experts(p, 16, p, 4, p, 16, p, 0, p, p, 1, 4, 16, p, 0, 4, 0, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8_experts(p, 16, p, 4, p, 16, p, 2, p, p, 1025, 4, 16, p, 0, 4, 0, None) == L.ERR_LIMIT
    assert h.b200moe_matmul_fp8_experts(p, 16, p, 4, p, 16, p, 2, None, p, 1, 4, 16, p, 0, 4, 0, None) == L.ERR_ARG
    assert h.b200moe_matmul_fp8_experts(p, 16, p, 4, p, 16, p, 2, p, p, 0, 4, 16, p, 0, 4, 0, None) == 0      # no runs, nothing to zero


def test_calls_go_to_the_tensors_device(monkeypatch):
    """A call on a device that is not the current one makes it current for the launch, and takes that device's current stream."""
    import contextlib
    import sm120fp4_b200._lib as L
    here, seen = [0], []

    @contextlib.contextmanager
    def guard(device):
        before, here[0] = here[0], device.index
        yield
        here[0] = before
    monkeypatch.setattr(torch.cuda, "device", guard)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: here[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    fn = lambda *args: seen.append((here[0], *args)) or 0
    L.call(torch.device("cuda", 0), "x", fn, 1)
    L.call(torch.device("cuda", 3), "x", fn, 2)
    assert seen == [(0, 1, 100), (3, 2, 103)] and here == [0]
    with pytest.raises(L.B200MoEError):
        L.call(torch.device("cuda", 3), "x", lambda *args: L.ERR_ARG)
    a, b = torch.zeros(1), torch.zeros(1)
    with pytest.raises(RuntimeError, match="GPU"):
        L.one_device("x", a, b)
