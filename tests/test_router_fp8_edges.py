"""Corners of the router and FP8 operators that show without a GPU: what is refused, and before anything else."""
import re
from pathlib import Path

import pytest
import torch

import sm120fp4_b200 as pkg

fwd = torch.autograd.forward_ad


def test_forward_mode_is_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: pkg.top_k_gate(dual, 2), lambda: pkg.top_k_gate(dual, 2, renormalize=False), lambda: pkg.balance_loss(dual, ids)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="GPU"):      # plain tensors get as far as ever
            pkg.top_k_gate(x, 2)


def test_the_host_extension_has_no_cxx_library_of_its_own():
    """Two C++ libraries in a process share some of their objects and not others: numbers written to a stream end it."""
    import sm120fp4_b200._lib as L
    host = L.host()
    assert host is not L.NO_HOST
    with open(host.__file__, "rb") as f:
        assert b"St7codecvtIDsc" not in f.read()      # (a part of the library that nothing here names)


def test_fp8_calls_refuse_inputs_that_ask_for_a_derivative():
    """Outputs without a history would read as a derivative of zero."""
    codes = lambda *shape: torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    a, sa, w, sw, we, swe = codes(4, 256), torch.ones(4, 2), codes(32, 256), torch.ones(1, 2), codes(3, 32, 256), torch.ones(3, 1, 2)
    experts, offsets = torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    calls = [(pkg.quantize_fp8, [torch.zeros(4, 8)], [0]), (pkg.quantize_fp8_weight, [torch.zeros(4, 8)], [0]), (pkg.quantize_fp8_weight, [torch.zeros(2, 4, 8)], [0]),
             (pkg.matmul_fp8, [a, sa, w, sw], [1, 3]), (pkg.matmul_fp8_experts, [a, sa, we, swe, experts, offsets], [1, 3])]
    for call, args, floats in calls:
        for i in floats:
            asked = [t.clone().requires_grad_(True) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="no derivative"):
                call(*asked)
            with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):      # gets as far as ever
                call(*asked)
            with fwd.dual_level(), pytest.raises(RuntimeError, match="no derivative"):
                call(*[fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)])
    for call, args in ((pkg.matmul_fp8, (a, sa, w, sw)), (pkg.matmul_fp8_experts, (a, sa, we, swe, experts, offsets))):
        with pytest.raises(RuntimeError, match="no derivative"):
            call(*args, out=torch.zeros(4, 32, requires_grad=True))


def test_instructions_of_a_whole_warp_stay_where_they_are_called():
    """An asm statement that is not volatile may be moved into a branch that uses its result, where not all lanes are."""
    csrc = Path(pkg.__path__[0]) / "csrc"
    for f in sorted(csrc.glob("*.cu*")):
        for statement in re.findall(r"\basm\s*\([^;]*", f.read_text()):      # (up to the first semicolon: the instruction)
            assert not re.search(r"\b(redux|shfl|vote|match|bar|barrier|elect)\.", statement), f"{f.name}: {statement}"


def test_a_capture_that_cannot_be_checked_is_refused(monkeypatch):
    """Without the host extension nobody sees whether an eager graph of the same leaf is alive, beside which a captured backward pass ends the process."""
    import contextlib
    import sm120fp4_b200._lib as L
    from sm120fp4_b200 import gate
    monkeypatch.setattr(L, "_host", L.NO_HOST)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    capturing = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: bool(capturing))
    leaf = torch.zeros(4, 8, requires_grad=True)
    gate._check_capture(leaf, "x")
    capturing.append(1)
    with pytest.raises(RuntimeError, match="without the host extension"):
        gate._check_capture(leaf, "x")
    gate._check_capture(leaf * 1.0, "x")
    gate._check_capture(leaf.detach(), "x")
    with torch.no_grad():
        gate._check_capture(leaf, "x")


def test_more_pairs_than_a_count_holds_are_refused():
    """Counts are of 32 bits: 2^31 pairs of one expert would come out negative."""
    import sm120fp4_b200._lib as L
    tokens, h, p = 1 << 29, L.lib(), 4096      # (an address that is never read)
    x, ids = torch.zeros(1, 8).expand(tokens, 8), torch.zeros(1, 4, dtype=torch.int32).expand(tokens, 4)
    with pytest.raises(ValueError, match="pairs"):
        pkg.balance_loss(x, ids)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.balance_loss(x[:-1], ids[:-1])
    assert h.b200moe_balance_loss(p, 0, 8, tokens, 8, p, 4, p, p, p, p, 1 << 30, None) == L.ERR_LIMIT
    assert h.b200moe_balance_backward(p, p, 0, 8, tokens, 8, p, 4, p, p, p, None) == L.ERR_LIMIT
    assert h.b200moe_balance_loss(p, 0, 8, tokens - 1, 8, p, 4, p, p, p, p, 3, None) == L.ERR_WORKSPACE


def test_status_of_a_device_that_is_no_gpu_is_refused():
    """It would have been that of the current GPU, and its flag cleared."""
    for device in ("cpu", torch.device("meta")):
        with pytest.raises(ValueError, match="GPU"):
            pkg.matmul_fp8_status(device)


def test_tables_and_sums_off_4_bytes_are_refused():
    """Every pointer to words, one at a time; the kernels would fault on it. (Addresses are never read: a call that is not refused cannot run here.)"""
    import sm120fp4_b200._lib as L
    if torch.cuda.is_available():
        pytest.skip("calls with addresses that are none, refused or not")
    h, p = L.lib(), 4096
    calls = [(h.b200moe_gate, [p, 0, 8, 4, 8, 2, 1, p, p, None], [7, 8]), (h.b200moe_gate_backward, [p, p, p, p, 0, 8, 4, 8, 2, 0, p, None], [0, 1, 2]),
             (h.b200moe_balance_loss, [p, 0, 8, 4, 8, p, 2, p, p, p, p, 1 << 20, None], [5, 7, 8, 9, 10]), (h.b200moe_balance_backward, [p, p, 0, 8, 4, 8, p, 2, p, p, p, None], [0, 6, 8, 9]),
             (h.b200moe_quantize_fp8, [p, 0, 16, 4, p, 4, 16, p, 16, p, None, 0, None], [4, 9]), (h.b200moe_quantize_fp8_blocks, [p, 0, 1, 4, 16, p, 16, p, None], [7]),
             (h.b200moe_matmul_fp8, [p, 16, p, p, 16, p, 4, 4, 16, p, 0, 4, None], [2, 5]),
             (h.b200moe_matmul_fp8_experts, [p, 16, p, 4, p, 16, p, 2, p, p, 1, 4, 16, p, 0, 4, 0, None], [2, 6, 8, 9]),
             (h.b200moe_matmul_fp8_probe, [p, 16, p, 4, p, 16, p, 2, p, p, 1, 4, 16, p, 0, 4, 0, None], [2, 6, 8, 9])]
    for call, args, words in calls:
        assert call(*args) in (L.ERR_CUDA, L.ERR_DEVICE)      # as it stands it gets as far as the device that is not here
        for i in words:
            assert call(*args[:i], p + 2, *args[i + 1:]) == L.ERR_ARG, f"{call.__name__}, argument {i}"


def test_route_runs_on_the_gpu_that_its_tables_are_on(monkeypatch):
    """Tables on the host reached the kernels, those of another GPU the current one's stream."""
    import contextlib
    from types import SimpleNamespace
    import sm120fp4_b200._lib as L
    from sm120fp4_b200 import router
    ids, tables = torch.zeros(4, 2, dtype=torch.int32), [torch.zeros(n, dtype=torch.int32) for n in (8, 9, 8)]
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.route(ids, 8, *tables)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.route_tables(ids, 8)
    here, seen = [0], []

    @contextlib.contextmanager
    def guard(device):
        before, here[0] = here[0], device.index
        yield
        here[0] = before
    monkeypatch.setattr(torch.cuda, "device", guard)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: here[0], raising=False)
    monkeypatch.setattr(L, "stream_ptr", lambda: 100 + here[0])
    monkeypatch.setattr(router, "_workspace", lambda device, stream, n: torch.zeros(n, dtype=torch.uint8))
    monkeypatch.setattr(L, "lib", lambda: SimpleNamespace(b200moe_route_workspace_bytes=lambda p, e: 64, b200moe_route=lambda *args: seen.append((here[0], args[1:4], args[-1])) or 0))
    for index in (0, 3):
        monkeypatch.setattr(torch.Tensor, "device", property(lambda self: torch.device("cuda", index)))
        monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
        pkg.route(ids, 8, *tables)
    assert seen == [(0, (8, 8, 8), 100), (3, (8, 8, 8), 103)] and here == [0]
    with pytest.raises(ValueError, match="contiguous"):
        pkg.route(ids, 8, torch.zeros(16, dtype=torch.int32)[::2], *tables[1:])
