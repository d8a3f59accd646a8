"""The native host side of the router and FP8 operators (csrc/host.cpp) against the general path: same outputs and gradients, and None - so that the general path runs, with
its checks and errors - for everything that is not plain. Then what belongs to either: graphs of autograd, captures, places beyond 32 bits."""
import math

import pytest
import torch

import sm120fp4_b200 as pkg
from sm120fp4_b200 import _lib

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def general(monkeypatch, fn):
    with monkeypatch.context() as m:
        m.setattr(_lib, "_host", _lib.NO_HOST)
        return fn()


def same(a, b):
    assert len(a) == len(b)
    for s, t in zip(a, b):
        assert s.shape == t.shape and s.stride() == t.stride() and s.dtype == t.dtype and s.device == t.device and s.requires_grad == t.requires_grad
        s, t = s.detach(), t.detach()
        assert torch.equal(s.contiguous().view(torch.uint8) if s.dim() else s, t.contiguous().view(torch.uint8) if t.dim() else t)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_router_outputs_and_gradients(monkeypatch, dtype):
    big = randn(40, 160, seed=3).to(dtype)
    for x in (big, big[:, :60], big[::2, 1:34], big[:1]):
        for renormalize in (True, False):
            assert _lib.host().top_k_gate(x, 4, renormalize) is not None
            same(pkg.top_k_gate(x, 4, renormalize), general(monkeypatch, lambda: pkg.top_k_gate(x, 4, renormalize)))

            def step():
                leaf = x.detach().clone().requires_grad_(True)
                w, ids = pkg.top_k_gate(leaf, 4, renormalize)
                loss, counts = pkg.balance_loss(leaf, ids)
                g = torch.autograd.grad([w, loss], leaf, [randn(*w.shape, seed=1), torch.tensor(0.5, device="cuda")])
                return w, ids, loss, counts, *g
            same(step(), general(monkeypatch, step))
        ids = pkg.top_k_gate(x, 4)[1]
        assert _lib.host().balance_loss(x, ids) is not None
        same(pkg.balance_loss(x, ids), general(monkeypatch, lambda: pkg.balance_loss(x, ids)))


def test_fp8_outputs(monkeypatch):
    for m, k in [(1, 100), (33, 256), (1200, 1040)]:
        x = randn(m, k, seed=k).bfloat16()
        src = torch.randint(-1, m, (m * 9,), generator=torch.Generator().manual_seed(m)).int().cuda()
        for s in (None, src):
            assert _lib.host().quantize_fp8(x, s) is not None
            same(pkg.quantize_fp8(x, src_row=s), general(monkeypatch, lambda: pkg.quantize_fp8(x, src_row=s)))
        a, sa = pkg.quantize_fp8(x)
        for v in (randn(3, 200, k, seed=1), randn(131, k, seed=2).half(), randn(1, 1, k, seed=3).bfloat16()):
            assert _lib.host().quantize_fp8_weight(v) is not None
            same(pkg.quantize_fp8_weight(v), general(monkeypatch, lambda: pkg.quantize_fp8_weight(v)))
        w, sw = pkg.quantize_fp8_weight(randn(3, 200, k, seed=1))
        for dtype in (torch.bfloat16, torch.float32):
            assert _lib.host().matmul_fp8(a, sa, w[0], sw[0], dtype) is not None
            same([pkg.matmul_fp8(a, sa, w[0], sw[0], out_dtype=dtype)], [general(monkeypatch, lambda: pkg.matmul_fp8(a, sa, w[0], sw[0], out_dtype=dtype))])
        experts, offsets = torch.tensor([2, 0], dtype=torch.int32, device="cuda"), torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda")
        assert _lib.host().matmul_fp8_experts(a, sa, w, sw, experts, offsets, torch.bfloat16) is not None
        same([pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets)], [general(monkeypatch, lambda: pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets))])


def test_what_is_left_to_the_general_path():
    h = _lib.host()
    x, ids = randn(8, 64), torch.zeros(8, 2, dtype=torch.int32, device="cuda")
    for v in (x.t(), x[:0], x[0], x.double(), x.cpu(), x[None], x.to_sparse(), randn(2, 513), None, 3):
        assert h.top_k_gate(v, 2, True) is None and h.balance_loss(v, ids) is None
    assert h.top_k_gate(x, 0, True) is None and h.top_k_gate(x, 65, True) is None and h.top_k_gate(x, 2.0, True) is None and h.top_k_gate(x, 2, 1) is None and h.top_k_gate(x, 2) is None
    assert h.top_k_gate(x, 1 << 70, True) is None
    for i in (ids.long(), ids[:4], ids.cpu(), ids[0], ids.t(), torch.zeros(8, 33, dtype=torch.int32, device="cuda"), None):
        assert h.balance_loss(x, i) is None
    for v in (x.t(), x[:0], x[0], x.double(), x.cpu(), None):
        assert h.quantize_fp8(v, None) is None and h.quantize_fp8_weight(v) is None
    assert h.quantize_fp8_weight(x[:, :32]) is None and h.quantize_fp8_weight(x[None, None]) is None
    for s in (ids, ids[:, 0], ids[0].long(), ids[0].cpu(), 3):
        assert h.quantize_fp8(x, s) is None
    a, sa = pkg.quantize_fp8(randn(4, 256))
    w, sw = pkg.quantize_fp8_weight(randn(32, 256))
    good = (a, sa, w, sw, torch.bfloat16)
    assert h.matmul_fp8(*good) is not None
    for at, bad in [(0, a.view(torch.uint8)), (0, a[:0]), (0, a[:, 8:]), (0, a.t()), (1, sa.half()), (1, sa[:2]), (1, sa.cpu()), (2, w[:, :128]), (2, w[None]), (3, sw[:, :1]), (4, torch.float64), (4, "bf16")]:
        assert h.matmul_fp8(*good[:at], bad, *good[at + 1:]) is None
    from torch.overrides import TorchFunctionMode

    class Seen(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Seen():
        assert h.top_k_gate(x, 2, True) is None and h.balance_loss(x, ids) is None and h.quantize_fp8(x, None) is None and h.matmul_fp8(*good) is None
    with pytest.raises(TypeError):
        h.bind_ops(1, 2)


def test_gradients_are_taken_once(monkeypatch):
    for run in (lambda f: f(), lambda f: general(monkeypatch, f)):
        def twice():
            x = randn(5, 16, seed=1).requires_grad_(True)
            w, ids = pkg.top_k_gate(x, 3)
            loss, _ = pkg.balance_loss(x, ids)
            for out in (w.square().sum(), loss):
                g, = torch.autograd.grad(out, x, create_graph=True)
                assert bool(torch.isfinite(g).all())
                with pytest.raises(RuntimeError, match="once"):
                    g.sum().backward()
        run(twice)


def test_autograd_manners(monkeypatch):
    for run in (lambda f: f(), lambda f: general(monkeypatch, f)):
        def manners():
            x = randn(6, 32, seed=2).requires_grad_(True)
            with torch.no_grad():
                assert not pkg.top_k_gate(x, 2)[0].requires_grad
            with torch.inference_mode():
                w, ids = pkg.top_k_gate(x, 2)
                assert w.is_inference() and pkg.balance_loss(x, ids)[0].is_inference()
            w, ids = pkg.top_k_gate(x, 2)
            loss, counts = pkg.balance_loss(x, ids)
            assert w.requires_grad and loss.requires_grad and not ids.requires_grad and not counts.requires_grad
            y = x * 1.0      # not a leaf; changed after it was saved
            loss, _ = pkg.balance_loss(y, ids)
            with torch.no_grad():
                y.mul_(2)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
            w = pkg.top_k_gate(x, 2, renormalize=False)[0]
            w.sum().backward()
            with pytest.raises(RuntimeError, match="second time"):
                w.sum().backward()
            assert w.grad_fn is not None and x.grad.shape == x.shape
            with torch.autograd.forward_ad.dual_level():
                dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
                assert _lib.host().top_k_gate(dual, 2, True) is None and _lib.host().balance_loss(dual, ids) is None
            seen = []
            with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
                pkg.top_k_gate(x, 2, renormalize=False)[0].sum().backward()
            assert len(seen) >= 3
        run(manners)


def test_capture_beside_a_live_graph_is_refused():
    """What the engine would do with it ends the process, so the call says no."""
    x = randn(20, 16, seed=5).requires_grad_(True)
    ids = pkg.top_k_gate(x.detach(), 2)[1]
    alive = pkg.balance_loss(x, ids)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    for call in (lambda: pkg.top_k_gate(x, 2), lambda: pkg.balance_loss(x, ids)):
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(graph):
                call()
        graph = torch.cuda.CUDAGraph()
    del alive
    with torch.cuda.graph(graph):
        loss, _ = pkg.balance_loss(x, ids)
        g, = torch.autograd.grad(loss, x)
    graph.replay()
    want, = torch.autograd.grad(pkg.balance_loss(x, ids)[0], x)
    assert torch.equal(g, want)


def test_two_captures_of_the_same_call():
    """Graphs share nothing: replayed side by side on two streams, each gives its own inputs' outputs."""
    xs = [randn(3000, 1024, seed=i).bfloat16() for i in range(2)]
    logits = [randn(3000, 64, seed=10 + i) for i in range(2)]
    w, sw = pkg.quantize_fp8_weight(randn(64, 256, 1024, seed=4))

    def step(x, logit):
        weights, ids = pkg.top_k_gate(logit, 4)
        loss, counts = pkg.balance_loss(logit, ids)
        experts, offsets, pairs = pkg.route_tables(ids, 64)
        q, s = pkg.quantize_fp8(x, src_row=pairs // 4)
        return weights, loss, counts, experts, offsets, pairs, s, pkg.matmul_fp8_experts(q, s, w, sw, experts, offsets)

    want = [step(x, l) for x, l in zip(xs, logits)]
    want = [[t.clone() for t in o] for o in want]
    graphs, outs = [], []
    for x, l in zip(xs, logits):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x, l))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, want):
            assert [bool(torch.equal(a, b)) for a, b in zip(o, e)] == [True] * len(e)
    pkg.matmul_fp8_status()
    pkg.matmul_fp8_status("cuda")
    pkg.matmul_fp8_status(0)


def test_a_stream_of_its_own():
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        x = randn(50, 128, seed=1).requires_grad_(True)
        w, ids = pkg.top_k_gate(x, 8)
        loss, counts = pkg.balance_loss(x, ids)
    torch.cuda.current_stream().wait_stream(st)
    (w.sum() + loss).backward()      # the gradient runs on the forward's stream, and this one waits for it
    y = x.detach().clone().requires_grad_(True)
    w2, ids2 = pkg.top_k_gate(y, 8)
    (w2.sum() + pkg.balance_loss(y, ids2)[0]).backward()
    assert torch.equal(x.grad, y.grad) and torch.equal(ids, ids2)


def test_places_beyond_32_bits():
    """Inputs, codes and outputs of more than 2^32 bytes and 2^31 values: the last rows are right."""
    rows, k = 70000, 32768
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    tail = randn(5, k, seed=1).bfloat16()
    x[-5:] = tail
    q, s = pkg.quantize_fp8(x)
    tq, ts = pkg.quantize_fp8(tail)
    assert torch.equal(q[-5:].view(torch.uint8), tq.view(torch.uint8)) and torch.equal(s[-5:], ts) and int(q[-6].view(torch.uint8).max()) == 0
    w, sw = pkg.quantize_fp8_weight(randn(16, k, seed=2))
    got = pkg.matmul_fp8(q, s, w, sw)
    want = pkg.matmul_fp8(tq, ts, w, sw)      # (another form: other orders of the sums)
    assert bool(((got[-5:].float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-3 * float(want.float().abs().max())).all())
    assert float(got[:-5].float().abs().max()) == 0.0
    del x, q, s
    a, sa = pkg.quantize_fp8(randn(rows, 128, seed=3))
    w, sw = pkg.quantize_fp8_weight(randn(k, 128, seed=4))
    out = pkg.matmul_fp8(a, sa, w, sw)
    part = pkg.matmul_fp8(a[-300:], sa[-300:], w, sw)
    assert torch.equal(out[-300:], part)      # (the same form, one group: the same sums)
    del out
    stacked = torch.zeros(300, 4096, 2048, dtype=torch.bfloat16, device="cuda")
    stacked[-1] = randn(4096, 2048, seed=5).bfloat16()
    wq, ws = pkg.quantize_fp8_weight(stacked)
    lq, ls = pkg.quantize_fp8_weight(stacked[-1])
    assert torch.equal(wq[-1].view(torch.uint8), lq.view(torch.uint8)) and torch.equal(ws[-1], ls)
    a, sa = pkg.quantize_fp8(randn(40, 2048, seed=6))
    experts, offsets = torch.tensor([299], dtype=torch.int32, device="cuda"), torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    got = pkg.matmul_fp8_experts(a, sa, wq, ws, experts, offsets, out_dtype=torch.float32)
    want = pkg.matmul_fp8(a, sa, lq, ls, out_dtype=torch.float32)
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max()) * math.sqrt(2048)
    big = torch.full((5_000_000, 512), -1.0, dtype=torch.bfloat16, device="cuda")
    big[-1] = randn(512, seed=7).bfloat16()
    w1, ids = pkg.top_k_gate(big, 8)
    w2, ids2 = pkg.top_k_gate(big[-1:], 8)
    assert torch.equal(w1[-1:], w2) and torch.equal(ids[-1:], ids2)


def test_empty_source():
    q, s = pkg.quantize_fp8(torch.zeros(0, 256, device="cuda"), src_row=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert q.shape == (3, 256) and float(q.float().abs().max()) == 0.0 and float(s.abs().max()) == 0.0
    q, s = pkg.quantize_fp8(randn(4, 256), src_row=torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (0, 2)
