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


def test_fp8_calls_refuse_inputs_that_ask_for_a_derivative(path):
    x, w = randn(8, 256, seed=1), randn(32, 256, seed=2)
    a, sa = pkg.quantize_fp8(x)
    wq, sw = pkg.quantize_fp8_weight(w)
    ask = lambda t: t.clone().requires_grad_(True)
    refused = [lambda: pkg.quantize_fp8(ask(x)), lambda: pkg.quantize_fp8(x * ask(x)), lambda: pkg.quantize_fp8_weight(ask(w)), lambda: pkg.quantize_fp8_weight(torch.nn.Parameter(w)),
               lambda: pkg.matmul_fp8(a, ask(sa), wq, sw), lambda: pkg.matmul_fp8(a, sa, wq, ask(sw))]
    for call in refused:
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
        with torch.no_grad():
            out = call()
        assert not any(t.requires_grad for t in (out if type(out) is tuple else (out,)))
    with fwd.dual_level():
        for call in (lambda: pkg.quantize_fp8(fwd.make_dual(x, torch.ones_like(x))), lambda: pkg.matmul_fp8(a, fwd.make_dual(sa, torch.ones_like(sa)), wq, sw)):
            with pytest.raises(RuntimeError, match="no derivative"):
                call()
    with torch.inference_mode():
        assert same(pkg.quantize_fp8(ask(x))[0], a)


def test_saved_tensors_that_come_back_as_others(path):
    """Hooks on saved tensors may move and copy them: what comes back is looked at before its memory is read."""
    hooks = torch.autograd.graph.saved_tensors_hooks
    big = randn(12, 80, seed=3)

    def grads(pack, unpack, renormalize):
        x = big[:, 5:69].detach().clone().requires_grad_(True)
        with hooks(pack, unpack):
            w, ids = pkg.top_k_gate(x, 3, renormalize)
            loss = pkg.balance_loss(x, ids)[0]
        return torch.autograd.grad(w.square().sum(), x)[0], torch.autograd.grad(loss, x)[0]
    spread = lambda t: torch.stack([t, t], t.dim())[..., 0]      # the same values, apart in memory
    for renormalize in (True, False):
        want = grads(lambda t: t, lambda t: t, renormalize)
        for pack, unpack in ((lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t.clone(), spread), (lambda t: t.detach().clone(), lambda t: t.t().contiguous().t() if t.dim() == 2 else t),
                             (lambda t: -t if t.is_floating_point() else t.clone(), lambda t: torch._neg_view(t) if t.is_floating_point() else t)):
            for a, b in zip(grads(pack, unpack, renormalize), want):
                assert torch.equal(a, b)
        bad = [lambda t: t.cpu(), lambda t: t.double() if t.is_floating_point() else t.long(), lambda t: t[:1], lambda t: t[None], lambda t: t.bfloat16() if t.is_floating_point() else t.short()]
        for unpack in bad:
            x = big.clone().requires_grad_(True)
            with hooks(lambda t: t, unpack):
                w, ids = pkg.top_k_gate(x, 3, renormalize)
                loss = pkg.balance_loss(x, ids)[0]
            for out in (w.square().sum(), loss):
                with pytest.raises(RuntimeError, match="gave back"):
                    torch.autograd.grad(out, x)
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        x = big.clone().requires_grad_(True)
        pkg.top_k_gate(x, 3, False)[0].sum().backward()
    assert bool(torch.isfinite(x.grad).all())


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


def test_capture_beside_a_live_graph_is_refused_on_either_path(path):
    """Logits that the native side does not take as they are (here a matrix stored by columns) are looked at all the same."""
    x = randn(16, 20, seed=5).t().requires_grad_(True)
    assert x.is_leaf and x.stride(1) != 1
    ids = pkg.top_k_gate(x.detach(), 2)[1]
    alive = pkg.balance_loss(x, ids)[0]
    torch.cuda.synchronize()
    why = "still alive" if path == "native" else "without the host extension"
    for call in (lambda: pkg.top_k_gate(x, 2), lambda: pkg.balance_loss(x, ids)):
        with pytest.raises(RuntimeError, match=why):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive
    if path == "native":
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            g, = torch.autograd.grad(pkg.balance_loss(x, ids)[0], x)
        graph.replay()
        assert torch.equal(g, torch.autograd.grad(pkg.balance_loss(x, ids)[0], x)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,e,k", [(64, 8, 8), (4096, 64, 4), (4096, 60, 1), (2048, 512, 8), (6, 1, 1)])
def test_balance_gradient_where_experts_are_used_almost_evenly(t, e, k, dtype):
    """With f_e = 1/E + d_e the gradient is g E/T p_e (d_e - sum p d): it is 0 where all d are, and its roundings count against d, not against f. Per term: d is a quotient of
    whole numbers (5 roundings: two of the numerator, 1/sum n, that over E, the product), p as in a softmax (a numerator 2.25 |x - m| + 4 roundings, twice, a sum of V + 5 and a quotient), the sum over
    E of V + 5 additions more, and six products and differences. |x - m| <= 8 here."""
    values = next(v for v in (1, 2, 4, 8, 16) if e <= 32 * v)
    x = (torch.rand(t, e, generator=torch.Generator().manual_seed(e)) * 8 - 4).to(dtype).cuda()
    ids = (torch.arange(t * k) % e).int().view(t, k).cuda()
    for moved in (0, 1, 3):
        if e == 1 and moved:
            continue
        ids.view(-1)[:moved] = e - 1
        counts = torch.bincount(ids.view(-1).long(), minlength=e)
        d = (counts.double() * e - t * k) / (t * k * e)
        leaf = x.clone().requires_grad_(True)
        loss, got_counts = pkg.balance_loss(leaf, ids)
        assert torch.equal(got_counts, counts.int())
        g, = torch.autograd.grad(loss, leaf)
        p = torch.softmax(x.double(), 1)
        want, size = e / t * p * (d - (p @ d)[:, None]), e / t * p * (d.abs() + (p @ d.abs())[:, None])
        rel_p = 2 * (2.25 * 8 + 4) + values + 6
        tol = 2.0 ** -24 * (5 + 2 * rel_p + values + 5 + 6) * size + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -126
        assert bool(((g.double() - want).abs() <= tol).all())
        if int(counts.min()) == int(counts.max()):
            assert float(g.abs().max()) == 0.0


# ---------------------------------------------------------------------------------------------------- tensors that are not stored as they read

def test_negated_views(path):
    """torch keeps the sign of some views (the imaginary part of a conjugate) as a mark beside the values."""
    x, ids = randn(20, 64, seed=1), torch.randint(0, 64, (20, 2), generator=torch.Generator().manual_seed(2)).int().cuda()
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        neg = torch._neg_view(y)
        assert neg.is_neg()
        for renormalize in (True, False):
            for a, b in zip(pkg.top_k_gate(neg, 4, renormalize), pkg.top_k_gate(-y, 4, renormalize)):
                assert torch.equal(a, b)
        for a, b in zip(pkg.balance_loss(neg, ids), pkg.balance_loss(-y, ids)):
            assert torch.equal(a, b)
        for call in (pkg.quantize_fp8, pkg.quantize_fp8_weight):
            for a, b in zip(call(neg), call(-y)):
                assert same(a, b)
    a, sa = pkg.quantize_fp8(randn(20, 256, seed=3))
    w, sw = pkg.quantize_fp8_weight(randn(40, 256, seed=4))
    for bad in (lambda: pkg.matmul_fp8(torch._neg_view(a), sa, w, sw), lambda: pkg.matmul_fp8(a, sa, torch._neg_view(w), sw),
                lambda: pkg.matmul_fp8(a, sa, w, sw, out=torch._neg_view(torch.zeros(20, 40, device="cuda")))):
        with pytest.raises((RuntimeError, ValueError)):      # codes cannot be negated, an output would read as its negative
            bad()
    assert torch.equal(pkg.matmul_fp8(a, torch._neg_view(sa), w, sw), pkg.matmul_fp8(a, -sa, w, sw))
    assert torch.equal(pkg.matmul_fp8(a, sa, w, torch._neg_view(sw)), pkg.matmul_fp8(a, sa, w, -sw))


def test_gradients_that_come_as_negated_views(path):
    """What arrives where weights are the imaginary part of a number whose conjugate is used."""
    logits, c = randn(20, 16, seed=1), torch.complex(randn(20, 4, seed=2), randn(20, 4, seed=3))
    for renormalize in (True, False):
        def grad_of(gate):
            x, seen = logits.clone().requires_grad_(True), []
            w = gate(x)
            w.register_hook(lambda g: seen.append(g.is_neg()) and None)
            (torch.complex(torch.ones_like(w), w).conj() * c).real.sum().backward()
            return x.grad, seen

        def plain(x):
            w = torch.softmax(x.double(), 1).gather(1, pkg.top_k_gate(logits, 4)[1].long())
            return (w / w.sum(1, keepdim=True) if renormalize else w).float()
        got, seen = grad_of(lambda x: pkg.top_k_gate(x, 4, renormalize)[0])
        assert seen == [True]
        want = grad_of(plain)[0]
        # a gradient is a few products and sums of terms that are at most |g| <= 4 in size, each step off by 2^-24 of them: 2^-16 is far above, a wrong sign far above that
        assert float((got - want).abs().max()) <= 2.0 ** -16 and float(want.abs().max()) > 2.0 ** -4
        x = logits.clone().requires_grad_(True)
        loss = pkg.balance_loss(x, pkg.top_k_gate(logits, 4)[1])[0]
        g1, = torch.autograd.grad(loss, x, torch._neg_view(torch.ones_like(loss)), retain_graph=True)
        g2, = torch.autograd.grad(loss, x, torch.full_like(loss, -1.0))
        assert torch.equal(g1, g2) and float(g1.abs().max()) > 0


def test_gradients_that_come_without_memory(path):
    """The gradient of sgn is a tensor of zeros that has no memory."""
    for renormalize in (True, False):
        x = randn(20, 16, seed=1).requires_grad_(True)
        torch.sgn(pkg.top_k_gate(x, 4, renormalize)[0]).sum().backward()
        assert float(x.grad.abs().max()) == 0.0
    x = randn(20, 16, seed=1).requires_grad_(True)
    torch.sgn(pkg.balance_loss(x, pkg.top_k_gate(x.detach(), 4)[1])[0]).backward()
    assert float(x.grad.abs().max()) == 0.0


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


@pytest.mark.parametrize("n", [1, 7, 8, 130, 1408, 5003])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_outside_every_run_are_zeros(n, dtype):
    """Before, between (experts that are not there) and behind the runs, with rows on 16 bytes and off them, whatever memory held."""
    p, k = 700, 256
    a, sa = pkg.quantize_fp8(randn(p, k, seed=1))
    w, sw = pkg.quantize_fp8_weight(randn(3, n, k, seed=2))
    experts = torch.tensor([2, -1, 0, 7, 1], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([5, 40, 290, 291, 400, 410], dtype=torch.int32, device="cuda")
    kept = torch.full((p, n), 3.0, dtype=dtype, device="cuda")
    pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out=kept)
    dirty = torch.full((p, n), 7.0, dtype=dtype, device="cuda")      # (the next new tensor of this size is that memory)
    del dirty
    got = pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out_dtype=dtype)
    for s in (slice(0, 5), slice(40, 290), slice(291, 400), slice(410, p)):
        assert float(got[s].abs().max()) == 0.0 and bool((kept[s] == 3).all())
    for s in (slice(5, 40), slice(290, 291), slice(400, 410)):
        assert torch.equal(got[s], kept[s])


def test_rows_outside_every_run_beyond_31_bits():
    """A row of 2^29 values of 32 bits is 2^31 bytes."""
    n = 1 << 29
    a, sa = pkg.quantize_fp8(randn(2, 16, seed=1))
    w, sw = torch.zeros(1, n, 16, dtype=torch.uint8, device="cuda").view(FP8), torch.ones(1, n // 128, 1, device="cuda")
    w.view(torch.uint8)[0, -1] = 0x38      # ones
    dirty = torch.full((2, n), 7.0, device="cuda")
    del dirty
    got = pkg.matmul_fp8_experts(a, sa, w, sw, torch.tensor([0], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), out_dtype=torch.float32)
    assert float(got[1].abs().max()) == 0.0 and float(got[0, :-1].abs().max()) == 0.0
    want = float((a[0].double() * sa[0].double()).sum())      # 16 exact products, summed in fp32, times a scale
    assert abs(float(got[0, -1]) - want) <= 17 * 2.0 ** -23 * float((a[0].double() * sa[0].double()).abs().sum())


def test_rows_outside_every_run_take_the_time_of_their_bytes():
    """Half of a prompt's pairs are padding. The rows that are zeroed are 100 MB, 16 us at the rate of memory; a single SM would need more than a millisecond."""
    p, n, k = 32768, 1536, 256
    a, sa = pkg.quantize_fp8(randn(p, k, seed=1))
    w, sw = pkg.quantize_fp8_weight(randn(16, n, k, seed=2))
    experts, offsets = torch.arange(16, dtype=torch.int32, device="cuda"), (torch.arange(17, device="cuda") * (p // 32)).int()
    out = torch.empty(p, n, dtype=torch.bfloat16, device="cuda")
    left = best_us(lambda: pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out=out))
    zeroed = best_us(lambda: pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets))
    assert zeroed <= left + 200, f"{left:.0f} us without the zeros, {zeroed:.0f} with them"


# ---------------------------------------------------------------------------------------------------- padded batches

@pytest.mark.parametrize("tokens,k,e,static", [(3, 2, 8, False), (40, 4, 16, False), (512, 8, 256, False), (513, 8, 256, False), (700, 8, 300, False), (5000, 4, 60, False), (20000, 8, 128, False),
                                               (3, 2, 8, True), (513, 8, 256, True), (8192, 8, 256, True)])
def test_pairs_behind_the_last_run(tokens, k, e, static):
    """Empty slots and ids that are not there stand in no run; what is behind the last one is -1, not what memory held."""
    p = tokens * k
    for empty in (0.0, 0.4, 1.0):
        g = torch.Generator().manual_seed(tokens)
        ids = torch.randint(0, e, (p,), generator=g).int()
        ids[torch.rand(p, generator=g) < empty] = -1
        if empty == 0.4:
            ids[1] = e + 3
        umax = min(e, p)
        ex, off, pairs = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (umax, umax + 1, p))
        dev = ids.cuda()
        if static:
            L.check(L.lib().b200moe_route_static(L.ptr(dev), p, e, umax, L.ptr(ex), L.ptr(off), L.ptr(pairs), L.stream_ptr()))
        else:
            pkg.route(dev, e, ex, off, pairs)
        used = (ids >= 0) & (ids < e)
        routed = int(used.sum())
        order = torch.where(used, ids, torch.tensor(e)).sort(stable=True)[1].int()
        assert int(off[-1]) == routed and torch.equal(pairs.cpu()[:routed], order[:routed]) and bool((pairs[routed:] == -1).all())
        if not static:
            assert torch.equal(pkg.route_tables(dev, e)[2], pairs)


def test_tables_with_room_for_fewer_experts_than_are_touched():
    ids = torch.arange(64, dtype=torch.int32, device="cuda").repeat(100)
    ids[::3] = -1
    for p in (600, 6400):
        ex, off, pairs = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (10, 11, p))
        pkg.route(ids[:p], 64, ex, off, pairs)
        routed = int((ids[:p] >= 0).sum())
        assert ex.tolist() == list(range(10)) and bool((pairs[:routed] >= 0).all()) and bool((pairs[routed:] == -1).all())


@pytest.mark.parametrize("t,live,k,inner", [(40, 25, 4, 256), (3000, 1801, 2, 256), (3000, 1801, 8, 1024), (4096, 1, 8, 512)])
def test_padded_batch_is_the_same_from_call_to_call(t, live, k, inner):
    """The documented way from ids to codes: rows behind the last run are zeros, codes and scales alike, whatever memory held."""
    x, logit = randn(t, inner, seed=1).bfloat16(), randn(t, 32, seed=2)
    logit[live:] = -math.inf
    ids = pkg.top_k_gate(logit, k)[1]
    for poison in (0, 5, 1 << 29):
        dirty = [torch.full((t * k,), poison, dtype=torch.int32, device="cuda") for _ in range(4)]
        del dirty
        experts, offsets, pairs = pkg.route_tables(ids, 32)
        q, s = pkg.quantize_fp8(x, src_row=pairs // k)
        assert int(offsets[-1]) == live * k
        assert int(q.view(torch.uint8)[live * k:].max()) == 0 and float(s[live * k:].abs().max()) == 0.0
        rq, rs = pkg.quantize_fp8(x[(pairs[:live * k] // k).long()])
        assert same(q[:live * k].contiguous(), rq.contiguous()) and torch.equal(s[:live * k], rs)


# ---------------------------------------------------------------------------------------------------- rows that are asked for very often

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_that_are_asked_for_very_often(dtype):
    """One row for half of the destinations, a few rows for all of them, counts that differ, and one row in all."""
    x = randn(4096, 1056, seed=1).to(dtype)
    q, s = pkg.quantize_fp8(x)
    g = torch.Generator().manual_seed(3)
    src = torch.arange(32768) // 8
    half = src.clone()
    half[16384:] = 11
    for src in (half, half.flip(0), torch.full((32768,), 4095), src % 3, torch.randint(0, 4096, (32768,), generator=g), torch.randint(-500, 5000, (30001,), generator=g),
                (torch.rand(32768, generator=g) ** 4 * 4096).long(), torch.arange(32768) % 4096):
        src = src.int().cuda()
        inside = (src >= 0) & (src < 4096)
        at = src.clamp(0, 4095).long()
        gq, gs = pkg.quantize_fp8(x, src_row=src)
        want = torch.where(inside[:, None], q.view(torch.uint8)[at], torch.zeros((), dtype=torch.uint8, device="cuda"))
        assert torch.equal(gq.view(torch.uint8), want) and torch.equal(gs, torch.where(inside[:, None], s[at], torch.zeros((), device="cuda")))
    one = x[:1]
    gq, gs = pkg.quantize_fp8(one, src_row=torch.zeros(20000, dtype=torch.int32, device="cuda"))
    assert torch.equal(gq.view(torch.uint8), q[:1].view(torch.uint8).expand(20000, -1)) and torch.equal(gs, s[:1].expand(20000, -1))


def test_a_row_that_is_asked_for_very_often_takes_the_time_of_its_bytes():
    """16384 destinations of one row are 46 MB of codes, 7 us at the rate of memory; one after the other, 80 ns each, they would take more than a millisecond."""
    x = randn(4096, 2816, seed=1).bfloat16()
    even = (torch.arange(32768, device="cuda") // 8).int()
    skewed = even.clone()
    skewed[16384:] = 11
    usual = best_us(lambda: pkg.quantize_fp8(x, src_row=even))
    often = best_us(lambda: pkg.quantize_fp8(x, src_row=skewed))
    one = best_us(lambda: pkg.quantize_fp8(x[:2], src_row=skewed.clamp(max=1)))
    assert often <= usual + 400 and one <= usual + 400, f"{usual:.0f} us evenly, {often:.0f} with one row for half of them, {one:.0f} with two rows in all"


# ---------------------------------------------------------------------------------------------------- waits that run out

FORMS = [(1, 1000, 512, 0), (1, 2048, 2048, 0), (40, 20000, 2048, 0), (100, 2048, 2048, 0), (16, 700, 1024, 8), (1000, 1408, 2816, 8), (512, 4096, 4096, 0), (6000, 1000, 1024, 8)]


@pytest.mark.parametrize("m,n,k,experts,give_up", [(*f, g) for f in FORMS for g in (1, 2, 4, 8, 15)] + [(*FORMS[f], 16 + g) for f in (1, 6, 7) for g in (1, 2, 4, 8, 15)])
def test_waits_that_run_out(m, n, k, experts, give_up):
    """One side of a product's pipeline stops where it would first have to wait (the copies', the products', the scales', the sums', all; in all blocks, or in the first of a
    cluster): the others stop after it, the call ends, its status says so once, and the next call is right. Few rows whole and split over clusters, tiles of 64 and 128 rows,
    experts' runs of few rows and of many, pairs of blocks for one matrix and for several."""
    import time
    a, sa = pkg.quantize_fp8(randn(m, k, seed=1))
    w, sw = pkg.quantize_fp8_weight(randn(max(experts, 1), n, k, seed=2))
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    tables = (torch.arange(experts, dtype=torch.int32, device="cuda"), (torch.arange(experts + 1, device="cuda") * (m // max(experts, 1))).int()) if experts else (None, None)

    def call(side):
        L.check(L.lib().b200moe_matmul_fp8_probe(a.data_ptr(), a.stride(0) if m > 1 else k, sa.data_ptr(), m, w.data_ptr(), w.stride(1), sw.data_ptr(), w.shape[0], L.ptr(tables[0]),
                                                 L.ptr(tables[1]), experts, n, k, out.data_ptr(), 0, n, side, L.stream_ptr()), "probe")
    pkg.matmul_fp8_status()
    call(0)
    pkg.matmul_fp8_status()
    want = out.clone()
    assert torch.equal(want, pkg.matmul_fp8_experts(a, sa, w, sw, *tables) if experts else pkg.matmul_fp8(a, sa, w[0], sw[0]))
    torch.cuda.synchronize()
    start = time.perf_counter()
    call(give_up)
    torch.cuda.synchronize()
    assert time.perf_counter() - start < 5
    try:
        pkg.matmul_fp8_status()
        assert give_up & 15 in (2, 4, 8) and torch.equal(out, want)      # (that side never had to wait; the copies' begins with a wait)
    except L.B200MoEError as e:
        assert e.code == L.ERR_TIMEOUT
        pkg.matmul_fp8_status()
    out.fill_(7)
    call(0)
    pkg.matmul_fp8_status()
    assert torch.equal(out, want)
