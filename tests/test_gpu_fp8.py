"""GPU parity of the FP8 quantisers and products. The quantisers are bit-exact with their definition; a product is compared with 64 bits.

Tolerance of a product: per group the tensor core adds 128 exact products in fp32, whatever the order and with at most one unit of 2^-23 each (truncation
included): 128 * 2^-23 of the sum of magnitudes S; the sum over G groups is G fma and two products of scales: (G + 3) * 2^-24 of S, and with a split inner size
up to 8 more additions; the result is rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
FP8 = torch.float8_e4m3fn


def groups(n):
    return -(-n // 128)


def codes64(x, rows):
    """Definition of the quantisers, `rows` rows of a block sharing a scale: scale = fl(amax / 448), code = e4m3(fl(x * fl(448 / amax))). In 64 bits a quotient and a
    product of fp32 values are rounded to fp32 as one rounding would."""
    n, k = x.shape
    p = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -n % rows))
    nb, kb = p.shape[0] // rows, p.shape[1] // 128
    b = p.view(nb, rows, kb, 128)
    amax = torch.maximum(b.abs().amax((1, 3)), torch.tensor(1e-12, dtype=torch.float32, device=x.device).double())
    factor = (448.0 / amax.cpu()).float().double().to(x.device)
    y = (b * factor[:, None, :, None]).float().view(nb * rows, kb * 128)[:n, :k]
    return y.to(FP8), (amax.cpu() / 448.0).float().to(x.device)


def same(a, b):
    """Equal bits, any NaN for any NaN."""
    a, b = a.float(), b.float()
    return bool((torch.isnan(a) == torch.isnan(b)).all()) and bool((a == b)[~torch.isnan(a)].all())


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (16, 2048), (3, 704), (7, 16), (5, 100), (130, 129), (33, 1000), (300, 2816), (2, 8192)])
def test_quantize_rows(dtype, m, k):
    import sm120fp4_b200 as pkg
    x = randn(m, k, seed=m + k, scale=3.0).to(dtype).cuda()
    x[:, ::7] *= 100
    x[m // 2, :] = 0
    q, s = pkg.quantize_fp8(x)
    wq, ws = codes64(x, 1)
    assert q.dtype == FP8 and q.shape == (m, k) and s.shape == (m, groups(k)) and q.stride(0) % 16 == 0
    assert same(q, wq) and torch.equal(s, ws)
    src = torch.randint(-2, m + 2, (2 * m + 3,), generator=torch.Generator().manual_seed(1)).int().cuda()
    q2, s2 = pkg.quantize_fp8(x, src_row=src)
    inside = (src >= 0) & (src < m)
    at = src.clamp(0, m - 1).long()
    assert same(q2, torch.where(inside[:, None], q.float()[at], torch.zeros(1, device="cuda")))
    assert torch.equal(s2, torch.where(inside[:, None], s[at], torch.zeros(1, device="cuda")))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,copies,k", [(1400, 8, 1024), (2000, 2, 2816), (600, 30, 704), (4000, 3, 1040), (4096, 8, 512), (9000, 8, 160)])
def test_quantize_many_copies(dtype, m, copies, k):
    """Rows that are asked for several times in calls large enough for the lists: some twice as often, some never, some indexes outside."""
    import sm120fp4_b200 as pkg
    x = randn(m, k, seed=m + k).to(dtype).cuda()
    src = torch.randint(-3, m + 3, (m * copies + 5,), generator=torch.Generator().manual_seed(copies)).int()
    src[:m // 2] = m // 3
    src = src.cuda()
    q, s = pkg.quantize_fp8(x)
    got_q, got_s = pkg.quantize_fp8(x, src_row=src)
    inside = (src >= 0) & (src < m)
    at = src.clamp(0, m - 1).long()
    assert same(got_q, torch.where(inside[:, None], q.float()[at], torch.zeros(1, device="cuda")))
    assert torch.equal(got_s, torch.where(inside[:, None], s[at], torch.zeros(1, device="cuda")))
    wide = torch.zeros(m, k + 8, dtype=dtype, device="cuda")[:, 4:4 + k]      # rows that start off 16 bytes: the other way to the same values
    wide.copy_(x)
    q2, s2 = pkg.quantize_fp8(wide, src_row=src)
    assert same(q2, got_q) and torch.equal(s2, got_s)


def test_quantize_every_value_of_a_group():
    """Every code and every border between two: values v / 448 of a group whose maximum is 448."""
    import sm120fp4_b200 as pkg
    v = torch.arange(127, dtype=torch.uint8).view(FP8).double()
    mid = (v[1:] + v[:-1]) / 2
    every = torch.cat([v, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    every = torch.cat([every, -every])
    x = torch.zeros(groups(every.numel()) * 128, dtype=torch.float32).view(-1, 128)
    x = torch.cat([torch.full((x.shape[0] * 2, 1), 448.0), torch.zeros(x.shape[0] * 2, 127)], 1)
    flat = every.float()
    for i in range(0, flat.numel(), 127):
        part = flat[i:i + 127]
        x[i // 127, 1:1 + part.numel()] = part
    q, s = pkg.quantize_fp8(x.cuda())
    wq, ws = codes64(x.cuda(), 1)
    assert same(q, wq) and torch.equal(s, ws) and float(s.max()) == 1.0


def test_quantize_zeros_infinities_nan_and_strides():
    import sm120fp4_b200 as pkg
    for dtype in TYPES:
        x = randn(4, 384, seed=2).to(dtype).cuda()
        x[0], x[1, 5], x[2, 300], x[3, 130] = 0, math.inf, math.nan, -math.inf
        q, s = pkg.quantize_fp8(x)
        q = q.float()
        assert float(q[0].abs().max()) == 0.0 and bool((s[0] > 0).all())
        assert math.isinf(float(s[1, 0])) and bool(q[1, 5].isnan()) and float(q[1, 6]) == 0.0 and bool(torch.isfinite(q[1, 128:]).all())
        assert bool(s[2, 2].isnan()) and bool(q[2, 256:].isnan().all()) and bool(torch.isfinite(q[2, :256]).all())
        assert math.isinf(float(s[3, 1])) and bool(torch.isfinite(q[3, :128]).all())
    big = randn(20, 400, seed=3).bfloat16().cuda()
    for x in (big[:, :256], big[:, 1:257], big[::3, 8:200], big.t()[:130, :16], big[:1].expand(5, 400)):
        q, s = pkg.quantize_fp8(x)
        q2, s2 = pkg.quantize_fp8(x.contiguous())
        assert same(q, q2) and torch.equal(s, s2)
    for x in (torch.zeros(0, 64), torch.zeros(0, 1)):
        q, s = pkg.quantize_fp8(x.cuda())
        assert q.shape == x.shape and s.shape == (0, 1)
    tiny = torch.full((2, 128), 1e-20).cuda()
    q, s = pkg.quantize_fp8(tiny)
    assert same(q, codes64(tiny, 1)[0]) and torch.equal(s, codes64(tiny, 1)[1])
    huge = torch.full((1, 128), torch.finfo(torch.float32).max).cuda()
    q, s = pkg.quantize_fp8(huge)
    assert float(q.float().min()) == 448.0 and math.isfinite(float(s))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (100, 70), (1408, 704), (3, 200, 144), (5, 129, 130), (2, 256, 2048), (1, 17, 16)])
def test_quantize_blocks(dtype, shape):
    import sm120fp4_b200 as pkg
    w = randn(*shape, seed=sum(shape), scale=0.02).to(dtype).cuda()
    w[..., : shape[-2] // 2, :] *= 30
    q, s = pkg.quantize_fp8_weight(w)
    n, k = shape[-2:]
    assert q.dtype == FP8 and q.shape == w.shape and s.shape == (*shape[:-2], groups(n), groups(k))
    for qi, si, wi in zip(q.reshape(-1, n, k) if q.dim() == 3 else [q], s.reshape(-1, groups(n), groups(k)), w.reshape(-1, n, k)):
        wq, ws = codes64(wi, 128)
        assert same(qi, wq) and torch.equal(si, ws)


def test_quantize_blocks_nan_stays_in_its_block():
    import sm120fp4_b200 as pkg
    w = randn(300, 300, seed=1).cuda()
    w[200, 10], w[0, 299] = math.nan, math.inf
    q, s = pkg.quantize_fp8_weight(w)
    assert torch.isnan(s).nonzero().tolist() == [[1, 0]] and torch.isinf(s).nonzero().tolist() == [[0, 2]]
    assert bool(torch.isnan(q.float()[128:256, :128]).all()) and int(torch.isnan(q.float()).sum()) == 128 * 128 + 1


# ---------------------------------------------------------------------------------------------------- products

def product64(a, sa, w, sw):
    """(out, sum of magnitudes) in 64 bits."""
    k, n = a.shape[1], w.shape[0]
    x = a.double() * sa.double().repeat_interleave(128, 1)[:, :k]
    y = w.double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ y.t(), x.abs() @ y.abs().t()


def allowed(want, size, k, dtype):
    fp32 = (128 * 2.0 ** -23 + (groups(k) + 3 + 8) * 2.0 ** -24) * size
    return fp32 + torch.finfo(dtype).eps / 2 * (want.abs() + fp32) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def close(got, a, sa, w, sw):
    want, size = product64(a, sa, w, sw)
    off = (got.double() - want).abs()
    tol = allowed(want, size, a.shape[1], got.dtype)
    assert bool((off <= tol).all()), f"{a.shape} x {w.shape}: {float((off / tol.clamp(min=1e-300)).max()):.2f} of the tolerance"


def operands(m, n, k, seed=0):
    import sm120fp4_b200 as pkg
    x, w = randn(m, k, seed=seed).cuda(), randn(n, k, seed=seed + 1, scale=0.02).cuda()
    x[:, ::50] *= 10
    w[: n // 2] *= 5
    return *pkg.quantize_fp8(x), *pkg.quantize_fp8_weight(w)


SIZES = [(1, 2048, 2048), (8, 1536, 2048), (48, 4096, 1024), (200, 4096, 512), (520, 4096, 256), (1, 1, 1), (1, 4096, 4096), (1, 128, 128), (2, 16, 16), (3, 130, 200), (16, 1536, 2048), (17, 300, 384), (32, 2816, 704), (33, 257, 100), (64, 64, 8192), (65, 129, 640),
         (100, 4096, 130), (128, 1408, 2816), (129, 100, 512), (200, 2048, 256), (333, 2816, 704), (500, 5001, 300), (1000, 4100, 272), (1024, 4096, 1024), (1300, 7000, 129), (2100, 2570, 640), (2048, 2560, 256)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(m, n, k):
    import sm120fp4_b200 as pkg
    a, sa, w, sw = operands(m, n, k, m + n + k)
    for dtype in TYPES:
        close(pkg.matmul_fp8(a, sa, w, sw, out_dtype=dtype), a, sa, w, sw)
    got = pkg.matmul_fp8(a, sa, w, sw)
    assert got.dtype == torch.bfloat16
    assert torch.equal(got, pkg.matmul_fp8(a, sa, w, sw))
    pkg.matmul_fp8_status()


def test_matmul_whole_numbers_are_exact():
    """Codes that are small whole numbers and scales that are powers of two: every sum is exact in fp32, so the result has no error at all."""
    import sm120fp4_b200 as pkg
    for m, n, k in [(5, 300, 700), (150, 260, 1000), (700, 4000, 512)]:
        g = torch.Generator().manual_seed(m)
        kp = (k + 15) // 16 * 16
        a = torch.randint(-4, 5, (m, kp), generator=g).float().to(FP8).cuda()[:, :k]
        w = torch.randint(-4, 5, (n, kp), generator=g).float().to(FP8).cuda()[:, :k]
        sa = (2.0 ** torch.randint(-2, 3, (m, groups(k)), generator=g)).cuda()
        sw = (2.0 ** torch.randint(-2, 3, (groups(n), groups(k)), generator=g)).cuda()
        want, _ = product64(a, sa, w, sw)
        assert torch.equal(pkg.matmul_fp8(a, sa, w, sw, out_dtype=torch.float32).double(), want)


def test_matmul_views_and_out():
    """Rows apart, in the codes and in the output (what lies between its rows stays), and outputs that do not start on 16 bytes."""
    import sm120fp4_b200 as pkg
    for m, n, k in [(7, 200, 256), (150, 300, 256), (1200, 4100, 256)]:
        a, sa, w, sw = operands(m, n, 512, m)
        av, wv = a[:, 128:384], w[:, 128:384]
        sav, swv = sa[:, 1:3], sw[:, 1:3]
        want = pkg.matmul_fp8(av, sav, wv, swv)
        close(want, av, sav, wv, swv)
        for dtype in TYPES:
            for left in (0, 1, 8):
                buf = torch.full((m, n + 24), 7.0, dtype=dtype, device="cuda")
                out = buf[:, left:left + n]
                got = pkg.matmul_fp8(av, sav, wv, swv, out=out)
                assert got is out
                assert torch.equal(out, pkg.matmul_fp8(av, sav, wv, swv, out_dtype=dtype))
                assert bool((buf[:, :left] == 7).all()) and bool((buf[:, left + n:] == 7).all())


def test_matmul_row_ends_inside_16_bytes():
    """Rows of the output on 16 bytes whose last values end inside 16: what stands behind them stays."""
    import sm120fp4_b200 as pkg
    for m, n, k in [(40, 150, 128), (1300, 5003, 256)]:
        a, sa, w, sw = operands(m, n, k, m)
        for dtype in TYPES:
            want = pkg.matmul_fp8(a, sa, w, sw, out_dtype=dtype)
            close(want, a, sa, w, sw)
            buf = torch.full((m, (n + 63) // 16 * 16), 7.0, dtype=dtype, device="cuda")
            assert torch.equal(pkg.matmul_fp8(a, sa, w, sw, out=buf[:, :n]), want) and bool((buf[:, n:] == 7).all())
    off = [0, 3, 500, 533, 900]      # runs that end inside a warp's 32 rows, results of both widths
    a, sa = pkg.quantize_fp8(randn(900, 256, seed=1).cuda())
    w, sw = pkg.quantize_fp8_weight(randn(4, 310, 256, seed=2).cuda())
    experts, offsets = torch.tensor([3, 1, 0, 2], dtype=torch.int32, device="cuda"), torch.tensor(off, dtype=torch.int32, device="cuda")
    for dtype in TYPES:
        buf = torch.full((900, 320), 7.0, dtype=dtype, device="cuda")
        pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out=buf[:, :310])
        assert bool((buf[:, 310:] == 7).all())
        for u, e in enumerate((3, 1, 0, 2)):
            r = slice(off[u], off[u + 1])
            close(buf[r, :310], a[r], sa[r], w[e], sw[e])


def test_matmul_nan_and_infinity_stay_in_their_rows():
    import sm120fp4_b200 as pkg
    for m in (20, 300, 1100):
        a, sa, w, sw = operands(m, 4096, 256, 5)
        clean = pkg.matmul_fp8(a, sa, w, sw)
        raw = a.view(torch.uint8).clone()
        raw[3, 200] = 0x7F
        sa2 = sa.clone()
        sa2[7, 0] = math.inf
        got = pkg.matmul_fp8(raw.view(FP8), sa2, w, sw)
        assert bool(got[3].isnan().all()) and not bool(torch.isfinite(got[7]).all())
        rest = [i for i in range(m) if i not in (3, 7)]
        assert torch.equal(got[rest], clean[rest])


def test_matmul_empty():
    import sm120fp4_b200 as pkg
    a, sa, w, sw = operands(4, 32, 128)
    assert pkg.matmul_fp8(a[:0], sa[:0], w, sw).shape == (0, 32)
    assert pkg.matmul_fp8(a, sa, w[:0], sw[:0]).shape == (4, 0)
    with pytest.raises(TypeError):
        pkg.matmul_fp8(a, sa, w, sw, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        pkg.matmul_fp8(a, sa, w, sw, out=torch.zeros(3, 32, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(TypeError):
        pkg.matmul_fp8(a, sa, w, sw, out_dtype=torch.float16, out=torch.zeros(4, 32, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError):
        pkg.matmul_fp8(a, sa, w, sw, out=torch.zeros(32, 4, dtype=torch.bfloat16, device="cuda").t())


def runs_of(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return off


@pytest.mark.parametrize("counts,n,k", [([1], 64, 128), ([1, 0, 2, 1], 1536, 256), ([5, 17, 0, 1, 40], 300, 704), ([200, 3, 129, 0, 1], 257, 300), ([0, 0, 0], 64, 64),
                                        ([16] * 40, 704, 512), ([130, 1, 500, 127, 128, 0, 300, 90], 1408, 640), ([1500], 200, 384), ([2] * 300, 48, 160), ([600, 255, 1, 900, 0, 513], 1400, 300), ([900, 130, 0, 1300], 1400, 300),
                                        ([3, 0, 5, 1, 9] * 8, 520, 640), ([40] + [1] * 50, 300, 512)])
def test_experts(counts, n, k):
    import sm120fp4_b200 as pkg
    e = len(counts) + 2
    off = runs_of(counts)
    p = off[-1] + 9      # rows behind the last run
    a, sa = pkg.quantize_fp8(randn(p, k, seed=n).cuda())
    w, sw = pkg.quantize_fp8_weight(randn(e, n, k, seed=k, scale=0.02).cuda())
    order = torch.randperm(e, generator=torch.Generator().manual_seed(4))[:len(counts)].int()
    experts, offsets = order.cuda(), torch.tensor(off, dtype=torch.int32, device="cuda")
    for dtype in (torch.bfloat16, torch.float32):
        got = pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out_dtype=dtype)
        for u, c in enumerate(counts):
            if c:
                s = slice(off[u], off[u + 1])
                close(got[s], a[s], sa[s], w[int(order[u])], sw[int(order[u])])
        assert float(got[off[-1]:].float().abs().max()) == 0.0
        kept = torch.full((p, n), 5.0, dtype=dtype, device="cuda")
        pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out=kept)
        assert torch.equal(kept[:off[-1]], got[:off[-1]]) and bool((kept[off[-1]:] == 5).all())
    pkg.matmul_fp8_status()


def test_experts_tables_with_gaps_and_unknown_experts():
    import sm120fp4_b200 as pkg
    a, sa = pkg.quantize_fp8(randn(60, 256, seed=1).cuda())
    w, sw = pkg.quantize_fp8_weight(randn(4, 130, 256, seed=2).cuda())
    experts = torch.tensor([2, -1, 9, 0, -1], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([4, 20, 25, 30, 50, 50], dtype=torch.int32, device="cuda")
    got = pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets)
    close(got[4:20], a[4:20], sa[4:20], w[2], sw[2])
    close(got[30:50], a[30:50], sa[30:50], w[0], sw[0])
    for s in (slice(0, 4), slice(20, 30), slice(50, 60)):
        assert float(got[s].float().abs().max()) == 0.0
    kept = torch.full((60, 130), 5.0, dtype=torch.bfloat16, device="cuda")
    pkg.matmul_fp8_experts(a, sa, w, sw, experts, offsets, out=kept)
    for s in (slice(0, 4), slice(20, 30), slice(50, 60)):
        assert bool((kept[s] == 5).all())
    far = torch.tensor([-7, 20, 25, 30, 1000, 2000], dtype=torch.int32, device="cuda")      # held to the rows there are
    got = pkg.matmul_fp8_experts(a, sa, w, sw, experts, far)
    close(got[:20], a[:20], sa[:20], w[2], sw[2])
    close(got[30:], a[30:], sa[30:], w[0], sw[0])
    none = pkg.matmul_fp8_experts(a, sa, w, sw, experts[:0], offsets[:1])
    assert none.shape == (60, 130) and float(none.float().abs().max()) == 0.0
    assert pkg.matmul_fp8_experts(a[:0], sa[:0], w, sw, experts, torch.zeros_like(offsets)).shape == (0, 130)


def test_experts_may_come_twice_and_in_any_order():
    import sm120fp4_b200 as pkg
    a, sa = pkg.quantize_fp8(randn(90, 256, seed=1).cuda())
    w, sw = pkg.quantize_fp8_weight(randn(3, 70, 256, seed=2).cuda())
    experts, off = [2, 0, 2, 1, 0], [0, 30, 31, 60, 60, 90]
    got = pkg.matmul_fp8_experts(a, sa, w, sw, torch.tensor(experts, dtype=torch.int32, device="cuda"), torch.tensor(off, dtype=torch.int32, device="cuda"))
    for u, e in enumerate(experts):
        r = slice(off[u], off[u + 1])
        if off[u + 1] > off[u]:
            close(got[r], a[r], sa[r], w[e], sw[e])


def test_experts_row_is_the_same_whatever_its_run():
    """A row's result does not depend on the rows beside it, within one form of the kernel."""
    import sm120fp4_b200 as pkg
    a, sa = pkg.quantize_fp8(randn(32, 512, seed=1).cuda())
    w, sw = pkg.quantize_fp8_weight(randn(2, 256, 512, seed=2).cuda())
    one = pkg.matmul_fp8_experts(a, sa, w, sw, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 16, 32], dtype=torch.int32, device="cuda"))
    two = pkg.matmul_fp8_experts(a, sa, w, sw, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 3, 32], dtype=torch.int32, device="cuda"))
    assert torch.equal(one[:3], two[:3]) and torch.equal(one[16:], two[16:])


def test_layer_from_router_to_combine():
    """The operators as a layer uses them: gate -> balance loss and counts -> route -> quantise by run -> first products -> SiLU * up -> quantise -> second products ->
    weighted sum. Each step is checked against 64 bits from the same inputs; the whole against the layer in 64 bits from the codes."""
    import sm120fp4_b200 as pkg
    t, e, h, inter, k = 70, 16, 256, 192, 4
    x, logit = randn(t, h, seed=1).bfloat16().cuda(), randn(t, e, seed=2).cuda()
    w1, s1 = pkg.quantize_fp8_weight(randn(e, 2 * inter, h, seed=3, scale=0.05).cuda())
    w2, s2 = pkg.quantize_fp8_weight(randn(e, h, inter, seed=4, scale=0.05).cuda())

    def layer(x, logit):
        weights, ids = pkg.top_k_gate(logit, k)
        loss, counts = pkg.balance_loss(logit, ids)
        experts, offsets, pairs = pkg.route_tables(ids, e)
        q, s = pkg.quantize_fp8(x, src_row=pairs // k)
        y = pkg.matmul_fp8_experts(q, s, w1, s1, experts, offsets)
        act = (y[:, :inter].float() * torch.nn.functional.silu(y[:, inter:].float())).bfloat16()
        q2, sc2 = pkg.quantize_fp8(act)
        z = pkg.matmul_fp8_experts(q2, sc2, w2, s2, experts, offsets, out_dtype=torch.float32)
        out = torch.zeros(t * k, h, device="cuda").index_copy_(0, pairs.long(), z) * weights.reshape(-1, 1)
        return out.view(t, k, h).sum(1), counts, (experts, offsets, pairs, q, s, y, q2, sc2, z)

    out, counts, (experts, offsets, pairs, q, s, y, q2, sc2, z) = layer(x, logit)
    begin, run = offsets.tolist(), experts.tolist()
    assert begin[-1] == t * k
    for u, i in enumerate(run):
        if i < 0:
            continue
        r = slice(begin[u], begin[u + 1])
        assert int(counts[i]) == begin[u + 1] - begin[u]
        close(y[r], q[r], s[r], w1[i], s1[i])
        close(z[r], q2[r], sc2[r], w2[i], s2[i])
    assert same(q, codes64(x[(pairs // k).long()], 1)[0])
    weights, _ = pkg.top_k_gate(logit, k)
    want = (torch.zeros(t * k, h, dtype=torch.float64, device="cuda").index_copy_(0, pairs.long(), z.double()) * weights.double().reshape(-1, 1)).view(t, k, h).sum(1)
    assert bool(((out.double() - want).abs() <= 6 * 2.0 ** -24 * (z.abs().amax() * 4)).all())

    graph = torch.cuda.CUDAGraph()      # the same, captured and replayed with other inputs
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, logit)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        captured = layer(x, logit)
    for seed in (7, 8):
        x.copy_(randn(t, h, seed=seed).bfloat16())
        logit.copy_(randn(t, e, seed=seed + 10))
        graph.replay()
        again = layer(x, logit)
        assert torch.equal(captured[0], again[0]) and torch.equal(captured[1], again[1])
    pkg.matmul_fp8_status()


def test_layer_of_a_padded_batch():
    """Tokens that may use no expert (logits of -inf) have ids of -1 from the gate on: no expert counts them, no run holds them, the rows behind the last run are zeros."""
    import sm120fp4_b200 as pkg
    for t, live, e, k in [(40, 25, 16, 4), (3000, 1801, 32, 2)]:
        x, logit = randn(t, 256, seed=1).bfloat16().cuda(), randn(t, e, seed=2).cuda()
        logit[live:] = -math.inf
        logit[:live, 3] = -math.inf      # an expert that is switched off
        w, sw = pkg.quantize_fp8_weight(randn(e, 130, 256, seed=3).cuda())
        weights, ids = pkg.top_k_gate(logit, k)
        loss, counts = pkg.balance_loss(logit, ids)
        experts, offsets, pairs = pkg.route_tables(ids, e)
        assert int(ids[live:].max()) == -1 and int(ids[:live].min()) >= 0 and float(weights[live:].abs().max()) == 0.0
        assert int(counts.sum()) == live * k == int(offsets[-1]) and int(counts[3]) == 0
        q, s = pkg.quantize_fp8(x, src_row=pairs // k)
        y = pkg.matmul_fp8_experts(q, s, w, sw, experts, offsets, out_dtype=torch.float32)
        begin = offsets.tolist()
        for u, i in enumerate(experts.tolist()):
            if begin[u + 1] > begin[u]:
                r = slice(begin[u], begin[u + 1])
                assert i != 3 and int(counts[i]) == begin[u + 1] - begin[u]
                close(y[r], q[r], s[r], w[i], sw[i])
                assert same(q[r], codes64(x[(pairs[r] // k).long()], 1)[0])
        assert float(y[live * k:].abs().max()) == 0.0


def test_products_on_two_streams_at_once():
    import sm120fp4_b200 as pkg
    sets = [operands(m, n, k, 31 * m) for m, n, k in [(8, 1024, 2048), (700, 4096, 512)]]
    want = [pkg.matmul_fp8(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(pkg.matmul_fp8(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    pkg.matmul_fp8_status()
