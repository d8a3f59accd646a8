"""The router's and the FP8 operators, each as work that can be timed and compared: in plain torch, and as this package's calls.

Kinds of cases:
  gate      router logits -> the k largest experts of each token with their softmax weights (`top_k_gate`); "step": and the gradient
            with respect to the logits, as in a training step
  balance   the load-balance loss of a batch and its pairs per expert (`balance_loss`), with the gradient with respect to the logits
  quantize  activations to E4M3 with a scale per 1x128 values (`quantize_fp8`); "copies" > 0: rows are gathered, each token that many times in
            expert order, as the experts' products take them
  weights   matrices to E4M3 with a scale per 128x128 block (`quantize_fp8_weight`), what a load does
  matmul    [M, K] x [N, K]^T of E4M3 codes with those scales (`matmul_fp8`): a projection, for one token and for a prompt
  experts   the same with a matrix per expert over rows sorted by expert (`matmul_fp8_experts`): the first or second half of an MoE layer

Inputs: hidden states N(0, 1) with a few columns ten times larger, weights N(0, 0.02), router logits N(0, 1), with "skewed" routing a bias per expert
of standard deviation 1.5; a padded batch has tokens whose expert ids are all -1, a masked one experts whose logit is -inf."""
from __future__ import annotations

import math

import torch

own = False

QWEN = dict(experts=128, hidden=2048, inter=768, top_k=8)
GEMMA = dict(experts=128, hidden=2816, inter=704, top_k=8)
TYPES = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)
GROUP, TOP, TINY = 128, 448.0, 1e-12      # values that share a scale, E4M3's largest value, the least maximum that a scale is made for
MOST_FLOPS, MOST_WEIGHTS, MOST_LOGITS = 8192 * 4096 * 4096, 128 * 1536 * 2048, 65536 * 256


def listed():
    return [
        # one user typing: the router of one layer
        dict(name="gate_t1", kind="gate", tokens=1, experts=128, top_k=8, dtype="bf16", renormalize=True, step=False, masked=False),
        # a training step's router, logits kept in 32 bits
        dict(name="gate_step_t16384", kind="gate", tokens=16384, experts=128, top_k=8, dtype="fp32", renormalize=True, step=True, masked=False),
        # fine-tuning on one short padded batch, a number of experts that is no power of two
        dict(name="balance_t333_e60", kind="balance", tokens=333, experts=60, top_k=4, dtype="fp32", padded=True),
        # a large training batch over many experts
        dict(name="balance_t65536_e256", kind="balance", tokens=65536, experts=256, top_k=8, dtype="bf16", padded=False),
        # a decode batch before a projection
        dict(name="quantize_m16", kind="quantize", rows=16, inner=2048, dtype="bf16", copies=0),
        # a prompt's tokens, laid out for the experts
        dict(name="quantize_t4096_x8", kind="quantize", rows=4096, inner=2816, dtype="bf16", copies=8),
        # a layer's gate and up weights at load time
        dict(name="weights_128", kind="weights", experts=128, outer=1536, inner=2048, dtype="bf16"),
        # a projection for one token: the weights' bytes and the launch
        dict(name="matmul_m1", kind="matmul", rows=1, outer=4096, inner=4096, out="bf16"),
        # a prompt of odd length, an inner size that ends inside a group, 32-bit results
        dict(name="matmul_m333", kind="matmul", rows=333, outer=2816, inner=704, out="fp32"),
        # the largest prompt
        dict(name="matmul_m8192", kind="matmul", rows=8192, outer=4096, inner=4096, out="bf16"),
        # a served batch: one or two rows for most experts
        dict(name="experts_t16", kind="experts", tokens=16, experts=128, top_k=8, outer=1536, inner=2048, routing="random", out="bf16"),
        # a prompt with hot and cold experts, an outer size that is no multiple of a tile
        dict(name="experts_t2050", kind="experts", tokens=2050, experts=128, top_k=8, outer=1408, inner=2816, routing="skewed", out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _draw_router(rng):
    experts = rng.choice([8, 16, 32, 60, 64, 96, 128, 128, 160, 256, 384, 512])
    top_k = min(rng.choice([1, 2, 4, 6, 8, 8, 10, 16]), experts)
    return dict(tokens=_log_int(rng, 1, MOST_LOGITS // max(experts, 256)), experts=experts, top_k=top_k, dtype=rng.choice(["bf16", "fp16", "fp32"]))


def draw(rng):
    kind = rng.choice(["gate", "gate", "balance", "balance", "quantize", "weights", "matmul", "matmul", "matmul", "experts", "experts", "experts"])
    if kind == "gate":
        return dict(kind=kind, **_draw_router(rng), renormalize=rng.random() < 0.7, step=rng.random() < 0.6, masked=rng.random() < 0.3)
    if kind == "balance":
        return dict(kind=kind, **_draw_router(rng), padded=rng.random() < 0.5)
    if kind == "quantize":
        copies, inner = rng.choice([0, 0, 2, 4, 8]), rng.choice([_log_int(rng, 16, 8192), 64 * _log_int(rng, 2, 128)])
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, 4096 * 2816 * 8 // (inner * max(copies, 1)))), inner=inner, dtype=rng.choice(["bf16", "fp16", "fp32"]), copies=copies)
    if kind == "weights":
        experts, inner = rng.choice([1, 1, 8, 60, 128]), 16 * _log_int(rng, 8, 512)
        return dict(kind=kind, experts=experts, outer=_log_int(rng, 16, max(16, min(8192, MOST_WEIGHTS // 2 // (experts * inner)))), inner=inner, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "matmul":
        outer, inner = rng.choice([16, 16, 64, 1]) * _log_int(rng, 16, 512), 16 * _log_int(rng, 8, 512)
        outer = max(16, min(outer, 16384))
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(16384, MOST_FLOPS // 2 // (outer * inner)))), outer=outer, inner=inner, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    s = dict(rng.choice([QWEN, GEMMA, dict(experts=64, hidden=2304, inter=1408, top_k=6), dict(experts=16, hidden=4096, inter=1344, top_k=2), dict(experts=256, hidden=1536, inter=512, top_k=8)]))
    outer, inner = (2 * s["inter"], s["hidden"]) if rng.random() < 0.5 else (s["hidden"], s["inter"])
    return dict(kind=kind, tokens=_log_int(rng, 1, max(1, MOST_FLOPS // 4 // (outer * inner * s["top_k"]))), experts=s["experts"], top_k=s["top_k"], outer=outer, inner=inner,
                routing=rng.choice(["random", "skewed"]), out=rng.choice(["bf16", "bf16", "fp32"]))


# ---------------------------------------------------------------------------------------------------- inputs

def _logits(case, gen, scale=1.0):
    e = case["experts"]
    x = torch.randn(case["tokens"], e, generator=gen, device="cuda") * scale
    if case.get("routing") == "skewed":
        x += 1.5 * torch.randn(e, generator=gen, device="cuda")
    return x


def _hidden(rows, inner, gen):
    x = torch.randn(rows, inner, generator=gen, device="cuda")
    x[:, torch.rand(inner, generator=gen, device="cuda") < 0.01] *= 10
    return x


def _sorted_by_expert(ids, experts):
    """(experts with rows, ascending, -1 behind them; where each one's rows begin; the pairs in that order): what `route_tables` gives."""
    flat = ids.reshape(-1)
    counts = torch.bincount(flat, minlength=experts)
    most = min(experts, flat.numel())
    has = torch.nonzero(counts).reshape(-1)
    table = torch.full((most,), -1, dtype=torch.int32, device="cuda")
    table[:has.numel()] = has.int()
    offsets = torch.full((most + 1,), flat.numel(), dtype=torch.int32, device="cuda")
    offsets[0] = 0
    offsets[1:has.numel() + 1] = torch.cumsum(counts[has], 0).int()
    return table, offsets, torch.sort(flat, stable=True)[1].int(), int(counts.max())


def _as_codes(x):
    """x [..., blocks, values that share a scale] -> (codes, scales): codes e4m3(fl(x * fl(448 / amax))), scale fl(amax / 448)."""
    amax = x.float().abs().amax(-1, keepdim=True).clamp(min=TINY).double()
    return (x.float() * (TOP / amax).float()).to(torch.float8_e4m3fn), (amax / TOP).float().squeeze(-1)


def _pad_to(x, dim, multiple):
    more = -x.shape[dim] % multiple
    if not more:
        return x
    shape = list(x.shape)
    shape[dim] = more
    return torch.cat([x, x.new_zeros(shape)], dim)


def _rows_to_codes(x):
    m, k = x.shape
    codes, scales = _as_codes(_pad_to(x, 1, GROUP).reshape(m, -1, GROUP))
    return codes.reshape(m, -1)[:, :k].contiguous(), scales


def _blocks_to_codes(w):
    e, n, k = w.shape
    p = _pad_to(_pad_to(w, 1, GROUP), 2, GROUP)
    nb, kb = p.shape[1] // GROUP, p.shape[2] // GROUP
    codes, scales = _as_codes(p.reshape(e, nb, GROUP, kb, GROUP).permute(0, 1, 3, 2, 4).reshape(e, nb, kb, GROUP * GROUP))
    codes = codes.reshape(e, nb, kb, GROUP, GROUP).permute(0, 1, 3, 2, 4).reshape(e, nb * GROUP, kb * GROUP)
    return codes[:, :n, :k].contiguous(), scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], dict(case)
    if kind == "gate":
        x = _logits(case, gen, 2.0)
        if case["masked"]:      # experts that are switched off, and a token that may use none
            x[torch.rand(x.shape, generator=gen, device="cuda") < 0.3] = -math.inf
            if case["tokens"] > 1:
                x[case["tokens"] // 2] = -math.inf
        state["logits"] = x.to(TYPES[case["dtype"]]).requires_grad_(case["step"])
        state["grad"] = torch.randn(case["tokens"], case["top_k"], generator=gen, device="cuda")
    elif kind == "balance":
        x = _logits({**case, "routing": "skewed"}, gen)
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top_k"]].int().contiguous()
        if case["padded"]:
            ids[case["tokens"] - case["tokens"] // 4:] = -1
        state["logits"], state["ids"] = x.to(TYPES[case["dtype"]]).requires_grad_(True), ids
        state["grad"] = torch.rand((), generator=gen, device="cuda") + 0.01
    elif kind == "quantize":
        state["x"] = _hidden(case["rows"], case["inner"], gen).to(TYPES[case["dtype"]])
        if case["copies"]:
            ids = torch.rand(case["rows"], 128, generator=gen, device="cuda").argsort(1)[:, :case["copies"]]
            state["source"] = (_sorted_by_expert(ids, 128)[2] // case["copies"]).int()
    elif kind == "weights":
        state["w"] = (torch.randn(case["experts"], case["outer"], case["inner"], generator=gen, device="cuda") * 0.02).to(TYPES[case["dtype"]])
    elif kind == "matmul":
        state["a"], state["a_scale"] = _rows_to_codes(_hidden(case["rows"], case["inner"], gen))
        w, s = _blocks_to_codes(torch.randn(1, case["outer"], case["inner"], generator=gen, device="cuda") * 0.02)
        state["w"], state["w_scale"] = w[0], s[0]
    else:
        ids = torch.sort(_logits(case, gen), dim=1, descending=True, stable=True)[1][:, :case["top_k"]]
        table, offsets, pairs, state["most"] = _sorted_by_expert(ids, case["experts"])
        a, s = _rows_to_codes(_hidden(case["tokens"], case["inner"], gen))
        source = (pairs // case["top_k"]).long()
        state["a"], state["a_scale"] = a.view(torch.uint8)[source].view(torch.float8_e4m3fn), s[source].contiguous()
        state["table"], state["offsets"] = table, offsets
        state["w"], state["w_scale"] = _blocks_to_codes(torch.randn(case["experts"], case["outer"], case["inner"], generator=gen, device="cuda") * 0.02)
    return state


# ---------------------------------------------------------------------------------------------------- the plain forms

def _softmax(x):
    """Rows of -inf alone get zeros."""
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _gate(state):
    x, k = state["logits"].detach().float(), state["top_k"]
    p = _softmax(x)
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    live = x.gather(1, ids) > -math.inf
    some = live.any(1, keepdim=True)
    w = p.gather(1, ids)
    if state["renormalize"]:
        w = w / torch.where(some, w.sum(1, keepdim=True), torch.ones_like(w[:, :1]))
    out = [w, torch.where(live, ids, -torch.ones_like(ids)).int()]
    if state["step"]:
        g = torch.where(live, state["grad"], torch.zeros_like(w))
        dot = (g * w).sum(1, keepdim=True)
        if state["renormalize"]:
            dx = torch.zeros_like(x).scatter_(1, ids, w * (g - dot))
        else:
            dx = p * (torch.zeros_like(x).scatter_(1, ids, g) - dot)
        out.append(dx.to(state["logits"].dtype))
    return out


def _balance(state):
    x, ids, e = state["logits"].detach().float(), state["ids"], state["experts"]
    p = _softmax(x)
    used = ids >= 0
    live = used.any(1, keepdim=True)
    tokens = live.sum().clamp(min=1).double()
    counts = torch.zeros(e + 1, dtype=torch.int32, device=x.device).index_add_(0, torch.where(used, ids, e).reshape(-1), torch.ones_like(ids).reshape(-1))[:e]
    f = (counts.double() / used.sum().clamp(min=1)).float()
    mean = torch.where(live, p, torch.zeros_like(p)).double().sum(0) / tokens
    loss = (e * (f.double() * mean).sum()).float()
    dx = p * (f - (p * f).sum(1, keepdim=True)) * (state["grad"] * (e / tokens).float())
    return [loss, counts, torch.where(live, dx, torch.zeros_like(dx)).to(state["logits"].dtype)]


def _spread(scale, dim, size):
    return scale.repeat_interleave(GROUP, dim).narrow(dim, 0, size)


def _matmul(state):
    a = state["a"].float() * _spread(state["a_scale"], 1, state["inner"])
    w = state["w"].float() * _spread(_spread(state["w_scale"], 0, state["outer"]), 1, state["inner"])
    return (a @ w.t()).to(TYPES[state["out"]])


def _experts(state):
    """Each expert's rows padded to the longest run, one product per expert, and the rows taken out again."""
    table, offsets, k, n = state["table"], state["offsets"].long(), state["inner"], state["outer"]
    a = state["a"].float() * _spread(state["a_scale"], 1, k)
    row = torch.arange(a.shape[0], device=a.device)
    run = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    at = row - offsets[run]
    padded = a.new_zeros(table.numel(), state["most"], k)
    padded[run, at] = a
    e = table.clamp(min=0).long()
    w = state["w"].view(torch.uint8)[e].view(torch.float8_e4m3fn).float() * _spread(_spread(state["w_scale"][e], 1, n), 2, k)
    return torch.bmm(padded, w.transpose(1, 2))[run, at].to(TYPES[state["out"]])


def run(state):
    kind = state["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "gate":
        return _gate(state)
    if kind == "balance":
        return _balance(state)
    if kind == "quantize":
        x = state["x"][state["source"]] if state["copies"] else state["x"]
        return _rows_to_codes(x)
    if kind == "weights":
        return _blocks_to_codes(state["w"])
    return _matmul(state) if kind == "matmul" else _experts(state)


# ---------------------------------------------------------------------------------------------------- this package's calls

def _run_own(state, kind):
    import sm120fp4_b200 as fp4
    if kind == "gate":
        weights, ids = fp4.top_k_gate(state["logits"], state["top_k"], renormalize=state["renormalize"])
        if not state["step"]:
            return [weights, ids]
        return [weights, ids, *torch.autograd.grad(weights, state["logits"], state["grad"])]
    if kind == "balance":
        loss, counts = fp4.balance_loss(state["logits"], state["ids"])
        return [loss, counts, *torch.autograd.grad(loss, state["logits"], state["grad"])]
    if kind == "quantize":
        return fp4.quantize_fp8(state["x"], src_row=state["source"] if state["copies"] else None)
    if kind == "weights":
        return fp4.quantize_fp8_weight(state["w"])
    if kind == "matmul":
        return fp4.matmul_fp8(state["a"], state["a_scale"], state["w"], state["w_scale"], out_dtype=TYPES[state["out"]])
    return fp4.matmul_fp8_experts(state["a"], state["a_scale"], state["w"], state["w_scale"], state["table"], state["offsets"], out_dtype=TYPES[state["out"]])


# ---------------------------------------------------------------------------------------------------- what a pass needs, and its value in 64 bits

def work(case):
    kind = case["kind"]
    if kind in ("gate", "balance"):
        size = TYPES[case["dtype"]].itemsize
        logits, slots = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        if kind == "gate":      # exponentials and comparisons are counted as one operation for each logit and slot
            return dict(bytes=logits * size + 8 * slots + case["step"] * (logits * size + 4 * slots), flops=logits * (4 + 4 * case["step"]))
        return dict(bytes=2 * logits * size + 4 * slots + 4 * case["experts"], flops=12 * logits)
    if kind == "quantize":
        rows, k = case["rows"] * max(1, case["copies"]), case["inner"]
        return dict(bytes=case["rows"] * k * TYPES[case["dtype"]].itemsize + rows * (k + 4 * -(-k // GROUP)) + 4 * rows * bool(case["copies"]), flops=3 * rows * k)
    if kind == "weights":
        n = case["experts"] * case["outer"] * case["inner"]
        return dict(bytes=n * (TYPES[case["dtype"]].itemsize + 1) + 4 * case["experts"] * -(-case["outer"] // GROUP) * -(-case["inner"] // GROUP), flops=3 * n)
    n, k = case["outer"], case["inner"]
    rows = case["rows"] if kind == "matmul" else case["tokens"] * case["top_k"]
    touched = 1 if kind == "matmul" else case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** case["tokens"])      # (random routing: what is expected)
    return dict(bytes=rows * (k + 4 * -(-k // GROUP)) + touched * (n * k + 4 * -(-n // GROUP) * -(-k // GROUP)) + rows * n * TYPES[case["out"]].itemsize, flops=2 * rows * n * k)


def _exact_codes(groups):
    """groups [number, values] in 64 bits -> codes and scales. The scale's and the factor's roundings to 32 bits, and the product's, belong to the
    definition; the nearest of E4M3's values is found among all of them, ties to the even code."""
    amax = torch.maximum(groups.abs().max(1)[0], torch.tensor(TINY, dtype=torch.float32, device=groups.device).double())
    y = (groups * (TOP / amax).float().double()[:, None]).float().double()
    value = torch.arange(127, dtype=torch.uint8, device=groups.device).view(torch.float8_e4m3fn).double()
    border = (value[1:] + value[:-1]) / 2
    v = y.abs()
    low = torch.searchsorted(border, v, right=False)
    up = torch.searchsorted(border, v, right=True)
    at = torch.where(low % 2 == 0, low, up)      # on a border low is the code below it, up the one above: the even one of the two
    return value[at] * torch.where(y < 0, -1.0, 1.0), (amax / TOP).float().double()


def _exact_product(a, a_scale, w, w_scale):
    """Group by group along the inner size, in 64 bits."""
    out = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=a.device)
    columns = torch.arange(w.shape[0], device=a.device) // GROUP
    for g in range(a_scale.shape[1]):
        part = a[:, g * GROUP:(g + 1) * GROUP].double() @ w[:, g * GROUP:(g + 1) * GROUP].double().t()
        out += part * a_scale[:, g, None].double() * w_scale[columns, g].double()
    return out


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind in ("gate", "balance"):
        x = state["logits"].detach().double()
        total = torch.logsumexp(x, 1, keepdim=True)
        p = torch.where(total == -math.inf, torch.zeros_like(x), torch.exp(x - total))
    if kind == "gate":
        chosen = torch.zeros_like(x, dtype=torch.bool)
        values, ids = torch.topk(x, case["top_k"], dim=1)      # (which of equal logits is taken changes no weight)
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top_k"]]
        chosen.scatter_(1, ids, values > -math.inf)
        q = torch.where(chosen, p, torch.zeros_like(p))
        if case["renormalize"]:
            q = q / q.sum(1, keepdim=True)
            q = torch.where(chosen, q, torch.zeros_like(q))
        out = [q.gather(1, ids), None]
        if case["step"]:
            g = torch.zeros_like(x).scatter_(1, ids, state["grad"].double())
            g = torch.where(chosen, g, torch.zeros_like(g))
            out.append((q if case["renormalize"] else p) * (g - (q * g).sum(1, keepdim=True)))
        return out
    if kind == "balance":
        ids, e = state["ids"].long(), case["experts"]
        live = (ids >= 0).sum(1) > 0
        counts = torch.bincount(ids[ids >= 0], minlength=e).double()
        f, tokens = counts / max(1.0, float(counts.sum())), max(1, int(live.sum()))
        p = p * live[:, None]
        dx = float(state["grad"].double()) * e / tokens * (p * f - p * (p @ f)[:, None])
        return [e / tokens * (p.sum(0) @ f), None, dx]
    if kind == "quantize":
        x = state["x"].double()
        m, k = x.shape
        codes, scales = _exact_codes(torch.nn.functional.pad(x, (0, -k % GROUP)).view(-1, GROUP))
        codes, scales = codes.view(m, -1)[:, :k], scales.view(m, -1)
        return [codes[state["source"].long()], scales[state["source"].long()]] if case["copies"] else [codes.contiguous(), scales]
    if kind == "weights":
        e, n, k = state["w"].shape
        nb, kb = -(-n // GROUP), -(-k // GROUP)
        codes = torch.empty(e, n, k, dtype=torch.float32, device="cuda")      # (E4M3's values are exact there)
        scales = torch.empty(e, nb, kb, dtype=torch.float64, device="cuda")
        for i in range(e):
            x = torch.nn.functional.pad(state["w"][i].double(), (0, -k % GROUP, 0, -n % GROUP))
            c, s = _exact_codes(x.view(nb, GROUP, kb, GROUP).transpose(1, 2).reshape(nb * kb, GROUP * GROUP))
            codes[i] = c.view(nb, kb, GROUP, GROUP).transpose(1, 2).reshape(nb * GROUP, kb * GROUP)[:n, :k].float()
            scales[i] = s.view(nb, kb)
        return [codes, scales]
    if kind == "matmul":
        return _exact_product(state["a"], state["a_scale"], state["w"], state["w_scale"])
    out = torch.zeros(state["a"].shape[0], case["outer"], dtype=torch.float64, device="cuda")
    begins, table = state["offsets"].tolist(), state["table"].tolist()
    for u, e in enumerate(table):
        b, t = begins[u], begins[u + 1]
        if e >= 0 and t > b:
            out[b:t] = _exact_product(state["a"][b:t], state["a_scale"][b:t], state["w"][e], state["w_scale"][e])
    return out
