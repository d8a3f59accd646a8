"""FP8 for the matrices of a model that are not NVFP4 (projections, shared experts, experts of FP8 checkpoints): E4M3 codes with one fp32 scale per 128 values
of a row (activations) or per 128x128 block (weights), the quantisers that make them and the products that take them. A value stands for code * scale;
`w_scale` is what such checkpoints call the inverse scale. No counterpart in the reference.

    q, s = quantize_fp8(x)                               # [M, K] -> codes [M, K], scales [M, ceil(K / 128)]
    y = matmul_fp8(q, s, w, w_scale)                     # w [N, K], w_scale [ceil(N / 128), ceil(K / 128)] -> [M, N]

    experts, offsets, pairs = route_tables(ids, E)       # the experts of a layer, one run of rows each
    q, s = quantize_fp8(x, src_row=pairs // top_k)       # (empty slots are -1 in pairs, and zero rows here)
    y = matmul_fp8_experts(q, s, w, w_scale, experts, offsets)      # row i is what pair pairs[i] gets

These calls have no derivatives: an input that requires a gradient, with gradients enabled, or that carries a tangent is refused (RuntimeError).
Nothing here synchronises or keeps state between calls; every call but matmul_fp8_status can be captured into a CUDA graph and runs on the tensors' device, on its current stream."""
from __future__ import annotations

import torch

from . import _lib

FP8 = torch.float8_e4m3fn
GROUP = 128


def _sizes(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and any(n > _lib.MAX_SIZE for n in t.shape):
            raise ValueError(f"{what} takes sizes up to {_lib.MAX_SIZE}, not {tuple(t.shape)}")


def _groups(n: int) -> int:
    return -(-n // GROUP)


def _pad16(n: int) -> int:
    return (n + 15) & ~15


def quantize_fp8(x: torch.Tensor, src_row: torch.Tensor | None = None):
    """x [M, K] bf16, fp16 or fp32 -> (codes float8_e4m3fn [R, K], scales f32 [R, ceil(K / 128)]), a scale for every 128 values of a row:
    scale = amax / 448, codes = x * (448 / amax) to nearest, amax at least 1e-12. With `src_row` (int32 [R]) row r is x[src_row[r]], which lays tokens out in runs per
    expert without a separate gather; an index outside x gives zero codes and scales. Rows of the codes start on 16 bytes: for K that is no multiple of 16
    they are further apart than K. A NaN makes its group NaN; with an infinity the group's scale is inf."""
    out = (_lib._host or _lib.host()).quantize_fp8(x, src_row)      # plain tensors in one native call (csrc/host.cpp), else None
    if out is not None:
        return out if type(out) is tuple else _lib.check(out, "quantize_fp8")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"expected [M, K] with K >= 1, got {tuple(x.shape)}")
    if x.dtype not in _lib.DTYPES:
        raise TypeError(f"quantize_fp8 takes bf16, fp16 or fp32, not {x.dtype}")
    _sizes("quantize_fp8", x, src_row)
    _lib.no_gradient("quantize_fp8", x)
    device = _lib.one_device("quantize_fp8", x)
    m, k = x.shape
    x = _lib.stored(x)
    if x.stride(1) != 1 and k > 1 or x.stride(0) < k and m > 1:
        x = x.contiguous()
    rows = m
    if src_row is not None:
        if src_row.dtype != torch.int32 or src_row.dim() != 1:
            raise TypeError("quantize_fp8: src_row is int32 [R]")
        _lib.one_device("quantize_fp8", x, src_row)
        src_row = _lib.stored(src_row).contiguous()
        rows = src_row.shape[0]
    ld = _pad16(k)
    codes = torch.empty_strided((rows, k), (ld, 1), dtype=FP8, device=device)
    scales = torch.empty((rows, _groups(k)), dtype=torch.float32, device=device)
    h = _lib.lib()
    nbytes = 0 if src_row is None else h.b200moe_quantize_fp8_workspace_bytes(m, rows, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _lib.call(device, "quantize_fp8", h.b200moe_quantize_fp8, x.data_ptr(), _lib.DTYPES[x.dtype], x.stride(0) if m > 1 else ld, m, _lib.ptr(src_row), rows, k,
              codes.data_ptr(), ld, scales.data_ptr(), _lib.ptr(ws), nbytes)
    return codes, scales


def quantize_fp8_weight(w: torch.Tensor):
    """w [N, K] or stacked experts [E, N, K], bf16, fp16 or fp32 -> (codes float8_e4m3fn of the same shape, scales f32 [..., ceil(N / 128), ceil(K / 128)]), a scale
    for every 128x128 block, as in quantize_fp8."""
    out = (_lib._host or _lib.host()).quantize_fp8_weight(w)      # (as in quantize_fp8)
    if out is not None:
        return out if type(out) is tuple else _lib.check(out, "quantize_fp8_weight")
    if w.dim() not in (2, 3) or w.shape[-1] < 1:
        raise ValueError(f"expected [N, K] or [E, N, K] with K >= 1, got {tuple(w.shape)}")
    if w.dtype not in _lib.DTYPES:
        raise TypeError(f"quantize_fp8_weight takes bf16, fp16 or fp32, not {w.dtype}")
    _sizes("quantize_fp8_weight", w)
    _lib.no_gradient("quantize_fp8_weight", w)
    device = _lib.one_device("quantize_fp8_weight", w)
    w = _lib.stored(w).contiguous()
    n, k = w.shape[-2:]
    e = w.shape[0] if w.dim() == 3 else 1
    ld = _pad16(k)
    codes = torch.empty_strided(w.shape, (n * ld, ld, 1)[3 - w.dim():], dtype=FP8, device=device)
    scales = torch.empty((*w.shape[:-2], _groups(n), _groups(k)), dtype=torch.float32, device=device)
    _lib.call(device, "quantize_fp8_weight", _lib.lib().b200moe_quantize_fp8_blocks, w.data_ptr(), _lib.DTYPES[w.dtype], e, n, k, codes.data_ptr(), ld, scales.data_ptr())
    return codes, scales


def _row_stride(codes: torch.Tensor, what: str, name: str) -> int:
    """Bytes from one row of codes to the next, which the copies want to be a multiple of 16."""
    if codes.dtype != FP8:
        raise TypeError(f"{what}: {name} are float8_e4m3fn codes, not {codes.dtype}")
    n, k = codes.shape[-2:]
    ld = codes.stride(-2) if n > 1 else _pad16(k)
    if codes.stride(-1) != 1 and k > 1 or ld < k or ld % 16 or codes.data_ptr() % 16:
        raise ValueError(f"{what}: rows of {name} must start on 16 bytes (strides {codes.stride()}); quantize_fp8 and quantize_fp8_weight lay them out so")
    return ld


def _scales(s: torch.Tensor, shape: tuple, what: str, name: str) -> torch.Tensor:
    if s.dtype != torch.float32:
        raise TypeError(f"{what}: {name} is fp32, not {s.dtype}")
    if tuple(s.shape) != shape:
        raise ValueError(f"{what}: expected {name} {list(shape)}, got {list(s.shape)}")
    return _lib.stored(s).contiguous()


def _output(out, out_dtype, m: int, n: int, device, what: str):
    if out is None:
        if out_dtype not in _lib.DTYPES:
            raise TypeError(f"{what} gives bf16, fp16 or fp32, not {out_dtype}")
        return torch.empty((m, n), dtype=out_dtype, device=device)
    if out.dtype not in _lib.DTYPES or (out_dtype is not None and out.dtype != out_dtype):
        raise TypeError(f"{what}: out is {out.dtype}, not {out_dtype}")
    if tuple(out.shape) != (m, n) or out.device != device:
        raise ValueError(f"{what}: expected out [{m}, {n}] on {device}, got {list(out.shape)} on {out.device}")
    if out.is_neg():
        raise ValueError(f"{what}: out is a negated view")
    if out.stride(1) != 1 and n > 1 or out.stride(0) < n and m > 1:
        raise ValueError(f"{what}: rows of out must be contiguous and apart from one another (strides {out.stride()})")
    return out


def matmul_fp8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, out_dtype: torch.dtype | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """a [M, K] x w [N, K]^T -> [M, N] in out_dtype (bf16 where neither it nor `out` says; fp16, fp32), for one row to many: codes and scales as quantize_fp8 (a) and
    quantize_fp8_weight (w) give them, any M, N and K >= 1. Products are exact, sums fp32, rounded once. `out` may be a view whose rows are apart."""
    if out is None:
        new = (_lib._host or _lib.host()).matmul_fp8(a, a_scale, w, w_scale, out_dtype or torch.bfloat16)      # (as in quantize_fp8)
        if new is not None:
            return new if type(new) is not int else _lib.check(new, "matmul_fp8")
    if a.dim() != 2 or w.dim() != 2 or a.shape[1] != w.shape[1] or a.shape[1] < 1:
        raise ValueError(f"matmul_fp8: expected [M, K] and [N, K] with K >= 1, got {tuple(a.shape)} and {tuple(w.shape)}")
    _sizes("matmul_fp8", a, w)
    _lib.no_gradient("matmul_fp8", a, a_scale, w, w_scale, out)
    a, w = _lib.stored(a), _lib.stored(w)
    lda, ldw = _row_stride(a, "matmul_fp8", "a"), _row_stride(w, "matmul_fp8", "w")
    (m, k), n = a.shape, w.shape[0]
    a_scale = _scales(a_scale, (m, _groups(k)), "matmul_fp8", "a_scale")
    w_scale = _scales(w_scale, (_groups(n), _groups(k)), "matmul_fp8", "w_scale")
    device = _lib.one_device("matmul_fp8", a, a_scale, w, w_scale)
    out = _output(out, out_dtype or (torch.bfloat16 if out is None else None), m, n, device, "matmul_fp8")
    _lib.call(device, "matmul_fp8", _lib.lib().b200moe_matmul_fp8, a.data_ptr(), lda, a_scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(), m, n, k, out.data_ptr(),
              _lib.DTYPES[out.dtype], max(out.stride(0), n))
    return out


def matmul_fp8_experts(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, experts: torch.Tensor, offsets: torch.Tensor,
                       out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows offsets[u] .. offsets[u + 1] - 1 of a [P, K] times w[experts[u]] [N, K]^T -> [P, N]; w [E, N, K], experts int32 [U], offsets int32 [U + 1] as `route_tables`
    gives them (ascending offsets, at most 1024 runs; -1 and empty runs where fewer experts have rows). Types and arithmetic as in matmul_fp8. Rows outside
    every run, and those of an expert outside 0..E-1, are zeros; in an `out` that was given they are left as they were."""
    what = "matmul_fp8_experts"
    if out is None:
        new = (_lib._host or _lib.host()).matmul_fp8_experts(a, a_scale, w, w_scale, experts, offsets, out_dtype or torch.bfloat16)      # (as in quantize_fp8)
        if new is not None:
            return new if type(new) is not int else _lib.check(new, what)
    if a.dim() != 2 or w.dim() != 3 or a.shape[1] != w.shape[2] or a.shape[1] < 1 or w.shape[0] < 1:
        raise ValueError(f"{what}: expected [P, K] and [E, N, K] with K >= 1, got {tuple(a.shape)} and {tuple(w.shape)}")
    _sizes(what, a, w)
    _lib.no_gradient(what, a, a_scale, w, w_scale, out)
    a, w = _lib.stored(a), _lib.stored(w)
    lda, ldw = _row_stride(a, what, "a"), _row_stride(w, what, "w")
    (m, k), (e, n, _) = a.shape, w.shape
    if e > 1 and w.stride(0) != n * ldw:
        raise ValueError(f"{what}: the experts' matrices must follow one another (strides {w.stride()})")
    if experts.dtype != torch.int32 or offsets.dtype != torch.int32:
        raise TypeError(f"{what} takes int32 tables")
    if experts.dim() != 1 or offsets.dim() != 1 or offsets.numel() != experts.numel() + 1:
        raise ValueError(f"{what}: expected experts [U] and offsets [U + 1], got {list(experts.shape)} and {list(offsets.shape)}")
    a_scale = _scales(a_scale, (m, _groups(k)), what, "a_scale")
    w_scale = _scales(w_scale, (e, _groups(n), _groups(k)), what, "w_scale")
    device = _lib.one_device(what, a, a_scale, w, w_scale, experts, offsets)
    experts, offsets = _lib.stored(experts).contiguous(), _lib.stored(offsets).contiguous()
    zero = out is None
    out = _output(out, out_dtype or (torch.bfloat16 if zero else None), m, n, device, what)
    _lib.call(device, what, _lib.lib().b200moe_matmul_fp8_experts, a.data_ptr(), lda, a_scale.data_ptr(), m, w.data_ptr(), ldw, w_scale.data_ptr(), e, experts.data_ptr(),
              offsets.data_ptr(), experts.numel(), n, k, out.data_ptr(), _lib.DTYPES[out.dtype], max(out.stride(0), n), int(zero))
    return out


def matmul_fp8_status(device: torch.device | str | int | None = None) -> None:
    """Raises if a bounded wait inside a matmul_fp8 / matmul_fp8_experts call ran out on this device (default: the current one) since the last look: results are then
    incomplete. Synchronises the device's current stream."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"matmul_fp8_status looks at a GPU, not at {device}")
    _lib.call(torch.device("cuda", torch.cuda.current_device()) if device.index is None else device, "matmul_fp8_status", _lib.lib().b200moe_matmul_fp8_status)
