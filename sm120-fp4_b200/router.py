"""Token-to-expert routing tables on the GPU: `route(ids, num_experts, experts, offsets, pairs)` has the signature of the
reference's pybind function (sm120fp4/kernels/moe_w4a16.py:85-91) and fills the caller's buffers in its padded form."""
from __future__ import annotations

import torch

from . import _lib


_WS: dict = {}   # (device index, stream) -> scratch tensor, grown on demand: steady-state calls allocate nothing


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Kept for the eager calls of one stream, which the stream runs one after the other. A captured call is replayed on any stream, beside graphs that
    were captured on the same one: it gets scratch of its own, from the graph's memory."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, stream)
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
        _WS[key] = ws
    return ws


def route(ids: torch.Tensor, num_experts: int, experts: torch.Tensor, offsets: torch.Tensor, pairs: torch.Tensor) -> None:
    """Fills the caller's tables, on the current stream of the GPU that they are on. An id below 0 (or from num_experts on) is an empty slot, whose pair
    is in no run: `pairs` is -1 behind the last one. The scratch memory of the counting sort is kept per (device, stream) and only grows, so a call of a size
    seen before allocates nothing, and calls on different streams do not share scratch. A call that is captured into a CUDA graph has scratch of its own, in the
    graph's memory."""
    if ids.dtype != torch.int32 or experts.dtype != torch.int32 or offsets.dtype != torch.int32 or pairs.dtype != torch.int32:
        raise TypeError("route takes int32 tensors")
    p = ids.numel()
    if offsets.numel() != experts.numel() + 1 or pairs.numel() != p:
        raise RuntimeError("shape")   # the reference's TORCH_CHECK message
    _lib.one_device("route", ids, experts, offsets, pairs)
    if not (experts.is_contiguous() and offsets.is_contiguous() and pairs.is_contiguous()):
        raise ValueError("route fills contiguous tables")
    _route(ids.contiguous(), p, num_experts, experts, offsets, pairs)


def _route(ids, p: int, num_experts: int, experts, offsets, pairs) -> None:
    h = _lib.lib()
    nbytes = h.b200moe_route_workspace_bytes(p, num_experts)
    if nbytes < 0:
        _lib.check(nbytes, "route")
    device = ids.device
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _route(ids, p, num_experts, experts, offsets, pairs)
    st = _lib.stream_ptr()
    ws = _workspace(device, st, nbytes)
    rc = h.b200moe_route(ids.data_ptr(), p, num_experts, experts.numel(), experts.data_ptr(), offsets.data_ptr(), pairs.data_ptr(), ws.data_ptr(), ws.numel(), st)
    if rc:
        _lib.check(rc, "route")


def route_tables(ids: torch.Tensor, num_experts: int):
    """Allocate and fill (experts [min(E, P)], offsets [min(E, P) + 1], pairs [P]) for `ids`; behind the last run -1 in experts and in pairs."""
    if not ids.is_cuda:
        raise RuntimeError("route_tables runs on the GPU; there is no CPU path in this package")
    ids = ids.to(torch.int32).contiguous()
    p = ids.numel()
    umax = min(num_experts, p)
    experts = torch.empty(umax, dtype=torch.int32, device=ids.device)
    offsets = torch.empty(umax + 1, dtype=torch.int32, device=ids.device)
    pairs = torch.empty(p, dtype=torch.int32, device=ids.device)
    _route(ids, p, num_experts, experts, offsets, pairs)
    return experts, offsets, pairs
