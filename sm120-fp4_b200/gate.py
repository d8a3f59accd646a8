"""The router from its logits on: `top_k_gate` gives the (weights, ids) that `Weights.forward` and `route` take, `balance_loss` the auxiliary loss that
keeps experts evenly used, with the number of pairs of each. Both have gradients with respect to the logits (reverse mode; forward mode is refused). The reference leaves this part to
torch (softmax, top-k, renormalise: sm120fp4/kernels/moe_layer.py:195-200).

Nothing here synchronises or keeps state between calls: forward and backward can be captured into a CUDA graph. A capture of a backward pass wants, as with
every autograd function, that no graph of the same leaves that was made on another stream is alive: logits that are such a leaf are refused (RuntimeError), all that are
a leaf where the host extension, which can tell, is not there; for leaves further back it is the caller's to see to."""
from __future__ import annotations

import torch

from . import _lib

MAX_EXPERTS, MAX_TOP_K, MAX_PAIRS = 512, 16, (1 << 31) - 1


def _logits(logits: torch.Tensor, what: str) -> torch.Tensor:
    if torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:      # outputs without a tangent would read as a derivative of zero
        raise NotImplementedError(f"{what} has no forward-mode derivative")
    if logits.dim() != 2:
        raise ValueError(f"{what}: expected logits [tokens, experts], got {tuple(logits.shape)}")
    if logits.dtype not in _lib.DTYPES:
        raise TypeError(f"{what} takes bf16, fp16 or fp32 logits, not {logits.dtype}")
    if not 1 <= logits.shape[1] <= MAX_EXPERTS or logits.shape[0] > _lib.MAX_SIZE:
        raise ValueError(f"{what} takes 1 to {MAX_EXPERTS} experts and at most {_lib.MAX_SIZE} tokens, not {tuple(logits.shape)}")
    _lib.one_device(what, logits)
    logits = _lib.stored(logits)
    if logits.stride(1) != 1 and logits.shape[1] > 1 or logits.stride(0) < logits.shape[1] and logits.shape[0] > 1:
        return logits.contiguous()
    return logits


def _check_capture(logits: torch.Tensor, what: str) -> None:
    """A leaf's gradient is handed over on the stream on which its accumulator was made. Where an eager graph keeps that alive, a backward pass that is being captured on
    another stream ends the process: refused while it still can be."""
    if not (logits.requires_grad and logits.is_leaf and torch.is_grad_enabled()):
        return
    with torch.cuda.device(logits.device):
        if torch.cuda.is_current_stream_capturing():
            (_lib._host or _lib.host()).check_capture(logits, what)


def _gate(logits: torch.Tensor, top_k: int, renormalize: bool):
    tokens, e = logits.shape
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device)
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
    _lib.call(logits.device, "top_k_gate", _lib.lib().b200moe_gate, logits.data_ptr(), _lib.DTYPES[logits.dtype], max(logits.stride(0), e), tokens, e, top_k,
              int(renormalize), weights.data_ptr(), ids.data_ptr())
    return weights, ids


def _once(out: torch.Tensor, what: str) -> torch.Tensor:
    """The gradient of a gradient is not there: whoever asks for it is told so."""
    if not torch.is_grad_enabled():
        return out
    return torch._C._functions.DelayedError(f"{what} is differentiable once".encode(), 1)(out.detach().requires_grad_(True))


def _unpacked(t: torch.Tensor, shape: tuple, dtype: torch.dtype, grad: torch.Tensor, what: str) -> torch.Tensor:
    """A saved tensor as the forward pass saw it. Hooks on saved tensors may give back another one, whose memory would be read as if it were the first."""
    if t.layout != torch.strided or t.device != grad.device or t.dtype != dtype or tuple(t.shape) != shape:
        raise RuntimeError(f"{what} backward: a hook gave back a saved tensor of another size, type or device")
    t = _lib.stored(t.detach())
    return t if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize):
        weights, ids = _gate(logits, top_k, renormalize)
        ctx.mark_non_differentiable(ids)
        ctx.save_for_backward(weights, ids, None if renormalize else logits)      # (normalised weights do not depend on the experts left out)
        ctx.like, ctx.renormalize = (logits.dtype, *logits.shape, top_k), renormalize
        return weights, ids

    @staticmethod
    def backward(ctx, grad, _):
        weights, ids, logits = ctx.saved_tensors
        dtype, tokens, e, k = ctx.like
        weights, ids = (_unpacked(t, (tokens, k), of, grad, "top_k_gate").contiguous() for t, of in ((weights, torch.float32), (ids, torch.int32)))
        if logits is not None:
            logits = _unpacked(logits, (tokens, e), dtype, grad, "top_k_gate")
        out = torch.empty((tokens, e), dtype=dtype, device=weights.device)
        grad = _lib.stored(grad.detach()).contiguous()
        _lib.call(out.device, "top_k_gate backward", _lib.lib().b200moe_gate_backward, grad.data_ptr(), weights.data_ptr(), ids.data_ptr(), _lib.ptr(logits),
                  _lib.DTYPES[dtype], e if logits is None else max(logits.stride(0), e), tokens, e, k, int(ctx.renormalize), out.data_ptr())
        return _once(out, "top_k_gate"), None, None


def top_k_gate(logits: torch.Tensor, top_k: int, renormalize: bool = True):
    """logits [T, E] bf16, fp16 or fp32 -> (weights f32 [T, top_k], ids int32 [T, top_k]): each token's top_k largest logits in falling order (ties to
    the lowest index) and their softmax probabilities, divided by their sum where `renormalize`. Up to 512 experts and 16 of them a token; rows may be any
    stride apart. A logit of -inf is an expert that may not be taken: a slot for which none is left gets id -1 (an empty slot of the layer calls) and weight 0. A NaN
    ranks above all numbers and makes its token's weights NaN. Differentiable with respect to the logits through the weights."""
    out = (_lib._host or _lib.host()).top_k_gate(logits, top_k, renormalize)      # plain tensors in one native call (csrc/host.cpp), else None
    if out is not None:
        return out if type(out) is tuple else _lib.check(out, "top_k_gate")
    top_k = int(top_k)
    leaf, logits = logits, _logits(logits, "top_k_gate")
    if not 1 <= top_k <= min(MAX_TOP_K, logits.shape[1]):
        raise ValueError(f"top_k_gate takes 1 to {min(MAX_TOP_K, logits.shape[1])} of {logits.shape[1]} experts, not {top_k}")
    _check_capture(leaf, "top_k_gate")
    if logits.requires_grad and torch.is_grad_enabled():
        return _Gate.apply(logits, top_k, bool(renormalize))
    return _gate(logits, top_k, bool(renormalize))


def _balance(logits: torch.Tensor, ids: torch.Tensor):
    tokens, e = logits.shape
    h = _lib.lib()
    nbytes = h.b200moe_balance_workspace_bytes(tokens, e)
    ws = torch.empty(max(nbytes, 4), dtype=torch.uint8, device=logits.device)
    loss, stats = torch.empty((), dtype=torch.float32, device=logits.device), torch.empty(2, dtype=torch.float32, device=logits.device)
    counts = torch.empty(e, dtype=torch.int32, device=logits.device)
    _lib.call(logits.device, "balance_loss", h.b200moe_balance_loss, logits.data_ptr(), _lib.DTYPES[logits.dtype], max(logits.stride(0), e), tokens, e, ids.data_ptr(),
              ids.shape[1], loss.data_ptr(), counts.data_ptr(), stats.data_ptr(), ws.data_ptr(), nbytes)
    return loss, counts, stats


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids):
        loss, counts, stats = _balance(logits, ids)
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(logits, ids, counts, stats)
        ctx.like = (logits.dtype, *logits.shape, ids.shape[1])
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        dtype, tokens, e, k = ctx.like
        logits, ids, counts, stats = (_unpacked(t, shape, of, grad, "balance_loss") for t, shape, of in zip(
            ctx.saved_tensors, ((tokens, e), (tokens, k), (e,), (2,)), (dtype, torch.int32, torch.int32, torch.float32)))
        ids, out = ids.contiguous(), torch.empty((tokens, e), dtype=dtype, device=logits.device)
        grad = _lib.stored(grad.detach()).contiguous()
        _lib.call(out.device, "balance_loss backward", _lib.lib().b200moe_balance_backward, grad.data_ptr(), logits.data_ptr(), _lib.DTYPES[logits.dtype],
                  max(logits.stride(0), e), tokens, e, ids.data_ptr(), ids.shape[1], counts.data_ptr(), stats.data_ptr(), out.data_ptr())
        return _once(out, "balance_loss"), None


def balance_loss(logits: torch.Tensor, ids: torch.Tensor):
    """logits [T, E], ids int32 [T, k] (the router's choice) -> (loss f32 [], counts int32 [E]):
    loss = E * sum_e f_e P_e with f_e expert e's share of all pairs and P_e the mean over tokens of softmax(logits)_e; it is 1 where experts are used
    evenly. counts are the pairs of each expert. An id outside 0..E-1 is an empty slot, and a token of empty slots alone (padding) counts nowhere; without any
    live token the loss is 0. Differentiable with respect to the logits through P (f is a count). k up to 32, experts up to 512, pairs up to 2^31 - 1."""
    out = (_lib._host or _lib.host()).balance_loss(logits, ids)      # (as in top_k_gate)
    if out is not None:
        return out if type(out) is tuple else _lib.check(out, "balance_loss")
    if ids.numel() > MAX_PAIRS:
        raise ValueError(f"balance_loss takes at most {MAX_PAIRS} pairs (counts are of 32 bits), not {ids.numel()}")
    leaf, logits = logits, _logits(logits, "balance_loss")
    if ids.dtype != torch.int32:
        raise TypeError(f"balance_loss takes int32 ids, not {ids.dtype}")
    if ids.dim() != 2 or ids.shape[0] != logits.shape[0] or not 1 <= ids.shape[1] <= 32:
        raise ValueError(f"balance_loss: expected ids [{logits.shape[0]}, 1 to 32], got {tuple(ids.shape)}")
    _lib.one_device("balance_loss", logits, ids)
    ids = _lib.stored(ids).contiguous()
    _check_capture(leaf, "balance_loss")
    if logits.requires_grad and torch.is_grad_enabled():
        return _Balance.apply(logits, ids)
    return _balance(logits, ids)[:2]
