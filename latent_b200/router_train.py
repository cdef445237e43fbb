"""Training side of the router: the balance loss with its gradient, and the gradient of the routing weights.

For recalibrating the router of a compressed layer (the experts stay packed
and frozen): ``router_topk`` routes the logits, ``ExpertFFN`` runs the
experts (its per-slot rows give d_weights = <d_out, y_slot>),
``router_topk_grad`` carries that back to the logits and ``balance_loss``
adds the load-balance and z losses.  The reference has no training code.
Both kernels return explicit gradients, which add up in one buffer
(``out=``) and can be captured into a CUDA graph.  Where autograd is on and
the logits require a gradient, ``balance_loss`` and, when asked,
``router_topk`` are differentiable through it as well (outside graph capture).
The explicit gradients are constants to autograd; forward-mode tangents are
refused.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .runtime import _X_TYPES

__all__ = ["BalanceLoss", "balance_loss", "router_topk_grad"]


class BalanceLoss(NamedTuple):
    """What ``balance_loss`` returns."""

    loss: torch.Tensor             # balance_coef * balance + z_coef * z, 0-dim fp32
    balance: torch.Tensor          # 0-dim fp32
    z: torch.Tensor                # 0-dim fp32
    counts: torch.Tensor           # kept slots per expert, int32 [S, E] ([E] without cu_seqlens)
    grad: Optional[torch.Tensor]   # d loss / d logits in the logits' dtype, with gradient=True


def _on(device: torch.device, fn, *args) -> int:
    """Calls a C entry point with ``device`` current (kernels launch on the current device), on its current stream."""
    index = device.index
    if torch.cuda.current_device() == index:
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(device):
        return fn(*args, _raw_stream(index))


def _raw_stream(index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index)


def _with_workspace(device: torch.device, size: int, fn, what: str, desc, fields) -> None:
    """Calls ``fn`` on the descriptor ``fields`` + (workspace, size), with ``device`` current, on its current stream.

    The workspace is the caching allocator's memory of that stream, as a tensor's would be (a captured call's comes
    from its graph's pool), given back behind the call; without a tensor around it, which costs 1 us of a call's 9."""
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(device):
            return _with_workspace(device, size, fn, what, desc, fields)
    stream = _raw_stream(index)
    ws = torch._C._cuda_cudaCachingAllocator_raw_alloc(size, stream)
    try:
        _lib.check(fn(desc.pack(*fields, ws, size), stream), what)
    finally:
        torch._C._cuda_cudaCachingAllocator_raw_delete(ws)


_WS_BYTES = {}    # workspace size by (sequences, experts)


def _workspace_bytes(n_seq: int, n_expert: int) -> int:
    n = _WS_BYTES.get((n_seq, n_expert))
    if n is None:
        size = C.c_size_t(0)
        d = _lib.BalanceDesc(n_sequences=n_seq, n_expert=n_expert)
        _lib.check(_lib.lib().latent_balance_workspace_size(C.byref(d), C.byref(size)), "latent_balance_workspace_size")
        n = size.value
        if len(_WS_BYTES) < 4096:
            _WS_BYTES[n_seq, n_expert] = n
    return n


def _router_inputs(logits: torch.Tensor, ids: torch.Tensor, name: str):
    """(logits, ids) contiguous, T, E, k, latent_type; raises ValueError on anything else than [T, E] and int32 [T, k]."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    shape, slots = logits.shape, ids.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{name} must be [T, E], got {tuple(shape)}")
    kind = _X_TYPES.get(logits.dtype)
    if kind is None:
        raise ValueError(f"{name} dtype {logits.dtype} unsupported")
    if len(slots) != 2 or slots[0] != shape[0] or slots[1] < 1 or ids.dtype != torch.int32:
        raise ValueError("ids must be int32 [T, k]")
    if ids.get_device() != logits.get_device():
        raise ValueError(f"ids must be on {logits.device}")
    return logits.contiguous(), ids.contiguous(), shape[0], shape[1], slots[1], kind


def _no_tangents(what: str, *tensors) -> None:
    """Raises where one of the tensors carries a forward-mode tangent, which ``what`` would drop."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise ValueError(f"{what} has no forward-mode derivative: its inputs must not carry tangents")


def _no_capture(what: str) -> None:
    # Autograd ties a leaf's gradient to the stream that first used it: a
    # captured backward pass beside an eager one of the same leaves would end
    # the process.  The explicit gradients capture.
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} is not differentiated by autograd during graph capture: pass detached logits and "
                           "use the explicit gradient")


def _balance(logits, ids, balance_coef, z_coef, valid, cu, n_seq, gradient, d_losses=None):
    T, E = logits.shape
    dev = logits.device
    n = _WS_BYTES.get((n_seq, E)) or _workspace_bytes(n_seq, E)
    losses = torch.empty(3, dtype=torch.float32, device=dev)
    # [E] when the rows are one sequence without borders
    counts = torch.empty(E, dtype=torch.int32, device=dev) if cu is None else \
        torch.empty(n_seq, E, dtype=torch.int32, device=dev)
    grad = torch.empty_like(logits) if gradient else None
    _with_workspace(dev, n, _lib.lib().latent_balance_loss, "latent_balance_loss", _lib.BALANCE_DESC,
                    (T, E, ids.shape[1], n_seq, _X_TYPES[logits.dtype], 0 if d_losses is None else _lib.BALANCE_D_LOSSES,
                     balance_coef, z_coef, logits.data_ptr(),
                     ids.data_ptr(), 0 if valid is None else valid.data_ptr(), 0 if cu is None else cu.data_ptr(),
                     0 if d_losses is None else d_losses.data_ptr(), losses.data_ptr(), counts.data_ptr(),
                     0 if grad is None else grad.data_ptr()))
    return losses, counts, grad


class _BalanceLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, balance_coef, z_coef, valid, cu, n_seq):
        _no_capture("balance_loss")
        flat = logits.detach().contiguous()
        losses, counts, _ = _balance(flat, ids, balance_coef, z_coef, valid, cu, n_seq, False)
        ctx.save_for_backward(flat, ids, valid, cu)
        ctx.args = (balance_coef, z_coef, n_seq)
        ctx.mark_non_differentiable(counts)
        return losses, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_losses, _):
        _no_capture("balance_loss")
        flat, ids, valid, cu = ctx.saved_tensors
        balance_coef, z_coef, n_seq = ctx.args
        d = d_losses.to(torch.float32).contiguous()
        grad = _balance(flat, ids, balance_coef, z_coef, valid, cu, n_seq, True, d)[2]
        return grad, None, None, None, None, None, None


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, balance_coef: float = 0.01, z_coef: float = 0.0,
                 valid: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                 gradient: bool = False) -> BalanceLoss:
    """Load-balance and z losses of a router, the expert counts and the gradient (latent_balance_loss).

    logits [T, E] fp32, bf16 or fp16 on a CUDA device, ids int32 [T, k] as
    ``router_topk`` returns them (negative: dropped slot).  ``cu_seqlens``
    int32 [S + 1]: the balance loss is taken per packed sequence and averaged
    over the sequences that have a row; rows behind the last one take no
    part.  ``valid`` bool [T]: False marks padded rows, which take no part
    whatever they hold.  The loss is
    ``balance_coef * mean_s E sum_e f_se P_se + z_coef * mean_t logsumexp^2``
    with f the share of the kept slots and P the mean softmax probability.

    With ``gradient`` the result carries d loss / d logits (the logits'
    dtype), made in the same pass.  An fp16 gradient of a mean over many rows
    underflows: scale the two coefficients up.  The losses beside it are constants
    to autograd.  Without it, logits that require a gradient make ``loss``,
    ``balance`` and ``z`` differentiable by autograd.
    """
    flat, ids, T = _router_inputs(logits, ids, "logits")[:3]
    _no_tangents("balance_loss", logits)
    n_seq = 1
    if cu_seqlens is not None:
        n_seq = cu_seqlens.numel() - 1
        if cu_seqlens.dim() != 1 or n_seq < 1 or cu_seqlens.dtype != torch.int32 or \
                cu_seqlens.get_device() != flat.get_device():
            raise ValueError(f"cu_seqlens must be int32 [S + 1] on {flat.device}")
        cu_seqlens = cu_seqlens.contiguous()
    if valid is not None:
        if tuple(valid.shape) != (T,) or valid.dtype != torch.bool or valid.get_device() != flat.get_device():
            raise ValueError(f"valid must be bool [{T}] on {flat.device}")
        valid = valid.contiguous()
    balance_coef, z_coef = float(balance_coef), float(z_coef)
    if not gradient and logits.requires_grad and torch.is_grad_enabled():
        losses, counts = _BalanceLossFn.apply(logits, ids, balance_coef, z_coef, valid, cu_seqlens, n_seq)
        # one by one: of views made in one call none may be changed in place
        loss, balance, z, grad = losses[0], losses[1], losses[2], None
    else:
        losses, counts, grad = _balance(flat, ids, balance_coef, z_coef, valid, cu_seqlens, n_seq, gradient)
        loss, balance, z = losses.unbind()
    return BalanceLoss(loss, balance, z, counts, grad)


def router_topk_grad(scores: torch.Tensor, ids: torch.Tensor, d_weights: torch.Tensor, renormalize: bool = True,
                     logits: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``router_topk``'s weights with respect to its scores (latent_router_grad).

    ``scores`` [T, E], ``renormalize`` and ``logits`` as given to
    ``router_topk``, ``ids`` int32 [T, k] as it returned them, ``d_weights``
    fp32 [T, k].  Returns [T, E] in the scores' dtype; the kept set is held
    fixed.  ``out``: a contiguous tensor of the scores' shape and dtype that
    the gradient is added into (for instance ``balance_loss(...).grad``); it
    shares no memory with the inputs.  The result is a constant to autograd,
    whether or not ``scores`` or ``d_weights`` require a gradient.
    """
    flat, ids, T, E, k, kind = _router_inputs(scores, ids, "scores")
    if d_weights.shape != ids.shape or d_weights.dtype != torch.float32 or d_weights.get_device() != flat.get_device():
        raise ValueError(f"d_weights must be float32 {tuple(ids.shape)} on {flat.device}")
    _no_tangents("router_topk_grad", scores, d_weights, out)
    flags = (_lib.ROUTER_RENORMALIZE if renormalize else 0) | (_lib.ROUTER_SOFTMAX if logits else 0)
    if out is None:
        g = torch.empty_like(flat)   # (never carries requires_grad)
    else:
        if out.shape != flat.shape or out.dtype != flat.dtype or out.device != flat.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {flat.dtype} {tuple(flat.shape)} tensor on {flat.device}")
        if out.data_ptr() == flat.data_ptr() and flat.numel():
            raise ValueError("out must not be the scores")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out must not require a gradient")
        flags |= _lib.ROUTER_ACCUMULATE
        g = out
    d_weights = d_weights.contiguous()
    d = _lib.ROUTER_GRAD_DESC.pack(T, E, k, kind, flags, 0, flat.data_ptr(), ids.data_ptr(), d_weights.data_ptr(),
                                   g.data_ptr())
    _lib.check(_on(flat.device, _lib.lib().latent_router_grad, d), "latent_router_grad")
    return g


class RouterTopK(torch.autograd.Function):
    """``router_topk(..., differentiable=True)``: weights that autograd can differentiate."""

    @staticmethod
    def forward(ctx, scores, top_k, threshold, renormalize, logits, expert_counts):
        from .runtime import router_topk
        _no_capture("router_topk")
        flat = scores.detach().contiguous()
        out = router_topk(flat, top_k, threshold, renormalize, logits, expert_counts)
        ids, w, n_kept = out[:3]
        counts = out[3] if expert_counts else None
        ctx.save_for_backward(flat, ids)
        ctx.args = (renormalize, logits)
        ctx.mark_non_differentiable(ids, n_kept, *([counts] if expert_counts else []))
        return ids, w, n_kept, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_ids, d_w, *_):
        _no_capture("router_topk")
        flat, ids = ctx.saved_tensors
        renormalize, logits = ctx.args
        exact = flat if flat.dtype in _X_TYPES else flat.to(torch.float32)
        g = router_topk_grad(exact, ids, d_w.to(torch.float32), renormalize, logits)
        return g.to(flat.dtype), None, None, None, None, None
