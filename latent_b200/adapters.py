"""Low-rank adapters of many requests beside one shared projection.

``AdapterSet`` lays the adapters out once on the device; ``adapter_project``
multiplies a batch by the shared weight and adds, row by row, the product of
that row's own adapter:

    y[t] = x[t] . W + scale_a (x[t] . A_a) . B_a,   a = ids[t]  (< 0: W alone)

The shared projection is a dense fp16/bf16 matrix (either memory order) or a
packed ``FactorPair``.  The rows of a batch may be single tokens of many
requests or packed prompts, in any order.  An inference operator: inputs that
require a gradient or carry a tangent are refused; a set holds copies of its
factors, detached.  The reference has no adapters; its low-rank
projection is loader/latent_runtime.py:35-36.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .router_train import _no_tangents, _on, _with_workspace
from .runtime import FactorPair, project

__all__ = ["AdapterSet", "adapter_project"]

_TYPES = {torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}


def _tensor(a, device, dtype) -> torch.Tensor:
    return (a.detach() if torch.is_tensor(a) else torch.from_numpy(np.ascontiguousarray(a))).to(device, dtype)


class AdapterSet:
    """Device-resident adapters (A [K, r], B [r, N], scale) of one projection.

    ``adapters``: one triple per adapter (scale may be left out: 1.0), ranks
    may differ.  They are stored at one padded rank (16, 32, 64 or 128; zero
    rows change no finite result) in ``dtype``: A transposed, so that a rank column
    is contiguous, B as given.  Factors that are not finite in ``dtype`` are
    refused: rows of several adapters share tiles in which a foreign factor
    is multiplied by zero.
    """

    def __init__(self, adapters: Sequence[Tuple], device="cuda", dtype: Optional[torch.dtype] = None):
        if not adapters:
            raise ValueError("an AdapterSet needs at least one adapter")
        dev = torch.device(device)
        if dev.type == "cuda" and dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        if dtype is None:
            first = adapters[0][0]
            dtype = first.dtype if torch.is_tensor(first) and first.dtype in _TYPES else torch.bfloat16
        if dtype not in _TYPES:
            raise ValueError(f"adapter dtype {dtype} unsupported (float16 or bfloat16)")
        K, N = int(adapters[0][0].shape[0]), int(adapters[0][1].shape[1])
        rmax = 0
        for ad in adapters:
            a, b = ad[0], ad[1]
            if a.ndim != 2 or b.ndim != 2 or a.shape[0] != K or b.shape[1] != N or a.shape[1] != b.shape[0] or \
                    a.shape[1] < 1:
                raise ValueError(f"adapter factors {tuple(a.shape)}, {tuple(b.shape)} do not match [{K}, r], [r, {N}]")
            rmax = max(rmax, int(a.shape[1]))
        rank = 16
        while rank < rmax:
            rank *= 2
        if rank > 128:
            raise ValueError(f"adapter rank {rmax} unsupported (at most 128)")
        n = len(adapters)
        self.device, self.dtype, self.rank = dev, dtype, rank
        self.n_adapter, self.n_in, self.n_out = n, K, N
        self.ranks = [int(ad[0].shape[1]) for ad in adapters]
        # rows padded to 16 bytes
        self.a = torch.zeros((n, rank, (K + 7) // 8 * 8), dtype=dtype, device=dev)
        self.b = torch.zeros((n, rank, (N + 7) // 8 * 8), dtype=dtype, device=dev)
        # one copy per factor kind: A's columns and B's rows side by side, then to their padded places
        live = torch.tensor([i * rank + j for i in range(n) for j in range(self.ranks[i])], device=dev)
        self.a.view(n * rank, -1)[live, :K] = torch.cat([_tensor(ad[0], dev, dtype) for ad in adapters], 1).t()
        self.b.view(n * rank, -1)[live, :N] = torch.cat([_tensor(ad[1], dev, dtype) for ad in adapters], 0)
        scales = [float(ad[2]) if len(ad) > 2 else 1.0 for ad in adapters]
        self.scale = torch.tensor(scales, dtype=torch.float32, device=dev)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        # (reads the result: a set can be used on any stream from here on)
        if not bool(torch.isfinite(self.scale).all() & torch.isfinite(self.a).all() & torch.isfinite(self.b).all()):
            raise ValueError(f"adapter factors must be finite in {dtype}, scales in float32")
        # a, lda, b, ldb, scale as a call's descriptor takes them
        self._factors = (self.a.data_ptr(), self.a.shape[2], self.b.data_ptr(), self.b.shape[2], self.scale.data_ptr())
        self._err_ptr = self.err.data_ptr()
        self._type = _TYPES[dtype]
        self._keep = (self.a, self.b, self.scale, self.err)
        self._ws = {}

    def workspace_bytes(self, n_tokens: int) -> int:
        """Workspace a call on this many rows needs (latent_adapter_workspace_size)."""
        n = self._ws.get(n_tokens)
        if n is None:
            d = _lib.AdapterDesc(self.n_adapter, self.rank, self.n_in, self.n_out, n_tokens, _TYPES[self.dtype],
                                 _TYPES[self.dtype])
            size = C.c_size_t(0)
            _lib.check(_lib.lib().latent_adapter_workspace_size(C.byref(d), C.byref(size)),
                       "latent_adapter_workspace_size")
            n = size.value
            if len(self._ws) < 4096:
                self._ws[n_tokens] = n
        return n

    def check(self) -> None:
        """Synchronises the current stream and raises if a call ordered before on it recorded a device-side error
        since the last check (an id >= n_adapter, which counts as no adapter, or a bounded wait that ran out).
        Errors of calls still on their way on other streams are raised now or by the next check, never lost."""
        _lib.check(_on(self.device, _lib.lib().latent_adapter_check, self.err.data_ptr()), "device check")


def adapter_project(x: torch.Tensor, weight, adapters: AdapterSet, ids: torch.Tensor,
                    out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x . W plus each row's own adapter (latent_adapter_project).

    x [T, K] in the set's dtype (rows may be strided); ``weight`` [K, N] of
    the same dtype, row-major or the transposed view of a linear layer's
    [N, K] weight, or a ``FactorPair`` (its fp32 ``project`` is then summed
    with the adapters' part in fp32); ids int32 [T], negative: no adapter,
    >= n_adapter: none either, and ``adapters.check()`` reports it.  Returns
    [T, N] in ``out_dtype`` (x's dtype or float32; x's by default), fp32 sums
    rounded once, or fills ``out`` (rows may be strided; it must not share
    memory with the inputs).

    The tensor cores need rows of x and of the weight that start at multiples
    of 16 bytes (N itself may be odd); others run on the CUDA cores, 20 to 70
    times slower.
    """
    s = adapters
    dev, dt, K, N = s.device, s.dtype, s.n_in, s.n_out
    shape = x.shape
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f"x must be [T, {K}], got {tuple(shape)}")
    if x.dtype != dt:
        raise ValueError(f"x must be {dt} like the adapters, got {x.dtype}")
    T = shape[0]
    if ids.shape != (T,) or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise ValueError(f"ids must be contiguous int32 [{T}]")
    pair = isinstance(weight, FactorPair)
    if not pair and (weight.shape != (K, N) or weight.dtype != dt):
        raise ValueError(f"weight must be {dt} [{K}, {N}]")
    if x.device != dev or ids.device != dev or (not pair and weight.device != dev) or \
            (out is not None and out.device != dev) or not x.is_cuda:
        raise ValueError("x, weight, ids and out must be on the adapters' device, a CUDA device")
    if (x.requires_grad or (not pair and weight.requires_grad) or (out is not None and out.requires_grad)) and \
            torch.is_grad_enabled():
        raise ValueError("adapter_project computes no gradients: call it under torch.no_grad() or on detached tensors")
    _no_tangents("adapter_project", x, None if pair else weight, out)
    if out is not None:
        if out_dtype not in (None, out.dtype):
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        out_dtype = out.dtype
        if tuple(out.shape) != (T, N) or (N > 1 and out.stride(1) != 1) or (T > 1 and out.stride(0) < N):
            raise ValueError(f"out must be [{T}, {N}] with contiguous rows")
    if out_dtype is None or out_dtype == dt:
        out_dtype, y_type = dt, s._type
    elif out_dtype == torch.float32:
        y_type = _lib.TYPE_F32
    else:
        raise ValueError(f"out_dtype {out_dtype} unsupported ({dt} or float32)")
    if T == 0:
        return out if out is not None else torch.empty((0, N), dtype=out_dtype, device=dev)
    ldx, inner = x.stride()
    if (inner != 1 and K > 1) or (T > 1 and ldx < K):
        x = x.contiguous()
        ldx = K
    if T == 1:
        ldx = (K + 7) // 8 * 8  # no second row: a stride that tensor maps take
    flags, w_ptr, ldw = 0, 0, 0
    if pair:
        y = project(x, weight)
        if y.shape[1] != N:
            raise ValueError(f"the factor pair has {y.shape[1]} columns, the adapters {N}")
    else:
        ws0, ws1 = weight.stride()
        if (ws1 == 1 or N == 1) and (ws0 >= N or K == 1):
            ldw = max(ws0, N)
        elif (ws0 == 1 or K == 1) and (ws1 >= K or N == 1):
            flags, ldw = _lib.ADAPTER_W_TRANSPOSED, max(ws1, K)
        else:
            raise ValueError("weight must be row-major or the transposed view of a row-major matrix")
        w_ptr = weight.data_ptr()
        y = out if out is not None else torch.empty(T, N, dtype=out_dtype, device=dev)
    if pair:
        y_type = _lib.TYPE_F32
    _with_workspace(dev, s._ws.get(T) or s.workspace_bytes(T), _lib.lib().latent_adapter_project,
                    "latent_adapter_project", _lib.ADAPTER_DESC,
                    (s.n_adapter, s.rank, K, N, T, s._type, y_type, flags, x.data_ptr(), ldx, w_ptr, ldw, *s._factors,
                     ids.data_ptr(), y.data_ptr(), y.stride(0) if T > 1 else N, s._err_ptr))
    if pair:
        return y.to(out_dtype) if out is None else out.copy_(y)
    return y
