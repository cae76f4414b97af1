"""Products over 16-bit experts chosen per route, and their gradients.

The counterpart of ``vq_switch`` for experts (or single projections of a layer) that stay in fp16 or
bf16, as the reference's ``HighPrecisionSwitchLinear`` (``src/ramp/nn/``) keeps them:

* ``switch_matmul(x, weight, indices)``         ``out[r] = W[e] x[row(r)]``
* ``switch_matmul_grads(grad, x, weight, indices)``  the gradients of ``x`` and ``weight``

``x`` leading shape equals ``indices.shape[:-1]`` (token layout: result ``[..., k, out]``) or
``indices.shape`` (a row per route: result ``[..., out]``), as in ``vq_switch_qmv``.  ``weight`` is
``[experts, out, in]`` in x's dtype, ``in`` a multiple of 8.  Routes may come in any order; an index outside
``[0, experts)`` is a dead route: zeros, and no part of any gradient.  Sums are fp32 with one rounding, in
an order that depends on the call alone: the same call gives the same bits.

``switch_matmul`` records a gradient formula where grad mode is on and an input requires one.  A CUDA graph
captures ``switch_matmul`` under ``torch.no_grad()`` and ``switch_matmul_grads``, not a recorded backward
pass: autograd would tie the capture to the streams of whatever other graphs of the same leaves are alive.
The kernels' waits are bounded: ``switch_matmul_wait_expired`` tells whether one gave up (on a device that has stopped making
progress), after which the outputs since the last time of asking are not to be used.
There are no derivatives of gradients and no forward-mode ones: arguments that carry a tangent are refused.
"""

from __future__ import annotations

from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib
from .vq import as_device

__all__ = ["switch_matmul", "switch_matmul_grads", "switch_matmul_wait_expired"]

_DTYPES = (torch.float16, torch.bfloat16)


def _indices(indices, device) -> torch.Tensor:
    if not (isinstance(indices, torch.Tensor) and indices.dtype in (torch.int32, torch.int64) and indices.device == device):
        indices = as_device(indices, device)
        if indices.dtype.is_floating_point or indices.dtype.is_complex or indices.dtype == torch.bool:
            raise ValueError(f"indices must use an integer dtype, found {indices.dtype}")
        if indices.dtype == torch.uint32:  # 0xFFFFFFFF, a pick without an expert, becomes -1: same bits
            indices = indices.view(torch.int32)
        elif indices.dtype not in (torch.int32, torch.int64):
            indices = indices.to(torch.int64)
    return indices.contiguous()


def _x_div(x_shape, indices_shape, in_dim: int) -> tuple[int, int]:
    """Routes per row of x (1, or the picks of a token), and routes."""
    if len(indices_shape) < 1:
        raise ValueError("indices must have at least one dimension")
    if len(x_shape) < 1 or x_shape[-1] != in_dim:
        raise ValueError(f"x trailing dimension must be {in_dim}, found {tuple(x_shape)}")
    if x_shape[:-1] == indices_shape:
        return 1, indices_shape.numel()
    if x_shape[:-1] == indices_shape[:-1]:
        return indices_shape[-1], indices_shape.numel()
    raise ValueError(
        "x leading shape must either match indices leading shape for "
        f"token routing or the full indices shape for per-route routing; found x {tuple(x_shape)} and indices {tuple(indices_shape)}")


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and on a 16-byte boundary (a view may start inside an allocation)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _grad_rows(grad: torch.Tensor, out_shape: tuple, dtype: torch.dtype) -> tuple[torch.Tensor, int]:
    """The output gradient as rows of a multiple of 8 values, zeros behind its own."""
    if tuple(grad.shape) != out_shape or grad.dtype != dtype:
        raise ValueError(f"grad must be {out_shape} {dtype}, found {tuple(grad.shape)} {grad.dtype}")
    ld = -(-out_shape[-1] // 8) * 8
    return _dense(grad if ld == out_shape[-1] else torch.nn.functional.pad(grad, (0, ld - out_shape[-1]))), ld


def _no_capture(what: str, grads: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise _lib.KeepVQError(f"{what}: a recorded gradient cannot be captured; capture the call under torch.no_grad() and {grads}")


def _no_tangents(what: str, *tensors) -> None:
    """Forward-mode derivatives are not formed: a result without a tangent would read as one that does not depend on its inputs."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _lib.KeepVQError(f"{what} has no forward-mode derivative: an argument carries a tangent")


@lru_cache(maxsize=1024)
def _problem(x_shape, weight_shape, indices_shape, x_dtype, weight_dtype) -> tuple:
    """What follows from shapes and types alone, checked once for each: (routes per row of x, routes, experts, out, in, dtype tag,
    result's shape)."""
    if x_dtype not in _DTYPES or weight_dtype != x_dtype:
        raise ValueError(f"x and weight must share one of fp16 / bf16, found {x_dtype} and {weight_dtype}")
    if len(weight_shape) != 3 or 0 in weight_shape:
        raise ValueError(f"weight must be [experts, out, in], found {tuple(weight_shape)}")
    experts, out_dim, in_dim = weight_shape
    if in_dim % 8 != 0:
        raise ValueError("the input dimension must be divisible by 8")
    x_div, routes = _x_div(x_shape, indices_shape, in_dim)
    return max(x_div, 1), routes, experts, out_dim, in_dim, _lib.dtype_tag(x_dtype), (*indices_shape, out_dim)


@lru_cache(maxsize=1024)
def _scratch_bytes(routes: int, experts: int, out_dim: int, in_dim: int, x_div: int, grads: bool) -> int:
    nbytes = int(_lib.load().keepvq_switch_matmul_workspace_bytes(routes, experts, out_dim, in_dim, x_div, int(grads)))
    if nbytes < 0:
        _lib.check(nbytes, "keepvq_switch_matmul_workspace_bytes")
    return nbytes


def _check(x: torch.Tensor, weight: torch.Tensor, indices):
    shape = indices.shape if isinstance(indices, torch.Tensor) else torch.as_tensor(indices).shape
    problem = _problem(x.shape, weight.shape, shape, x.dtype, weight.dtype)
    device = _lib.require_cuda(x, weight)
    return device, _indices(indices, device), problem


def _call(name: str, device, x, weight, grad, indices, problem, grad_ld, out, dx, dweight):
    x_div, routes, experts, out_dim, in_dim, tag, _ = problem
    nbytes = _scratch_bytes(routes, experts, out_dim, in_dim, x_div, grad is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)  # of this call alone, as every scratch of the operators
    args = _lib.pack_switch_matmul_args(
        x.data_ptr(), weight.data_ptr(), 0 if grad is None else grad.data_ptr(), tag, indices.data_ptr(), 64 if indices.dtype == torch.int64 else 32, x_div, routes,
        experts, out_dim, in_dim, grad_ld, 0 if out is None else out.data_ptr(), 0 if dx is None else dx.data_ptr(), 0 if dweight is None else dweight.data_ptr(),
        ws.data_ptr(), nbytes)
    with _lib.on_device(device):
        _lib.check(getattr(_lib.load(), name)(args, _lib.raw_stream(device)), name)


def _forward(x, weight, indices) -> torch.Tensor:
    device, indices, problem = _check(x, weight, indices)
    out = torch.empty(problem[6], dtype=x.dtype, device=device)
    if problem[1]:
        _call("keepvq_switch_matmul", device, _dense(x), _dense(weight), None, indices, problem, 0, out, None, None)
    return out


def switch_matmul_grads(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, indices, *, x_grad: bool = True,
                        weight_grad: bool = True) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of ``x`` and ``weight`` where ``grad`` is that of ``switch_matmul(x, weight, indices)``,
    in their dtype; None for one that is not wanted.  A row's gradient is the fp32 sum over its picks,
    rounded once; experts without routes get zeros."""
    _no_tangents("switch_matmul_grads", grad, x, weight)
    device, indices, problem = _check(x, weight, indices)
    _lib.require_cuda(x, grad)
    grad, grad_ld = _grad_rows(grad, problem[6], x.dtype)
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if x_grad else None
    dweight = torch.empty(weight.shape, dtype=x.dtype, device=device) if weight_grad else None
    if indices.numel() == 0:
        return dx.zero_() if x_grad else None, dweight.zero_() if weight_grad else None
    if x_grad or weight_grad:
        _call("keepvq_switch_matmul_grads", device, _dense(x), _dense(weight), grad, indices, problem, grad_ld, None, dx, dweight)
    return dx, dweight


class _SwitchMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, indices):
        ctx.save_for_backward(x, weight, indices)
        return _forward(x, weight, indices)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_capture("switch_matmul", "switch_matmul_grads")
        x, weight, indices = ctx.saved_tensors
        dx, dweight = switch_matmul_grads(grad, x, weight, indices, x_grad=ctx.needs_input_grad[0], weight_grad=ctx.needs_input_grad[1])
        return dx, dweight, None


def switch_matmul(x: torch.Tensor, weight: torch.Tensor, indices) -> torch.Tensor:
    """``x`` [tokens, in] with ``indices`` [tokens, k] -> [tokens, k, out]; ``x`` [..., k, in] with
    ``indices`` [..., k] -> [..., k, out]: every route against the expert it names."""
    _no_tangents("switch_matmul", x, weight)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        _lib.require_cuda(x, weight)
        _no_capture("switch_matmul", "switch_matmul_grads")
        return _SwitchMatmul.apply(x, weight, as_device(indices, x.device))
    return _forward(x, weight, indices)


def switch_matmul_wait_expired(device=None) -> bool:
    """True when a bounded wait (2 s) expired in a call of ``switch_matmul`` or its gradients on ``device`` (the current one)
    since this was last asked: outputs of such calls are invalid.  Reads one word back: synchronises the current
    stream; calls on other streams count once they have finished."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise _lib.KeepVQError("keep_b200 operators need a CUDA device; there is no CPU path")
    with _lib.on_device(torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)):
        if torch.cuda.is_current_stream_capturing():
            raise _lib.KeepVQError("switch_matmul_wait_expired: a word cannot be read back inside a graph capture")
        word = torch.empty(1, dtype=torch.int32, device="cuda")
        _lib.check(_lib.load().keepvq_switch_matmul_wait_expired(_lib.ptr(word), _lib.stream_handle(word.device)), "keepvq_switch_matmul_wait_expired")
    return bool(word.item())
