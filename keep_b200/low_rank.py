"""Low-rank products chosen per route, added onto a base: adapters of many requests beside one
projection, or a correction per expert of a routed layer.

* ``switch_low_rank(x, left, right, indices, base=, scale=)``   ``out[r] = base[r] + scale * left[e] (right[e] x[row(r)])``
* ``switch_low_rank_grads(grad, x, left, right, indices, scale=)``   the gradients of ``x``, ``left`` and ``right``
  (that of ``base`` is ``grad`` itself)

Layouts, indices and the rules for captures and derivatives are those of ``dense_switch``; a dead route (a request without an
adapter) leaves its base as it is.  ``left`` is ``[sets, out, rank]``, ``right`` ``[sets, rank, in]``, both in x's
dtype (fp16 or bf16), rank 1 to 128: ranks that are not a multiple of 8 are padded on every call, so a caller
who keeps such adapters pads them once instead.  ``base`` has x's dtype or is fp32, and so has the result;
what flows back through an fp32 result reaches ``base`` as it is and the products rounded to x's dtype (for fp16:
infinite beyond its range, zero below it, as any gradient in that type).
Inner vectors are fp32 sums and enter the second product with 16 bits each (bf16), or with 22 bits of a row's
largest (fp16: their range does not matter).
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from .dense_switch import _DTYPES, _dense, _grad_rows, _indices, _no_capture, _no_tangents, _x_div
from .vq import as_device

__all__ = ["LowRank", "switch_low_rank", "switch_low_rank_grads"]

MAX_RANK = 128
_MAX_PITCH = 1 << 28  # values from one row of a base to the next


@dataclass
class LowRank:
    """A stack of low-rank corrections: ``left`` [sets, out, rank], ``right`` [sets, rank, in], one scale."""

    left: torch.Tensor
    right: torch.Tensor
    scale: float = 1.0

    def __post_init__(self):
        _check_pair(self.left.shape, self.right.shape, self.left.dtype, self.right.dtype)

    def add(self, base: torch.Tensor, x: torch.Tensor, indices) -> torch.Tensor:
        """``base`` plus the correction of the set that each route names."""
        return switch_low_rank(x, self.left, self.right, indices, base=base, scale=self.scale)


def _check_pair(left_shape, right_shape, left_dtype, right_dtype) -> None:
    if left_dtype not in _DTYPES or right_dtype != left_dtype:
        raise ValueError(f"left and right must share one of fp16 / bf16, found {left_dtype} and {right_dtype}")
    if len(left_shape) != 3 or len(right_shape) != 3 or left_shape[0] != right_shape[0] or left_shape[2] != right_shape[1] or 0 in left_shape or 0 in right_shape:
        raise ValueError(f"left must be [sets, out, rank] and right [sets, rank, in], found {tuple(left_shape)} and {tuple(right_shape)}")
    if left_shape[2] > MAX_RANK:
        raise ValueError(f"rank must be at most {MAX_RANK}, found {left_shape[2]}")
    if right_shape[2] % 8 != 0:
        raise ValueError("the input dimension must be divisible by 8")


@lru_cache(maxsize=1024)
def _problem(x_shape, left_shape, right_shape, indices_shape, x_dtype, left_dtype, right_dtype) -> tuple:
    """What follows from shapes and types alone, checked once for each: (routes per row of x, routes, sets, out, in, rank rounded
    up, dtype tag, result's shape, rank)."""
    _check_pair(left_shape, right_shape, left_dtype, right_dtype)
    if x_dtype != left_dtype:
        raise ValueError(f"x must be {left_dtype} as left and right, found {x_dtype}")
    sets, out_dim, rank = left_shape
    x_div, routes = _x_div(x_shape, indices_shape, right_shape[2])
    return max(x_div, 1), routes, sets, out_dim, right_shape[2], -(-rank // 8) * 8, _lib.dtype_tag(x_dtype), (*indices_shape, out_dim), rank


def _check(x, left, right, indices):
    shape = indices.shape if isinstance(indices, torch.Tensor) else torch.as_tensor(indices).shape
    problem = _problem(x.shape, left.shape, right.shape, shape, x.dtype, left.dtype, right.dtype)
    device = _lib.require_cuda(x, left, right)
    return device, _indices(indices, device), problem


def _whole_ranks(left, right):
    """left and right with the rank padded to a multiple of 8 (by zeros, which add nothing)."""
    short = -int(left.shape[2]) % 8
    if short:
        left, right = torch.nn.functional.pad(left, (0, short)), torch.nn.functional.pad(right, (0, 0, 0, short))
    return _dense(left), _dense(right)


@lru_cache(maxsize=1024)
def _scratch_bytes(routes: int, sets: int, out_dim: int, in_dim: int, rank: int, x_div: int, grads: bool) -> int:
    nbytes = int(_lib.load().keepvq_switch_low_rank_workspace_bytes(routes, sets, out_dim, in_dim, rank, x_div, int(grads)))
    if nbytes < 0:
        _lib.check(nbytes, "keepvq_switch_low_rank_workspace_bytes")
    return nbytes


def _call(name, device, x, left, right, grad, indices, problem, grad_ld, scale, out_tag, base, base_ld, out, dx, dleft, dright):
    x_div, routes, sets, out_dim, in_dim, rank, tag, _, ranks = problem
    nbytes = _scratch_bytes(routes, sets, out_dim, in_dim, rank, x_div, grad is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    args = _lib.pack_switch_low_rank_args(
        x.data_ptr(), left.data_ptr(), right.data_ptr(), 0 if grad is None else grad.data_ptr(), tag, indices.data_ptr(), 64 if indices.dtype == torch.int64 else 32,
        x_div, routes, sets, out_dim, in_dim, rank, grad_ld, scale, out_tag, 0 if base is None else base.data_ptr(), base_ld, 0 if out is None else out.data_ptr(), out_dim,
        0 if dx is None else dx.data_ptr(), 0 if dleft is None else dleft.data_ptr(), 0 if dright is None else dright.data_ptr(), 0 if ws is None else ws.data_ptr(), nbytes)
    with _lib.on_device(device):
        _lib.check(getattr(_lib.load(), name)(args, ranks, _lib.raw_stream(device)), name)


def _forward(x, left, right, indices, base, scale) -> torch.Tensor:
    device, indices, problem = _check(x, left, right, indices)
    out_shape, out_tag, base_ld = problem[7], problem[6], 0
    if base is None:
        out = torch.empty(out_shape, dtype=x.dtype, device=device)
    else:
        if base.shape != out_shape or base.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"base must be {out_shape} in {x.dtype} or fp32, found {tuple(base.shape)} {base.dtype}")
        _lib.require_cuda(x, base)
        out = torch.empty(out_shape, dtype=base.dtype, device=device)
        if base.dtype != x.dtype:
            out_tag = _lib.F32
        base_ld = out_shape[-1]
        if not base.is_contiguous():
            # rows may lie apart (one of several projections of a wider product), a row's values may not
            if base.ndim == 2 and base.stride(1) == 1 and base_ld <= base.stride(0) <= _MAX_PITCH:
                base_ld = base.stride(0) if base.shape[0] > 1 else base_ld
            else:
                base = base.contiguous()
    if problem[1]:
        left, right = _whole_ranks(left, right)
        _call("keepvq_switch_low_rank_padded", device, _dense(x), left, right, None, indices, problem, 0, scale, out_tag, base, base_ld, out, None, None, None)
    return out


def switch_low_rank_grads(grad: torch.Tensor, x: torch.Tensor, left: torch.Tensor, right: torch.Tensor, indices, *, scale: float = 1.0,
                          x_grad: bool = True, weight_grad: bool = True):
    """The gradients of ``x``, ``left`` and ``right`` where ``grad`` (in x's dtype) is that of
    ``switch_low_rank(x, left, right, indices, base=..., scale=scale)``; None for those not wanted."""
    _no_tangents("switch_low_rank_grads", grad, x, left, right)
    device, indices, problem = _check(x, left, right, indices)
    _lib.require_cuda(x, grad)
    grad, grad_ld = _grad_rows(grad, problem[7], x.dtype)
    rank = int(left.shape[2])
    left, right = _whole_ranks(left, right)
    empty = lambda t, wanted: torch.empty(t.shape, dtype=x.dtype, device=device) if wanted else None  # noqa: E731
    dx, dleft, dright = empty(x, x_grad), empty(left, weight_grad), empty(right, weight_grad)
    if indices.numel() == 0:
        for t in (dx, dleft, dright):
            if t is not None:
                t.zero_()
    elif x_grad or weight_grad:
        _call("keepvq_switch_low_rank_grads_padded", device, _dense(x), left, right, grad, indices, problem, grad_ld, float(scale), problem[6], None, 0, None, dx, dleft, dright)
    if weight_grad and int(left.shape[2]) != rank:
        dleft, dright = dleft[:, :, :rank].contiguous(), dright[:, :rank].contiguous()
    return dx, dleft, dright


class _SwitchLowRank(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, left, right, indices, base, scale):
        ctx.save_for_backward(x, left, right, indices)
        ctx.scale = scale
        return _forward(x, left, right, indices, base, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_capture("switch_low_rank", "switch_low_rank_grads")
        x, left, right, indices = ctx.saved_tensors
        of_x, of_left, of_right, _, of_base, _ = ctx.needs_input_grad
        dx = dleft = dright = None
        if of_x or of_left or of_right:
            dx, dleft, dright = switch_low_rank_grads(grad.to(x.dtype), x, left, right, indices, scale=ctx.scale, x_grad=of_x, weight_grad=of_left or of_right)
        return dx, dleft if of_left else None, dright if of_right else None, None, grad if of_base else None, None


def switch_low_rank(x: torch.Tensor, left: torch.Tensor, right: torch.Tensor, indices, *, base: torch.Tensor | None = None, scale: float = 1.0) -> torch.Tensor:
    """``x`` [rows, in] with ``indices`` [rows] -> [rows, out] (an adapter per row), or the routed layouts
    of ``dense_switch.switch_matmul``; ``base`` has the result's shape (zeros when None)."""
    _no_tangents("switch_low_rank", x, left, right, base)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, left, right, base)):
        _lib.require_cuda(x, left, right, base)
        _no_capture("switch_low_rank", "switch_low_rank_grads")
        return _SwitchLowRank.apply(x, left, right, as_device(indices, x.device), base, float(scale))
    return _forward(x, left, right, indices, base, float(scale))
