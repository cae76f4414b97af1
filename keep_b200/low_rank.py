"""Low-rank products chosen per route, added onto a base: adapters of many requests beside one
projection, or a correction per expert of a routed layer.

* ``switch_low_rank(x, left, right, indices, base=, scale=)``   ``out[r] = base[r] + scale * left[e] (right[e] x[row(r)])``
* ``switch_low_rank_grads(grad, x, left, right, indices, scale=)``   the gradients of ``x``, ``left`` and ``right``
  (that of ``base`` is ``grad`` itself)

Layouts, indices and the rules for captures are those of ``dense_switch``; a dead route (a request without an
adapter) leaves its base as it is.  ``left`` is ``[sets, out, rank]``, ``right`` ``[sets, rank, in]``, both in x's
dtype (fp16 or bf16), rank 1 to 128: ranks that are not a multiple of 8 are padded on every call, so a caller
who keeps such adapters pads them once instead.  ``base`` has x's dtype or is fp32, and so has the result.
Inner vectors are fp32 sums and enter the second product with 16 (bf16) or 22 (fp16) bits.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from .dense_switch import _DTYPES, _dense, _grad_rows, _indices, _no_capture, _x_div
from .vq import as_device

__all__ = ["LowRank", "switch_low_rank", "switch_low_rank_grads"]

MAX_RANK = 128


@dataclass
class LowRank:
    """A stack of low-rank corrections: ``left`` [sets, out, rank], ``right`` [sets, rank, in], one scale."""

    left: torch.Tensor
    right: torch.Tensor
    scale: float = 1.0

    def __post_init__(self):
        _check_pair(self.left, self.right)

    def add(self, base: torch.Tensor, x: torch.Tensor, indices) -> torch.Tensor:
        """``base`` plus the correction of the set that each route names."""
        return switch_low_rank(x, self.left, self.right, indices, base=base, scale=self.scale)


def _check_pair(left, right) -> None:
    if left.dtype not in _DTYPES or right.dtype != left.dtype:
        raise ValueError(f"left and right must share one of fp16 / bf16, found {left.dtype} and {right.dtype}")
    if left.ndim != 3 or right.ndim != 3 or left.shape[0] != right.shape[0] or left.shape[2] != right.shape[1] or 0 in left.shape or 0 in right.shape:
        raise ValueError(f"left must be [sets, out, rank] and right [sets, rank, in], found {tuple(left.shape)} and {tuple(right.shape)}")
    if int(left.shape[2]) > MAX_RANK:
        raise ValueError(f"rank must be at most {MAX_RANK}, found {int(left.shape[2])}")
    if int(right.shape[2]) % 8 != 0:
        raise ValueError("the input dimension must be divisible by 8")


def _check(x, left, right, indices):
    _check_pair(left, right)
    if x.dtype != left.dtype:
        raise ValueError(f"x must be {left.dtype} as left and right, found {x.dtype}")
    device = _lib.require_cuda(x, left, right)
    indices = _indices(indices, device)
    x_div = _x_div(x, indices, int(right.shape[2]))
    return device, indices, x_div, tuple(indices.shape) + (int(left.shape[1]),)


def _whole_ranks(left, right):
    """left and right with the rank padded to a multiple of 8 (by zeros, which add nothing)."""
    short = -int(left.shape[2]) % 8
    if short:
        left, right = torch.nn.functional.pad(left, (0, short)), torch.nn.functional.pad(right, (0, 0, 0, short))
    return _dense(left), _dense(right)


@lru_cache(maxsize=256)
def _scratch_bytes(routes: int, sets: int, out_dim: int, in_dim: int, rank: int, x_div: int, grads: bool) -> int:
    nbytes = int(_lib.load().keepvq_switch_low_rank_workspace_bytes(routes, sets, out_dim, in_dim, rank, x_div, int(grads)))
    if nbytes < 0:
        _lib.check(nbytes, "keepvq_switch_low_rank_workspace_bytes")
    return nbytes


def _call(name, device, x, left, right, grad, indices, x_div, grad_ld, scale, out_dtype, base, base_ld, out, dx, dleft, dright):
    (sets, out_dim, rank), in_dim, routes = (int(s) for s in left.shape), int(right.shape[2]), indices.numel()
    nbytes = _scratch_bytes(routes, sets, out_dim, in_dim, rank, max(x_div, 1), grad is not None)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    address = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    args = _lib.pack_switch_low_rank_args(
        x.data_ptr(), left.data_ptr(), right.data_ptr(), address(grad), _lib.dtype_tag(x.dtype), indices.data_ptr(), 8 * indices.element_size(), max(x_div, 1),
        routes, sets, out_dim, in_dim, rank, grad_ld, float(scale), _lib.dtype_tag(out_dtype), address(base), base_ld, address(out), out_dim,
        address(dx), address(dleft), address(dright), ws.data_ptr(), nbytes)
    with _lib.on_device(device):
        _lib.check(getattr(_lib.load(), name)(args, _lib.stream_handle(device)), name)


def _forward(x, left, right, indices, base, scale) -> torch.Tensor:
    device, indices, x_div, out_shape = _check(x, left, right, indices)
    out_dtype, base_ld, rows = x.dtype, 0, None
    if base is not None:
        _lib.require_cuda(x, base)
        if tuple(base.shape) != out_shape or base.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"base must be {out_shape} in {x.dtype} or fp32, found {tuple(base.shape)} {base.dtype}")
        out_dtype = base.dtype
        # rows may lie apart (one of several projections of a wider product), a row's values may not
        rows = base if base.ndim == 2 and base.stride(1) == 1 and base.stride(0) >= out_shape[-1] else base.contiguous()
        base_ld = rows.stride(0) if rows.ndim == 2 and rows.shape[0] > 1 else out_shape[-1]
    out = torch.empty(out_shape, dtype=out_dtype, device=device)
    if out.numel():
        left, right = _whole_ranks(left, right)
        _call("keepvq_switch_low_rank", device, _dense(x), left, right, None, indices, x_div, 0, scale, out_dtype, rows, base_ld, out, None, None, None)
    return out


def switch_low_rank_grads(grad: torch.Tensor, x: torch.Tensor, left: torch.Tensor, right: torch.Tensor, indices, *, scale: float = 1.0,
                          x_grad: bool = True, weight_grad: bool = True):
    """The gradients of ``x``, ``left`` and ``right`` where ``grad`` (in x's dtype) is that of
    ``switch_low_rank(x, left, right, indices, base=..., scale=scale)``; None for those not wanted."""
    device, indices, x_div, out_shape = _check(x, left, right, indices)
    _lib.require_cuda(x, grad)
    grad, grad_ld = _grad_rows(grad, out_shape, x.dtype)
    rank = int(left.shape[2])
    left, right = _whole_ranks(left, right)
    empty = lambda t, wanted: torch.empty(t.shape, dtype=x.dtype, device=device) if wanted else None  # noqa: E731
    dx, dleft, dright = empty(x, x_grad), empty(left, weight_grad), empty(right, weight_grad)
    if indices.numel() == 0:
        for t in (dx, dleft, dright):
            if t is not None:
                t.zero_()
    elif x_grad or weight_grad:
        _call("keepvq_switch_low_rank_grads", device, _dense(x), left, right, grad, indices, x_div, grad_ld, scale, x.dtype, None, 0, None, dx, dleft, dright)
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
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, left, right, base)):
        _lib.require_cuda(x, left, right, base)
        _no_capture("switch_low_rank", "switch_low_rank_grads")
        return _SwitchLowRank.apply(x, left, right, as_device(indices, x.device), base, float(scale))
    return _forward(x, left, right, indices, base, float(scale))
