"""Holders for stacked experts: one switch projection (E8P codes, or 16-bit weights), and the gate/up/down
trio of a routed MLP.

Mirrors of ``QuantizedVQSwitchLinear`` (``src/ramp/nn/switch_linear.py:93-571``) and
``QuantizedVQSwitchGLU`` (``src/ramp/models/glm4_moe_adapter.py:113-390``) over ``torch.Tensor``
on a CUDA device: the same constructor keywords, shape rules, error messages and call layouts.

What they hold is the hot path only: codes, scales, codebook, optional bias and the continuous
scale / output-bias sidecars.  The reference's other sidecars (low-rank and sparse residual rows,
RHT signs, rotation matrices) and ``from_weights`` (the RTN encoder) belong to conversion and
quality tooling; passing one raises ``NotImplementedError`` rather than being ignored.

``HighPrecisionSwitchLinear`` is the holder of a projection that stays in fp16 or bf16 (``src/ramp/nn/``); it
takes the place of a quantised one in ``QuantizedVQSwitchGLU``.  Either takes ``low_rank``, a
``low_rank.LowRank`` with one correction per expert that is added to its outputs.
"""

from __future__ import annotations

from typing import Callable

import torch

from . import _lib
from .dense_switch import _indices, _no_tangents, switch_matmul
from .kernels import e8p_m1_per_route, e8p_m1_token_layout, should_use_e8p_m1
from .low_rank import LowRank
from .vq import table_on
from .vq_switch import gather_vqmm, vq_switch_qmv

_ROUTE_STRATEGIES = ("auto", "direct", "sorted_tiled", "per_route_decoded")
_OUTSIDE = ("continuous_low_rank_left", "continuous_low_rank_right", "sparse_residual_expert_indices",
            "sparse_residual_output_indices", "sparse_residual_values", "rht_signs", "rotation_matrix")


def _check_low_rank(low_rank: LowRank | None, num_experts: int, output_dims: int, input_dims: int) -> None:
    if low_rank is not None:
        found = (int(low_rank.left.shape[0]), int(low_rank.left.shape[1]), int(low_rank.right.shape[2]))
        if found != (num_experts, output_dims, input_dims):
            raise ValueError(f"low_rank must correct (experts, out, in) = {(num_experts, output_dims, input_dims)}, found {found}")


def _refuse_gradient(x: torch.Tensor) -> None:
    """The product over codes has no gradient formula.  By itself its result requires no gradient, and a backward pass fails;
    beside an operator that records one, x would silently be left with that operator's part."""
    if x.requires_grad and torch.is_grad_enabled():
        raise _lib.KeepVQError("QuantizedVQSwitchLinear: the product over codes has no gradient, so its input cannot require one beside operators that "
                               "record theirs (low_rank, 16-bit projections); detach it, or call under torch.no_grad()")
    _no_tangents("QuantizedVQSwitchLinear", x)


class QuantizedVQSwitchLinear:
    """Switch-linear layer backed by stacked E8 VQ expert tensors.

    ``x [..., in]`` with ``indices [..., k]`` (token layout) gives ``[..., k, out]``; ``x [..., k, in]``
    with ``indices [..., k]`` (one row per route) gives the same shape.  With ``low_rank`` the factors are
    recorded by autograd where they require a gradient; an ``x`` that requires one is refused, for the
    product over codes has none.
    """

    def __init__(self, *, input_dims: int, output_dims: int, num_experts: int, codes: torch.Tensor, scales: torch.Tensor,
                 codebook: torch.Tensor | None = None, bias: torch.Tensor | None = None, group_size: int = 512,
                 code_bits: int = 8, use_gather_vqmm: bool = True, route_strategy: str = "auto",
                 gather_codebook_duplication: int = 8, continuous_scale_delta: torch.Tensor | None = None,
                 continuous_output_bias: torch.Tensor | None = None, low_rank: LowRank | None = None, **outside):
        for name, value in outside.items():
            if name not in _OUTSIDE:
                raise TypeError(f"unexpected keyword argument {name!r}")
            if value is not None:
                raise NotImplementedError(f"{name} belongs to the conversion tooling, not to the routed hot path")
        if input_dims <= 0 or output_dims <= 0 or num_experts <= 0:
            raise ValueError("input_dims, output_dims, and num_experts must be positive")
        if input_dims % 8 != 0:
            raise ValueError("input_dims must be divisible by 8")
        if input_dims % group_size != 0:
            raise ValueError("input_dims must be divisible by group_size")
        if code_bits not in (8, 16):
            raise ValueError("code_bits must be 8 or 16")
        if gather_codebook_duplication not in (1, 4, 8):
            raise ValueError("gather_codebook_duplication must be 1, 4, or 8")
        if route_strategy not in _ROUTE_STRATEGIES:
            raise ValueError("route_strategy must be 'auto', 'direct', 'sorted_tiled', or 'per_route_decoded'")
        expected_codes = (num_experts, output_dims, input_dims // 8)
        if tuple(codes.shape) != expected_codes:
            raise ValueError(f"codes must have shape {expected_codes}, found {tuple(codes.shape)}")
        expected_scales = (num_experts, output_dims, input_dims // group_size)
        if tuple(scales.shape) != expected_scales:
            raise ValueError(f"scales must have shape {expected_scales}, found {tuple(scales.shape)}")
        if bias is not None and tuple(bias.shape) != (num_experts, output_dims):
            raise ValueError(f"bias must have shape {(num_experts, output_dims)}, found {tuple(bias.shape)}")
        _check_low_rank(low_rank, num_experts, output_dims, input_dims)
        _lib.require_cuda(codes, scales)
        self.low_rank = low_rank
        self.input_dims, self.output_dims, self.num_experts = int(input_dims), int(output_dims), int(num_experts)
        self.group_size, self.code_bits = int(group_size), int(code_bits)
        self.use_gather_vqmm, self.route_strategy = bool(use_gather_vqmm), route_strategy
        self.gather_codebook_duplication = int(gather_codebook_duplication)
        if codebook is None:  # the default table of the code width, as the reference's holder resolves it
            codebook = table_on(codes.device, "e8p" if code_bits == 16 else "e8_1bit")
        self.codes, self.scales, self.codebook, self.bias = codes, scales, codebook, bias
        self.continuous_scale_delta = None if continuous_scale_delta is None else continuous_scale_delta.float()
        self.continuous_output_bias = None if continuous_output_bias is None else continuous_output_bias.float()

    @property
    def route_backend(self) -> str:
        return f"gather_vqmm_{self.route_strategy}" if self.use_gather_vqmm else "scalar_qmv"

    @property
    def has_continuous_sidecar(self) -> bool:
        return self.continuous_scale_delta is not None or self.continuous_output_bias is not None

    @property
    def has_sparse_residual_rows(self) -> bool:
        return False

    def effective_scales(self) -> torch.Tensor:
        """``scales * exp(continuous_scale_delta)`` in fp32 when the sidecar is set (``switch_linear.py:282-286``)."""
        if self.continuous_scale_delta is None:
            return self.scales
        return self.scales.float() * torch.exp(self.continuous_scale_delta)

    def __call__(self, x: torch.Tensor, indices: torch.Tensor, *, sorted_indices: bool = False) -> torch.Tensor:
        if self.low_rank is not None:
            _refuse_gradient(x)
        scales = self.effective_scales()
        common = dict(input_dims=self.input_dims, output_dims=self.output_dims, group_size=self.group_size, code_bits=self.code_bits)
        token_layout = x.ndim >= 2 and indices.ndim >= 2 and tuple(x.shape[:-1]) == tuple(indices.shape[:-1])
        per_route = x.ndim >= 2 and indices.ndim >= 1 and tuple(x.shape[:-1]) == tuple(indices.shape)
        if self.use_gather_vqmm and token_layout:
            top_k = int(indices.shape[-1])
            flat_x, flat_idx = x.reshape(-1, self.input_dims), indices.reshape(-1, top_k)
            few = should_use_e8p_m1(code_bits=self.code_bits, tokens=int(flat_x.shape[0]), sorted_indices=sorted_indices,
                                    route_strategy=self.route_strategy)
            if few:
                y = e8p_m1_token_layout(flat_x, self.codes, scales, self.codebook, flat_idx, output_dims=self.output_dims)
            else:
                y = gather_vqmm(flat_x, self.codes, scales, self.codebook, flat_idx, sorted_indices=sorted_indices,
                                route_strategy=self.route_strategy, codebook_duplication=self.gather_codebook_duplication, **common)
            y = y.reshape(tuple(indices.shape) + (self.output_dims,))
        elif self.use_gather_vqmm and per_route:
            flat_x, flat_idx = x.reshape(-1, self.input_dims), indices.reshape(-1)
            tokens = int(flat_idx.numel()) // int(indices.shape[-1]) if indices.ndim >= 2 else int(flat_idx.numel())
            few = indices.ndim >= 2 and should_use_e8p_m1(code_bits=self.code_bits, tokens=tokens, sorted_indices=sorted_indices,
                                                          route_strategy=self.route_strategy)
            if few:
                y = e8p_m1_per_route(flat_x, self.codes, scales, self.codebook, flat_idx, output_dims=self.output_dims)
            else:
                rows = torch.arange(int(flat_idx.numel()), device=flat_x.device, dtype=torch.int32)
                y = gather_vqmm(flat_x, self.codes, scales, self.codebook, flat_idx, lhs_indices=rows, sorted_indices=sorted_indices,
                                route_strategy=self.route_strategy, codebook_duplication=self.gather_codebook_duplication, **common)
            y = y.reshape(tuple(indices.shape) + (self.output_dims,))
        else:
            y = vq_switch_qmv(x, self.codes, scales, self.codebook, indices, **common)
        if self.low_rank is not None:
            y = self.low_rank.add(y, x, indices)
        gather = indices.long().clamp(min=0)
        if self.bias is not None:
            y = y + self.bias[gather].to(y.dtype)
        if self.continuous_output_bias is not None:
            y = y + self.continuous_output_bias[gather].to(y.dtype)
        return y


class HighPrecisionSwitchLinear:
    """Switch-linear layer over 16-bit expert weights ``[experts, out, in]``, with the call layouts of
    ``QuantizedVQSwitchLinear``; ``x`` has the weights' dtype.  Recorded by autograd where an input requires
    a gradient."""

    def __init__(self, *, input_dims: int, output_dims: int, num_experts: int, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 low_rank: LowRank | None = None):
        if input_dims <= 0 or output_dims <= 0 or num_experts <= 0:
            raise ValueError("input_dims, output_dims, and num_experts must be positive")
        if input_dims % 8 != 0:
            raise ValueError("input_dims must be divisible by 8")
        expected = (num_experts, output_dims, input_dims)
        if tuple(weight.shape) != expected:
            raise ValueError(f"weight must have shape {expected}, found {tuple(weight.shape)}")
        if weight.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"weight must be fp16 or bf16, found {weight.dtype}")
        if bias is not None and tuple(bias.shape) != (num_experts, output_dims):
            raise ValueError(f"bias must have shape {(num_experts, output_dims)}, found {tuple(bias.shape)}")
        _check_low_rank(low_rank, num_experts, output_dims, input_dims)
        _lib.require_cuda(weight, bias)
        self.input_dims, self.output_dims, self.num_experts = int(input_dims), int(output_dims), int(num_experts)
        self.weight, self.bias, self.low_rank = weight, bias, low_rank

    def __call__(self, x: torch.Tensor, indices: torch.Tensor, *, sorted_indices: bool = False) -> torch.Tensor:
        del sorted_indices  # routes may come in any order
        indices = _indices(indices, x.device)
        y = switch_matmul(x, self.weight, indices)
        if self.low_rank is not None:
            y = self.low_rank.add(y, x, indices)
        if self.bias is not None:  # (a dead route stays zeros, whatever number it holds)
            dead = (indices < 0) | (indices >= self.num_experts)
            y = y + self.bias[indices.clamp(0, self.num_experts - 1).long()].to(y.dtype).masked_fill(dead[..., None], 0)
        return y


def limited_swiglu(limit: float) -> Callable[[torch.Tensor, torch.Tensor], torch.Tensor]:
    """The activation of ``LimitedSwiGLU`` (``deepseek_v4_flash_adapter.py:963-967``) as an
    ``activation(up, gate)`` hook; the fused kernels recognise it by its ``limit`` attribute."""
    def act(up: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        if limit and limit > 0:
            gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        return torch.nn.functional.silu(gate) * up

    act.limit = float(limit)
    return act


class QuantizedVQSwitchGLU:
    """``down(act(up(x), gate(x)))`` per route: ``x [tokens, hidden]``, ``indices [tokens, k]`` ->
    ``[tokens, k, hidden]`` (``glm4_moe_adapter.py:367-372``).

    With 16-bit E8P codes, no bias, sidecars or low-rank corrections and plain or limited SwiGLU, a call
    runs the fused layer kernels (activation quantisation, gate + up + SwiGLU in one launch, down in
    another); any other configuration (a projection in 16 bits among them) composes the three
    projections as the reference does.  Where some of the three record gradients (16-bit weights, low-rank
    corrections) and a projection over codes would have to pass one on, the call is refused.
    """

    def __init__(self, *, gate_proj: QuantizedVQSwitchLinear, up_proj: QuantizedVQSwitchLinear, down_proj: QuantizedVQSwitchLinear,
                 prefill_engine: str = "auto", activation: Callable[[torch.Tensor, torch.Tensor], torch.Tensor] | None = None):
        if gate_proj.input_dims != up_proj.input_dims:
            raise ValueError("gate_proj and up_proj input dimensions must match")
        if gate_proj.output_dims != up_proj.output_dims:
            raise ValueError("gate_proj and up_proj output dimensions must match")
        if down_proj.input_dims != gate_proj.output_dims:
            raise ValueError("down_proj input dimension must match routed hidden dimension")
        if down_proj.output_dims != gate_proj.input_dims:
            raise ValueError("down_proj output dimension must match model hidden dimension")
        if len({gate_proj.num_experts, up_proj.num_experts, down_proj.num_experts}) != 1:
            raise ValueError("all switch projections must have the same expert count")
        if prefill_engine not in ("auto", "vq_metal", "nax_e8", "nax_e8p"):
            raise ValueError("prefill_engine must be 'auto', 'vq_metal', 'nax_e8', or 'nax_e8p'")
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj
        self.prefill_engine, self.activation = prefill_engine, activation
        self._fused: dict = {}

    def _apply_activation(self, up: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        if self.activation is None:
            return torch.nn.functional.silu(gate) * up
        return self.activation(up, gate)

    def _fused_layer(self, top_k: int):
        """The three projections as one ``RoutedMoELayer`` with ``top_k`` picks per token (its
        router unused), or None when the configuration does not fit the layer kernels."""
        projs = (self.gate_proj, self.up_proj, self.down_proj)
        plain = all(not isinstance(p, HighPrecisionSwitchLinear) and p.code_bits == 16 and p.bias is None and getattr(p, "low_rank", None) is None
                    and not p.has_continuous_sidecar and p.use_gather_vqmm for p in projs)
        if not plain or not (self.activation is None or hasattr(self.activation, "limit")):
            return None
        # a layer holds the tensors that it was made of: it stays while the projections hold the same ones
        held = (self.activation, *(t for p in projs for t in (p.codes, p.scales, p.codebook)))
        parts, layer = self._fused.get(top_k, ((), None))
        if len(parts) != len(held) or any(a is not b for a, b in zip(parts, held)):
            from .moe import Projection, RoutedMoELayer

            g, layer = self.gate_proj, None
            if all(p.codebook is g.codebook or (p.codebook is not None and g.codebook is not None and torch.equal(p.codebook, g.codebook)) for p in projs):
                layer = RoutedMoELayer(torch.zeros((g.num_experts, g.input_dims), dtype=torch.bfloat16, device=g.codes.device),
                                       Projection(g.codes, g.scales), Projection(self.up_proj.codes, self.up_proj.scales),
                                       Projection(self.down_proj.codes, self.down_proj.scales), top_k=top_k, codebook=g.codebook,
                                       swiglu_limit=float(getattr(self.activation, "limit", 0.0)))
                if layer.kernel_path != "tensor":
                    layer = None
            self._fused[top_k] = (held, layer)
        return layer

    def __call__(self, x: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
        fits = x.ndim == 2 and indices.ndim == 2 and x.shape[0] == indices.shape[0] and x.dtype in (torch.bfloat16, torch.float16)
        layer = self._fused_layer(int(indices.shape[1])) if fits else None
        if layer is not None:
            # token layout straight through the layer kernels: route t * k + j reads activation row t
            # (no copy of x per pick); the stages stop before the pick sum and the per-route rows
            # are what this operator returns
            tokens, k = indices.shape
            r = layer._buffers_for(tokens, x.dtype)["routing"]
            r.served_slot.copy_(indices)
            r.served_weight.fill_(1.0)
            layer.decode(x, stages=_lib.STAGE_PREPARE | _lib.STAGE_GATE_UP | _lib.STAGE_DOWN)
            out = layer.route_outputs(tokens, x.dtype).reshape(tokens, k, -1).clone()
            picks = indices.to(torch.int64)
            dead = (picks < 0) | (picks >= self.gate_proj.num_experts)  # rows the kernels never write
            return out.masked_fill_(dead[..., None], 0)
        projs = (self.gate_proj, self.up_proj, self.down_proj)
        records = any(isinstance(p, HighPrecisionSwitchLinear) or getattr(p, "low_rank", None) is not None for p in projs)

        def frozen(rows: torch.Tensor, *through) -> torch.Tensor:
            if records and any(isinstance(p, QuantizedVQSwitchLinear) for p in through):
                _refuse_gradient(rows)
            return rows

        x = frozen(x, self.gate_proj, self.up_proj)
        gate = self.gate_proj(x, indices)
        up = self.up_proj(x, indices)
        return self.down_proj(frozen(self._apply_activation(up, gate), self.down_proj), indices)
