"""Refusals of the products over 16-bit experts and low-rank adapters: they come before any device work."""

import ctypes

import pytest
import torch

from keep_b200 import _lib
from keep_b200.dense_switch import switch_matmul, switch_matmul_grads
from keep_b200.low_rank import LowRank, switch_low_rank, switch_low_rank_grads

NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED, CAPACITY = -1, -2, -3, -4, -5, -7
F16 = torch.float16


def rows(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("x,weight,message", [
    (rows(4, 16, dtype=torch.float32), rows(3, 8, 16, dtype=torch.float32), "fp16 / bf16"),
    (rows(4, 16), rows(3, 8, 16, dtype=torch.bfloat16), "fp16 / bf16"),
    (rows(4, 16), rows(8, 16), "weight must be"),
    (rows(4, 16), rows(0, 8, 16), "weight must be"),
    (rows(4, 12), rows(3, 8, 12), "divisible by 8")])
def test_matmul_refuses(x, weight, message):
    for call in (lambda: switch_matmul(x, weight, torch.zeros(4, 2, dtype=torch.int32)),
                 lambda: switch_matmul_grads(rows(4, 2, 8), x, weight, torch.zeros(4, 2, dtype=torch.int32))):
        with pytest.raises(ValueError, match=message):
            call()


@pytest.mark.parametrize("left,right,message", [
    (rows(3, 8, 4, dtype=torch.float32), rows(3, 4, 16, dtype=torch.float32), "fp16 / bf16"),
    (rows(3, 8, 4), rows(3, 5, 16), "left must be"),
    (rows(3, 8, 4), rows(2, 4, 16), "left must be"),
    (rows(3, 8, 0), rows(3, 0, 16), "left must be"),
    (rows(3, 8, 129), rows(3, 129, 16), "at most 128"),
    (rows(3, 8, 4), rows(3, 4, 12), "divisible by 8")])
def test_low_rank_refuses(left, right, message):
    x, indices = rows(4, 16), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: switch_low_rank(x, left, right, indices), lambda: switch_low_rank_grads(rows(4, 8), x, left, right, indices), lambda: LowRank(left, right)):
        with pytest.raises(ValueError, match=message):
            call()


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):
        switch_matmul(rows(4, 16), rows(3, 8, 16), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):
        switch_low_rank(rows(4, 16), rows(3, 8, 4), rows(3, 4, 16), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="found torch.bfloat16"):
        switch_low_rank(rows(4, 16, dtype=torch.bfloat16), rows(3, 8, 4), rows(3, 4, 16), torch.zeros(4, dtype=torch.int32))


# ---- the C entry points: arguments of a valid call, each case with one of them changed; none reaches a CUDA call ----

def matmul_args(**change):
    a = _lib.SwitchMatmulArgs(x=256, weight=256, grad=256, dtype=1, indices=256, index_bits=32, x_div=2, routes=8, experts=3, out_dim=24, in_dim=16, grad_ld=24,
                              out=256, dx=256, dweight=256, workspace=256, workspace_bytes=1 << 30)
    for name, value in change.items():
        setattr(a, name, value)
    return a


def low_rank_args(**change):
    a = _lib.SwitchLowRankArgs(x=256, left=256, right=256, grad=256, dtype=1, indices=256, index_bits=32, x_div=2, routes=800, sets=3, out_dim=24, in_dim=16, rank=8,
                               grad_ld=24, scale=1.0, out_dtype=1, base=256, base_ld=24, out=256, out_ld=24, dx=256, dleft=256, dright=256, workspace=256, workspace_bytes=1 << 30)
    for name, value in change.items():
        setattr(a, name, value)
    return a


BOTH = [(dict(dtype=0), DTYPE), (dict(dtype=7), DTYPE), (dict(index_bits=16), DTYPE), (dict(routes=-1), SHAPE), (dict(routes=801), SHAPE), (dict(x_div=0), SHAPE),
        (dict(in_dim=12), SHAPE), (dict(out_dim=0), SHAPE), (dict(routes=1 << 25), CAPACITY), (dict(workspace=None), NULL), (dict(workspace=264), ALIGN),
        (dict(workspace_bytes=64), CAPACITY), (dict(x=None), NULL), (dict(indices=None), NULL), (dict(x=258), ALIGN), (dict(indices=258), ALIGN)]


@pytest.mark.parametrize("change,status", BOTH + [(dict(experts=0), SHAPE), (dict(experts=1 << 15), CAPACITY), (dict(weight=None), NULL), (dict(weight=264), ALIGN)])
def test_the_matmul_entry_points_refuse(change, status):
    lib = _lib.load()
    assert lib.keepvq_switch_matmul(matmul_args(**change), None) == status
    assert lib.keepvq_switch_matmul_grads(matmul_args(**change), None) == status


@pytest.mark.parametrize("change,status", BOTH + [(dict(sets=0), SHAPE), (dict(sets=1 << 15), CAPACITY), (dict(left=None), NULL), (dict(right=264), ALIGN),
                                                  (dict(rank=12), SHAPE), (dict(rank=0), SHAPE), (dict(rank=136), UNSUPPORTED)])
def test_the_low_rank_entry_points_refuse(change, status):
    lib = _lib.load()
    assert lib.keepvq_switch_low_rank(low_rank_args(**change), None) == status
    assert lib.keepvq_switch_low_rank_grads(low_rank_args(**change), None) == status


def test_what_only_one_direction_looks_at():
    lib = _lib.load()
    assert lib.keepvq_switch_matmul(matmul_args(out=None), None) == NULL
    assert lib.keepvq_switch_matmul_grads(matmul_args(grad=None), None) == NULL
    assert lib.keepvq_switch_matmul_grads(matmul_args(grad_ld=16), None) == SHAPE
    assert lib.keepvq_switch_matmul_grads(matmul_args(grad_ld=28), None) == SHAPE
    assert lib.keepvq_switch_low_rank(low_rank_args(out=None), None) == NULL
    assert lib.keepvq_switch_low_rank(low_rank_args(out_dtype=2), None) == DTYPE
    assert lib.keepvq_switch_low_rank(low_rank_args(base_ld=23), None) == SHAPE
    assert lib.keepvq_switch_low_rank(low_rank_args(out_ld=23), None) == SHAPE
    for pitch in ("base_ld", "out_ld"):
        assert lib.keepvq_switch_low_rank(low_rank_args(**{pitch: 1 << 29}), None) == CAPACITY
    assert lib.keepvq_switch_low_rank_grads(low_rank_args(grad_ld=16), None) == SHAPE
    for name, args in (("keepvq_switch_matmul", matmul_args), ("keepvq_switch_low_rank", low_rank_args)):
        assert getattr(lib, name)(args(routes=0), None) == 0  # nothing to do, nothing launched
        assert getattr(lib, name)(ctypes.cast(None, ctypes.POINTER(type(args()))), None) == NULL
        assert getattr(lib, name + "_grads")(ctypes.cast(None, ctypes.POINTER(type(args()))), None) == NULL


def test_scratch_sizes():
    lib = _lib.load()
    assert lib.keepvq_switch_matmul_workspace_bytes(8, 3, 24, 12, 2, 0) == SHAPE
    assert lib.keepvq_switch_matmul_workspace_bytes(8, 1 << 15, 24, 16, 2, 0) == CAPACITY
    assert lib.keepvq_switch_low_rank_workspace_bytes(8, 3, 24, 16, 136, 2, 0) == UNSUPPORTED
    assert lib.keepvq_switch_low_rank_workspace_bytes(8, 3, 24, 16, 8, 2, 0) == 0  # a few rows need none
    assert lib.keepvq_switch_low_rank_workspace_bytes(8, 3, 24, 16, 8, 2, 1) > 0
    # a row's gradient is summed over its picks in fp32
    assert lib.keepvq_switch_matmul_workspace_bytes(4096, 8, 512, 1024, 2, 1) >= 4096 * 1024 * 4
    assert lib.keepvq_switch_matmul_workspace_bytes(0, 1, 8, 8, 1, 0) > 0


def test_the_sixteen_bit_holder_refuses():
    from keep_b200.switch import HighPrecisionSwitchLinear

    ok = dict(input_dims=16, output_dims=8, num_experts=3, weight=rows(3, 8, 16))
    for change, message in ((dict(num_experts=0), "must be positive"), (dict(input_dims=12, weight=rows(3, 8, 12)), "divisible by 8"), (dict(output_dims=9), "weight must have shape"),
                            (dict(weight=rows(3, 8, 16, dtype=torch.float32)), "fp16 or bf16"), (dict(bias=rows(3, 7)), "bias must have shape"),
                            (dict(low_rank=LowRank(rows(3, 8, 4), rows(3, 4, 24))), "low_rank must correct")):
        with pytest.raises(ValueError, match=message):
            HighPrecisionSwitchLinear(**{**ok, **change})
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):
        HighPrecisionSwitchLinear(**ok)


def holder_of_codes(monkeypatch, out=16, low_rank=None):
    """A quantised holder of CPU tensors: enough for what is refused in front of any product."""
    from keep_b200.switch import QuantizedVQSwitchLinear

    with monkeypatch.context() as m:
        m.setattr(_lib, "require_cuda", lambda *tensors: torch.device("cpu"))
        return QuantizedVQSwitchLinear(input_dims=16, output_dims=out, num_experts=3, codes=torch.zeros((3, out, 2), dtype=torch.uint16), scales=rows(3, out, 1),
                                       codebook=torch.zeros(256, dtype=torch.int32), group_size=16, code_bits=16, low_rank=low_rank)


def test_a_corrected_holder_of_codes_refuses_an_input_that_requires_a_gradient(monkeypatch):
    """The product over codes records nothing: the input would be left with the correction's part of its gradient."""
    factors = LowRank(rows(3, 16, 4).requires_grad_(), rows(3, 4, 16).requires_grad_())
    layer, indices = holder_of_codes(monkeypatch, low_rank=factors), torch.zeros(4, 2, dtype=torch.int32)
    for x in (rows(4, 16), rows(4, 2, 16)):
        with pytest.raises(_lib.KeepVQError, match="has no gradient"):
            layer(x.requires_grad_(), indices)
        with pytest.raises(_lib.KeepVQError, match="no CPU path"):  # as far as CPU tensors come: the factors may require one
            layer(x.detach(), indices)
        with torch.no_grad(), pytest.raises(_lib.KeepVQError, match="no CPU path"):
            layer(x, indices)
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):  # without a correction nothing records, and backward() says so
        holder_of_codes(monkeypatch)(rows(4, 16).requires_grad_(), indices)


def test_a_mixed_glu_refuses_where_a_gradient_would_have_to_pass_codes(monkeypatch):
    """Codes beside a 16-bit projection, or beside a correction: x would get a part of its gradient, or the projections in
    front of the codes none at all."""
    from keep_b200.switch import HighPrecisionSwitchLinear, QuantizedVQSwitchGLU

    indices, factors = torch.zeros(4, 2, dtype=torch.int32), LowRank(rows(3, 16, 4), rows(3, 4, 16))
    with monkeypatch.context() as m:
        m.setattr(_lib, "require_cuda", lambda *tensors: torch.device("cpu"))
        dense = HighPrecisionSwitchLinear(input_dims=16, output_dims=16, num_experts=3, weight=rows(3, 16, 16))
    codes, corrected = holder_of_codes(monkeypatch), holder_of_codes(monkeypatch, low_rank=factors)
    glu = lambda gate, up, down: QuantizedVQSwitchGLU(gate_proj=gate, up_proj=up, down_proj=down)  # noqa: E731
    for trio in ((dense, codes, dense), (codes, dense, codes), (codes, codes, dense), (codes, corrected, codes), (codes, codes, corrected)):
        with pytest.raises(_lib.KeepVQError, match="has no gradient"):
            glu(*trio)(rows(4, 16).requires_grad_(), indices)
        with pytest.raises(_lib.KeepVQError, match="no CPU path"):
            glu(*trio)(rows(4, 16), indices)
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):  # everything recorded
        glu(dense, dense, dense)(rows(4, 16).requires_grad_(), indices)


def test_a_hidden_row_that_requires_a_gradient_does_not_enter_codes(monkeypatch):
    from keep_b200.switch import HighPrecisionSwitchLinear, QuantizedVQSwitchGLU

    class Recorded(HighPrecisionSwitchLinear):
        def __init__(self):
            self.input_dims = self.output_dims = 16
            self.num_experts = 3

        def __call__(self, x, indices):
            return rows(4, 2, 16).requires_grad_()

    layer = QuantizedVQSwitchGLU(gate_proj=Recorded(), up_proj=Recorded(), down_proj=holder_of_codes(monkeypatch))
    with pytest.raises(_lib.KeepVQError, match="has no gradient"):
        layer(rows(4, 16), torch.zeros(4, 2, dtype=torch.int32))
    with torch.no_grad(), pytest.raises(_lib.KeepVQError, match="no CPU path"):
        layer(rows(4, 16), torch.zeros(4, 2, dtype=torch.int32))


def forward_calls():
    """(name, call over a list of arguments, those arguments) of everything that takes values which may carry tangents."""
    indices, low = torch.zeros(4, 2, dtype=torch.int32), (rows(3, 8, 4), rows(3, 4, 16))
    yield "switch_matmul", lambda t: switch_matmul(*t, indices), [rows(4, 16), rows(3, 8, 16)]
    yield "switch_matmul_grads", lambda t: switch_matmul_grads(*t, indices), [rows(4, 2, 8), rows(4, 16), rows(3, 8, 16)]
    yield "switch_low_rank", lambda t: switch_low_rank(*t[:3], indices, base=t[3]), [rows(4, 16), *low, rows(4, 2, 8)]
    yield "switch_low_rank_grads", lambda t: switch_low_rank_grads(*t, indices), [rows(4, 2, 8), rows(4, 16), *low]


def test_tangents_are_refused():
    """A result that came back without one would read as independent of the argument."""
    from torch.autograd import forward_ad

    for name, call, args in forward_calls():
        for i in range(len(args)):
            for leaf in (args[i], args[i].clone().requires_grad_()):
                with forward_ad.dual_level():
                    dual = forward_ad.make_dual(leaf, torch.ones_like(args[i]))
                    for grad_mode in (torch.enable_grad, torch.no_grad):
                        with grad_mode(), pytest.raises(_lib.KeepVQError, match=f"{name} has no forward-mode derivative"):
                            call([*args[:i], dual, *args[i + 1:]])
            with pytest.raises(_lib.KeepVQError, match="no forward-mode derivative"):
                torch.func.jvp(lambda t: call([*args[:i], t, *args[i + 1:]]), (args[i],), (torch.ones_like(args[i]),))
        with forward_ad.dual_level(), pytest.raises(_lib.KeepVQError, match="no CPU path"):  # nothing carries one
            call(args)


def test_a_mixed_glu_refuses_tangents_that_would_have_to_pass_codes(monkeypatch):
    from torch.autograd import forward_ad

    from keep_b200.switch import HighPrecisionSwitchLinear, QuantizedVQSwitchGLU

    with monkeypatch.context() as m:
        m.setattr(_lib, "require_cuda", lambda *tensors: torch.device("cpu"))
        dense = HighPrecisionSwitchLinear(input_dims=16, output_dims=16, num_experts=3, weight=rows(3, 16, 16))
    codes = holder_of_codes(monkeypatch)
    layer = QuantizedVQSwitchGLU(gate_proj=codes, up_proj=codes, down_proj=dense)
    with forward_ad.dual_level(), pytest.raises(_lib.KeepVQError, match="QuantizedVQSwitchLinear has no forward-mode derivative"):
        layer(forward_ad.make_dual(rows(4, 16), rows(4, 16)), torch.zeros(4, 2, dtype=torch.int32))


@pytest.mark.parametrize("ranks", [0, -1, 9, 1 << 20])
def test_ranks_beyond_the_factors_are_refused(ranks):
    lib = _lib.load()
    assert lib.keepvq_switch_low_rank_padded(low_rank_args(), ranks, None) == SHAPE
    assert lib.keepvq_switch_low_rank_grads_padded(low_rank_args(), ranks, None) == SHAPE
    assert lib.keepvq_switch_low_rank_padded(low_rank_args(routes=0), 5, None) == 0


def test_the_wait_entry_points_refuse():
    from keep_b200.dense_switch import switch_matmul_wait_expired

    lib = _lib.load()
    assert lib.keepvq_switch_matmul_wait_expired(None, None) == NULL
    assert lib.keepvq_switch_matmul_wait_expired(258, None) == ALIGN
    assert lib.keepvq_switch_matmul_wait_selftest(None, 0, 1000, None) == NULL
    for grads in (0, 1):
        for limit in (0, -1, 1_000_000_001):
            assert lib.keepvq_switch_matmul_wait_selftest(matmul_args(), grads, limit, None) == SHAPE
        assert lib.keepvq_switch_matmul_wait_selftest(matmul_args(weight=264), grads, 1000, None) == ALIGN
    with pytest.raises(_lib.KeepVQError, match="no CPU path"):
        switch_matmul_wait_expired("cpu")
