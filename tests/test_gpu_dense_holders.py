"""The 16-bit switch holder, low-rank corrections on either holder, adapters beside the shared expert, and the
custom ops over them."""

import numpy as np
import pytest
import torch

import switch_reference as ref
import synthetic

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rand(gen, *shape, scale=1.0, dtype=BF16):
    return (scale * torch.randn(shape, generator=gen, device=gen.device)).to(dtype)


def pair(gen, sets, out, inp, rank=16, scale=0.5):
    from keep_b200.low_rank import LowRank

    return LowRank(rand(gen, sets, out, rank, scale=rank ** -0.5), rand(gen, sets, rank, inp, scale=inp ** -0.5), scale)


def dense_linear(weight, **kw):
    from keep_b200.switch import HighPrecisionSwitchLinear

    experts, out, inp = weight.shape
    return HighPrecisionSwitchLinear(input_dims=inp, output_dims=out, num_experts=experts, weight=weight, **kw)


def near(got, want, rounds=3):
    """`rounds` roundings to the result's type one after the other, each of something as large as the result's largest value at most."""
    assert got.shape == want.shape
    assert (got.double() - want).abs().max() <= rounds * torch.finfo(got.dtype).eps / 2 * want.abs().max()


@pytest.mark.parametrize("tokens", [3, 90])
def test_high_precision_switch_linear(cuda, tokens):
    gen = torch.Generator(device=cuda).manual_seed(tokens)
    weight, bias, x, rows = rand(gen, 6, 72, 256, scale=1 / 16), rand(gen, 6, 72), rand(gen, tokens, 256), rand(gen, tokens, 2, 256)
    indices, low = ref.picks(gen, tokens, 2, 6), pair(gen, 6, 72, 256)
    layer = dense_linear(weight)
    ref.close(layer(x, indices), ref.matmul(x, weight, indices))
    ref.close(layer(rows, indices, sorted_indices=True), ref.matmul(rows, weight, indices))
    got = dense_linear(weight, bias=bias, low_rank=low)(x, indices.long())
    want = ref.matmul(x, weight, indices)[0] + ref.low_rank(x, low.left, low.right, indices, None, low.scale)[0] + bias[indices.long()].double()
    near(got, want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.uint32])
def test_dead_routes_get_no_bias(cuda, dtype):
    """Numbers below and beyond the experts: zeros, not another expert's bias, and no read outside of it."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    weight, bias, x = rand(gen, 6, 72, 256, scale=1 / 16), rand(gen, 6, 72).requires_grad_(True), rand(gen, 4, 256)
    indices = torch.tensor([[0, -1], [5, 6], [-7, 2], [1 << 30, -1]], device=cuda)
    out = dense_linear(weight, bias=bias)(x, indices.to(torch.int32).view(dtype) if dtype == torch.uint32 else indices.to(dtype))
    dead = (indices < 0) | (indices > 5)
    assert out[dead].eq(0).all()
    near(out[~dead], (ref.matmul(x, weight, indices)[0] + bias.double()[indices.clamp(0, 5)])[~dead], rounds=2)
    out.sum().backward()  # sums of ones: exact
    assert torch.equal(bias.grad[:, 0].float(), torch.tensor([1.0, 0, 1, 0, 0, 1], device=cuda))


def test_glu_of_mixed_projections(cuda):
    """Gate and up in E8P codes, down in 16 bits, against the same products one by one."""
    from keep_b200 import vq
    from keep_b200.switch import QuantizedVQSwitchGLU, QuantizedVQSwitchLinear

    gen, rng = torch.Generator(device=cuda).manual_seed(1), np.random.default_rng(1)
    hold = lambda w: QuantizedVQSwitchLinear(input_dims=256, output_dims=256, num_experts=5, codes=torch.from_numpy(w[0]).to(cuda),  # noqa: E731
                                             scales=torch.from_numpy(w[1]).to(cuda), group_size=256, code_bits=16)
    gate, up = hold(synthetic.projection(rng, 5, 256, 256)), hold(synthetic.projection(rng, 5, 256, 256))
    down = rand(gen, 5, 256, 256, scale=1 / 16)
    x, indices = rand(gen, 40, 256, scale=0.3), ref.picks(gen, 40, 2, 5)
    got = QuantizedVQSwitchGLU(gate_proj=gate, up_proj=up, down_proj=dense_linear(down))(x, indices)
    h = (torch.nn.functional.silu(gate(x, indices)) * up(x, indices))
    ref.close(got, ref.matmul(h, down, indices))
    dense = [vq.decode_weight_matrix(p.codes, p.scales, code_bits=16).to(BF16) for p in (gate, up)]  # the same layer, all in 16 bits
    whole = QuantizedVQSwitchGLU(gate_proj=dense_linear(dense[0]), up_proj=dense_linear(dense[1]), down_proj=dense_linear(down))(x, indices)
    gap = (whole.double() - got.double()).abs().max() / got.double().abs().max()
    assert gap <= 1e-2  # weights rounded to 16 bits


def test_quantized_switch_linear_with_a_correction_per_expert(cuda):
    from keep_b200.switch import QuantizedVQSwitchLinear

    gen, rng = torch.Generator(device=cuda).manual_seed(2), np.random.default_rng(2)
    codes, scales = (torch.from_numpy(t).to(cuda) for t in synthetic.projection(rng, 6, 48, 256))
    low = pair(gen, 6, 48, 256)
    kw = dict(input_dims=256, output_dims=48, num_experts=6, codes=codes, scales=scales, group_size=256, code_bits=16)
    plain, corrected = QuantizedVQSwitchLinear(**kw), QuantizedVQSwitchLinear(**kw, low_rank=low)
    for x, indices in ((rand(gen, 7, 256), ref.picks(gen, 7, 3, 6)), (rand(gen, 9, 2, 256), ref.picks(gen, 9, 2, 6, dead=0.3))):
        y = plain(x, indices)
        ref.close(corrected(x, indices), ref.low_rank(x, low.left, low.right, indices, y, low.scale))
    with pytest.raises(ValueError, match="low_rank must correct"):
        QuantizedVQSwitchLinear(**kw, low_rank=pair(gen, 6, 56, 256))


def test_shared_expert_with_adapters_of_the_requests(cuda):
    from keep_b200.moe import SharedExpert

    gen = torch.Generator(device=cuda).manual_seed(3)
    w1, w3, w2 = rand(gen, 264, 512, scale=1 / 22), rand(gen, 264, 512, scale=1 / 22), rand(gen, 512, 264, scale=1 / 16)
    shared, x = SharedExpert(w1, w3, w2), rand(gen, 33, 512)
    adapters = {"w1": pair(gen, 4, 264, 512, 8), "w3": pair(gen, 4, 264, 512, 16), "w2": pair(gen, 4, 512, 264, 5)}
    indices = torch.randint(-1, 4, (33,), generator=gen, device=cuda)
    got = shared(x, adapters=adapters, adapter_indices=indices)
    assert got.dtype == torch.float32
    inner = {}
    for name, w in (("w1", w1), ("w3", w3)):
        base = x.double() @ w.double().T
        inner[name] = base + ref.low_rank(x, adapters[name].left, adapters[name].right, indices, None, 0.5)[0]
    h = (torch.nn.functional.silu(inner["w1"]) * inner["w3"]).to(BF16)
    want = h.double() @ w2.double().T + ref.low_rank(h, adapters["w2"].left, adapters["w2"].right, indices, None, 0.5)[0]
    assert (got.double() - want).abs().max() <= 2.0 ** -8 * want.abs().max()  # h rounds to a neighbour where its fp32 sums differ
    none = indices < 0
    assert torch.equal(got[none], shared(x)[none])
    with pytest.raises(ValueError, match="adapter_indices"):
        shared(x, adapters=adapters)


def test_custom_ops(cuda):
    from keep_b200 import torch_ops  # noqa: F401
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    gen, ops = torch.Generator(device=cuda).manual_seed(4), torch.ops.keepvq
    x, weight, low, indices = rand(gen, 12, 64), rand(gen, 4, 48, 64), pair(gen, 4, 48, 64, 8), ref.picks(gen, 12, 2, 4)
    base, grad = rand(gen, 12, 2, 48), rand(gen, 12, 2, 48)
    cases = {"switch_matmul": (x, weight, indices), "switch_matmul_grads": (grad, x, weight, indices, True, True),
             "switch_low_rank": (x, low.left, low.right, indices, base, 0.5), "switch_low_rank_grads": (grad, x, low.left, low.right, indices, 0.5, True, True)}
    for name, args in cases.items():
        torch.library.opcheck(getattr(ops, name).default, args, test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_static"))
    leaves = [t.clone().requires_grad_() for t in (x, weight, low.left, low.right)]
    for name, args in (("switch_matmul", (*leaves[:2], indices)), ("switch_low_rank", (leaves[0], *leaves[2:], indices, base, 0.5))):
        torch.library.opcheck(getattr(ops, name).default, args, test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    assert torch.equal(ops.switch_matmul(x, weight, indices), switch_matmul(x, weight, indices))

    def layer(x, weight, left, right):
        return ops.switch_low_rank(x, left, right, indices, ops.switch_matmul(x, weight, indices), 0.5)

    compiled = torch.compile(layer, fullgraph=True, backend="aot_eager")
    y = compiled(*leaves)
    assert torch.equal(y, switch_low_rank(x, low.left, low.right, indices, base=switch_matmul(x, weight, indices), scale=0.5))
    y.backward(grad)
    dense, thin = switch_matmul_grads(grad, x, weight, indices), switch_low_rank_grads(grad, x, low.left, low.right, indices, scale=0.5)
    assert torch.equal(leaves[1].grad, dense[1]) and torch.equal(leaves[2].grad, thin[1]) and torch.equal(leaves[3].grad, thin[2])
    near(leaves[0].grad, dense[0].double() + thin[0].double(), rounds=1)


def test_custom_ops_refuse_recorded_captures(cuda):
    from keep_b200 import _lib, torch_ops  # noqa: F401

    gen, ops = torch.Generator(device=cuda).manual_seed(5), torch.ops.keepvq
    x, weight, low, indices = rand(gen, 12, 64), rand(gen, 4, 48, 64), pair(gen, 4, 48, 64, 8), ref.picks(gen, 12, 2, 4)
    leaf = x.clone().requires_grad_()
    calls = {"switch_matmul": lambda t: ops.switch_matmul(t, weight, indices), "switch_low_rank": lambda t: ops.switch_low_rank(t, low.left, low.right, indices, None, 0.5)}
    for name, call in calls.items():
        want, graph = call(x), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(_lib.KeepVQError, match=f"{name}: a recorded gradient cannot be captured"):
                call(leaf)
            got = call(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_gradients_of_a_correction_on_a_holder_of_codes(cuda):
    """The factors' gradients are those of the correction alone (the base is frozen); an input that requires one is refused."""
    from keep_b200 import _lib
    from keep_b200.low_rank import LowRank, switch_low_rank_grads
    from keep_b200.switch import QuantizedVQSwitchLinear

    gen, rng = torch.Generator(device=cuda).manual_seed(6), np.random.default_rng(6)
    codes, scales = (torch.from_numpy(t).to(cuda) for t in synthetic.projection(rng, 6, 48, 256))
    low = pair(gen, 6, 48, 256)
    leaves = [t.clone().requires_grad_() for t in (low.left, low.right)]
    layer = QuantizedVQSwitchLinear(input_dims=256, output_dims=48, num_experts=6, codes=codes, scales=scales, group_size=256, code_bits=16, low_rank=LowRank(*leaves, low.scale))
    x, indices, grad = rand(gen, 7, 256), ref.picks(gen, 7, 3, 6), rand(gen, 7, 3, 48)
    layer(x, indices).backward(grad)
    want = switch_low_rank_grads(grad, x, low.left, low.right, indices, scale=low.scale, x_grad=False)
    assert torch.equal(leaves[0].grad, want[1]) and torch.equal(leaves[1].grad, want[2])
    with pytest.raises(_lib.KeepVQError, match="has no gradient"):
        layer(x.requires_grad_(), indices)
    with torch.no_grad():
        assert torch.equal(layer(x, indices), layer(x.detach(), indices))


def codes_linear(cuda, rng, experts, out, inp, **kw):
    from keep_b200.switch import QuantizedVQSwitchLinear

    codes, scales = (torch.from_numpy(t).to(cuda) for t in synthetic.projection(rng, experts, out, inp))
    return QuantizedVQSwitchLinear(input_dims=inp, output_dims=out, num_experts=experts, codes=codes, scales=scales, group_size=256, code_bits=16, **kw)


def test_a_glu_follows_what_its_projections_hold(cuda):
    """The fused layer is kept from call to call; what is attached, exchanged or taken off between calls counts for the next one."""
    from keep_b200.switch import QuantizedVQSwitchGLU, limited_swiglu

    gen, rng = torch.Generator(device=cuda).manual_seed(7), np.random.default_rng(7)
    gate, up, down, other = (codes_linear(cuda, rng, 5, 256, 256) for _ in range(4))
    x, indices = rand(gen, 40, 256, scale=0.3), ref.picks(gen, 40, 2, 5)
    glu = QuantizedVQSwitchGLU(gate_proj=gate, up_proj=up, down_proj=down)
    fresh = lambda: QuantizedVQSwitchGLU(gate_proj=glu.gate_proj, up_proj=glu.up_proj, down_proj=glu.down_proj, activation=glu.activation)(x, indices)  # noqa: E731
    first = glu(x, indices)
    assert glu._fused_layer(2) is not None and glu._fused_layer(2) is glu._fused_layer(2)
    seen = [first]
    for change in (lambda: setattr(down, "low_rank", pair(gen, 5, 256, 256)), lambda: setattr(down, "low_rank", None), lambda: setattr(up, "bias", rand(gen, 5, 256)),
                   lambda: setattr(up, "bias", None), lambda: setattr(glu, "up_proj", other), lambda: setattr(other, "scales", other.scales * 2),
                   lambda: setattr(glu, "activation", limited_swiglu(0.01)), lambda: setattr(glu, "down_proj", dense_linear(rand(gen, 5, 256, 256, scale=1 / 16)))):
        change()
        got = glu(x, indices)
        assert torch.equal(got, fresh())
        assert not torch.equal(got, seen[-1])
        seen.append(got)
    assert torch.equal(seen[2], first) and torch.equal(seen[4], first)


def test_a_holder_of_its_own_class_runs_the_fused_layer(cuda):
    """A projection is known by what it holds: one that is no QuantizedVQSwitchLinear and knows nothing of corrections runs as before."""
    from types import SimpleNamespace

    from keep_b200.switch import QuantizedVQSwitchGLU

    gen, rng = torch.Generator(device=cuda).manual_seed(8), np.random.default_rng(8)
    trio = [codes_linear(cuda, rng, 5, 256, 256) for _ in range(3)]
    names = ("input_dims", "output_dims", "num_experts", "code_bits", "bias", "has_continuous_sidecar", "use_gather_vqmm", "codes", "scales", "codebook")
    own = [SimpleNamespace(**{n: getattr(p, n) for n in names}) for p in trio]
    x, indices = rand(gen, 40, 256, scale=0.3), ref.picks(gen, 40, 2, 5)
    make = lambda t: QuantizedVQSwitchGLU(gate_proj=t[0], up_proj=t[1], down_proj=t[2])  # noqa: E731
    assert torch.equal(make(own)(x, indices), make(trio)(x, indices))


def test_custom_ops_refuse_forward_mode_differentiation(cuda):
    from keep_b200 import _lib, torch_ops  # noqa: F401

    gen, ops = torch.Generator(device=cuda).manual_seed(9), torch.ops.keepvq
    x, weight, low, indices, grad = rand(gen, 12, 64), rand(gen, 4, 48, 64), pair(gen, 4, 48, 64, 8), ref.picks(gen, 12, 2, 4), rand(gen, 12, 2, 48)
    calls = {"switch_matmul": lambda t: ops.switch_matmul(t, weight, indices), "switch_matmul_grads": lambda t: ops.switch_matmul_grads(grad, t, weight, indices, True, True),
             "switch_low_rank": lambda t: ops.switch_low_rank(t, low.left, low.right, indices, None, 0.5),
             "switch_low_rank_grads": lambda t: ops.switch_low_rank_grads(grad, t, low.left, low.right, indices, 0.5, True, True)}
    for name, call in calls.items():
        with pytest.raises(_lib.KeepVQError, match=f"keepvq::{name} has no forward-mode derivative"):
            torch.func.jvp(call, (x,), (x,))
        with torch.autograd.forward_ad.dual_level(), pytest.raises(_lib.KeepVQError, match="no forward-mode derivative"):
            call(torch.autograd.forward_ad.make_dual(x, x))
        call(x)


def test_gradients_of_adapters_beside_the_shared_expert(cuda):
    """Those of w2 are its correction's; what would have to pass the library product fails instead of being left out."""
    from keep_b200.low_rank import LowRank, switch_low_rank_grads
    from keep_b200.moe import SharedExpert

    gen = torch.Generator(device=cuda).manual_seed(10)
    shared, x = SharedExpert(rand(gen, 264, 512, scale=1 / 22), rand(gen, 264, 512, scale=1 / 22), rand(gen, 512, 264, scale=1 / 16)), rand(gen, 33, 512)
    indices = torch.randint(-1, 4, (33,), generator=gen, device=cuda)
    low = {"w1": pair(gen, 4, 264, 512, 8), "w2": pair(gen, 4, 512, 264, 8)}
    leaves = {n: LowRank(p.left.clone().requires_grad_(), p.right.clone().requires_grad_(), p.scale) for n, p in low.items()}
    grad = rand(gen, 33, 512)
    shared(x, adapters={"w2": leaves["w2"]}, adapter_indices=indices).backward(grad.float())
    gate, up = torch.mm(x, shared.gate_up, out_dtype=torch.float32).split(264, dim=1)
    h = (torch.nn.functional.silu(gate) * up).to(BF16)
    want = switch_low_rank_grads(grad, h, low["w2"].left, low["w2"].right, indices, scale=0.5, x_grad=False)
    assert torch.equal(leaves["w2"].left.grad, want[1]) and torch.equal(leaves["w2"].right.grad, want[2])
    with pytest.raises(RuntimeError, match="not implemented"):
        shared(x, adapters=leaves, adapter_indices=indices).backward(grad.float())
