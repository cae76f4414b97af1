"""Low-rank products per route (switch_low_rank and its gradients) against a plain 64-bit form."""

import pytest
import torch

import switch_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def make(cuda, tokens, k, sets, inp, out, rank, dtype=BF16, per_route=False, dead=0.0, seed=0, base=None, size=1.0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=cuda)  # noqa: E731
    x = (size * rand(*((tokens, k, inp) if per_route else (tokens, inp)))).to(dtype)
    left, right = (rand(sets, out, rank) * rank ** -0.5).to(dtype), (rand(sets, rank, inp) * inp ** -0.5).to(dtype)
    indices = torch.randint(0, sets, (tokens, k), generator=gen, device=cuda, dtype=torch.int32)
    gone = torch.rand((tokens, k), generator=gen, device=cuda)
    indices = torch.where(gone < dead / 2, -1, torch.where(gone < dead, sets + 3, indices))
    rows = rand(tokens, k, out)
    return x, left, right, indices, None if base is None else rows.to(base), (0.1 * rand(tokens, k, out)).to(dtype)


# tokens, picks, sets, in, out, rank: single tokens, ranks and widths that fill no tile, one set for all rows, sets without
# rows, hundreds of rows a set
SIZES = [(1, 1, 1, 8, 8, 8), (1, 1, 64, 1024, 512, 16), (3, 2, 5, 72, 200, 8), (17, 4, 6, 136, 72, 24), (130, 1, 1, 128, 264, 64), (5, 6, 300, 64, 40, 128),
         (257, 6, 7, 520, 136, 40), (700, 2, 3, 64, 1000, 16), (61, 1, 30, 2048, 1024, 32), (1021, 1, 4, 392, 328, 64), (33, 1, 9, 264, 136, 5), (20, 2, 3, 64, 48, 1)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("per_route", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(cuda, size, per_route, dtype):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, *size, dtype=dtype, per_route=per_route, dead=0.2 if size[0] > 2 else 0.0, seed=sum(size), base=dtype)
    ref.close(switch_low_rank(x, left, right, indices, base=base, scale=0.5), ref.low_rank(x, left, right, indices, base, 0.5))
    got = switch_low_rank_grads(grad, x, left, right, indices, scale=0.5)
    for a, b in zip(got, ref.low_rank_grads(grad, x, left, right, indices, 0.5)):
        ref.close(a, b)


@pytest.mark.parametrize("base", [None, torch.float32])
@pytest.mark.parametrize("size", [(1, 1, 3, 256, 512, 16), (50, 2, 7, 136, 200, 8), (300, 1, 2, 264, 136, 64)])
def test_without_a_base_and_with_one_in_fp32(cuda, size, base):
    from keep_b200.low_rank import switch_low_rank

    for dtype in (BF16, FP16):
        x, left, right, indices, rows, _ = make(cuda, *size, dtype=dtype, dead=0.2, base=base)
        got = switch_low_rank(x, left, right, indices, base=rows, scale=-2.0)
        assert got.dtype == (dtype if base is None else base)
        ref.close(got, ref.low_rank(x, left, right, indices, rows, -2.0))


@pytest.mark.parametrize("out", [1, 7, 100, 513])
def test_output_widths_that_are_no_multiple_of_eight(cuda, out):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 37, 3, 5, 264, out, 16, dead=0.2, seed=out, base=BF16)
    ref.close(switch_low_rank(x, left, right, indices, base=base), ref.low_rank(x, left, right, indices, base, 1.0))
    for a, b in zip(switch_low_rank_grads(grad, x, left, right, indices), ref.low_rank_grads(grad, x, left, right, indices, 1.0)):
        ref.close(a, b)


def test_rows_without_an_adapter_keep_their_base_bit_for_bit(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 40, 1, 4, 128, 72, 16, base=BF16)
    indices[::3] = -1
    base[0, 0, :4] = torch.tensor([float("nan"), float("inf"), -0.0, 1e-40], device=cuda)
    got = switch_low_rank(x, left, right, indices, base=base)
    assert torch.equal(got[::3].view(torch.int16), base[::3].view(torch.int16))
    indices[:] = -1
    assert torch.equal(switch_low_rank(x, left, right, indices, base=base).view(torch.int16), base.view(torch.int16))
    assert not switch_low_rank(x, left, right, indices).any()
    assert not any(g.any() for g in switch_low_rank_grads(grad, x, left, right, indices))


def test_inner_vectors_beyond_the_range_of_fp16(cuda):
    """Rows of 30,000 and rows of 1e-6 (fp16): their inner vectors neither overflow nor vanish."""
    from keep_b200.low_rank import switch_low_rank

    x, left, right, indices, _, _ = make(cuda, 24, 1, 2, 256, 72, 16, dtype=FP16)
    right = right * 16
    x[::2], left = 6000 * x[::2].sign(), left * 2.0 ** -14
    want = ref.low_rank(x, left, right, indices, None, 1.0)
    inner = (x.double() @ right[0].double().T).abs().max()
    assert inner > 65504 and torch.isfinite(want[0]).all() and want[0].abs().max() < 60000
    ref.close(switch_low_rank(x, left, right, indices), want)
    small = (x.double() * 0 + 2.0 ** -20).to(FP16)
    left = left * 2.0 ** 14
    ref.close(switch_low_rank(small, left, right, indices, scale=2.0 ** 14), ref.low_rank(small, left, right, indices, None, 2.0 ** 14))


def test_gradients_of_rows_of_very_different_size(cuda):
    """Rows of one set whose gradients lie 2^-18 apart (fp16), the large ones zero where the small ones are not: what the small
    rows give a factor's gradient is not lost beside them."""
    from keep_b200.low_rank import switch_low_rank_grads

    for size in ((24, 1, 1, 64, 48, 16), (200, 1, 2, 128, 72, 8)):
        x, left, right, indices, _, grad = make(cuda, *size, dtype=FP16, seed=6)
        odd = torch.arange(size[0], device=cuda) % 2 == 1
        grad[odd] *= 2.0 ** -9
        grad[~odd] *= 2.0 ** 9
        x[odd, :32], x[~odd, 32:] = 0, 0
        for a, b in zip(switch_low_rank_grads(grad, x, left, right, indices), ref.low_rank_grads(grad, x, left, right, indices, 1.0)):
            ref.close(a, b)


def test_values_that_are_not_finite_stay_where_they_belong(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 40, 1, 3, 136, 200, 16, base=BF16, seed=3)
    indices[:] = torch.arange(40, device=cuda)[:, None] % 2
    want, grads = ref.low_rank(x, left, right, indices, base, 1.0), ref.low_rank_grads(grad, x, left, right, indices, 1.0)
    for bad in (float("nan"), float("inf")):
        l2, r2 = left.clone(), right.clone()
        l2[2], r2[2] = bad, bad
        ref.close(switch_low_rank(x, l2, r2, indices, base=base), want)
        ref.close(switch_low_rank_grads(grad, x, l2, r2, indices)[0], grads[0])
        rows, g = x.clone(), grad.clone()
        rows[7], g[9] = bad, bad  # both of set 1
        others = (torch.arange(40, device=cuda) != 7)
        got = switch_low_rank(rows, left, right, indices, base=base)
        ref.close(got[others], [t[others] for t in want])
        assert not torch.isfinite(got[7]).any()
        others = (torch.arange(40, device=cuda) != 9)
        dx, dleft, dright = switch_low_rank_grads(g, rows, left, right, indices)
        ref.close(dx[others], [t[others] for t in grads[0]])
        ref.close(dleft[0], [t[0] for t in grads[1]])
        ref.close(dright[0], [t[0] for t in grads[2]])


def test_layouts_strides_and_a_base_inside_a_wider_product(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 12, 1, 4, 64, 48, 8, base=BF16)
    idx, rows, g = indices[:, 0], base[:, 0], grad[:, 0]
    want = switch_low_rank(x, left, right, idx, base=rows)
    assert tuple(want.shape) == (12, 48) and torch.equal(switch_low_rank(x, left, right, indices, base=base)[:, 0], want)
    odd = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731
    across = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    grads = switch_low_rank_grads(g, x, left, right, idx)
    for change in (odd, across):
        assert torch.equal(switch_low_rank(change(x), change(left), change(right), idx, base=change(rows)), want)
        assert all(torch.equal(a, b) for a, b in zip(switch_low_rank_grads(change(g), change(x), change(left), change(right), idx), grads))
    for offset in (0, 3, 8):
        for dtype in (BF16, torch.float32):
            wide = torch.zeros((12, 61), dtype=dtype, device=cuda)
            wide[:, offset:offset + 48] = rows
            got = switch_low_rank(x, left, right, idx, base=wide[:, offset:offset + 48])
            if dtype == BF16:
                assert torch.equal(got, want)
            else:
                ref.close(got, ref.low_rank(x, left, right, idx, rows.float(), 1.0))


def test_no_rows(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 4, 2, 3, 64, 48, 8, base=BF16)
    assert tuple(switch_low_rank(x[:0], left, right, indices[:0], base=base[:0]).shape) == (0, 2, 48)
    dx, dleft, dright = switch_low_rank_grads(grad[:, :0], x, left, right, indices[:, :0])
    assert tuple(dx.shape) == (4, 64) and not dx.any() and not dleft.any() and not dright.any()


def test_a_call_repeats_bit_for_bit(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    for size in ((900, 1, 3, 520, 264, 32), (150, 6, 40, 264, 520, 8)):
        x, left, right, indices, base, grad = make(cuda, *size, base=BF16, dead=0.1)
        y, grads = switch_low_rank(x, left, right, indices, base=base), switch_low_rank_grads(grad, x, left, right, indices)
        for _ in range(3):
            assert torch.equal(switch_low_rank(x, left, right, indices, base=base), y)
            assert all(torch.equal(a, b) for a, b in zip(switch_low_rank_grads(grad, x, left, right, indices), grads))
        only_x = switch_low_rank_grads(grad, x, left, right, indices, weight_grad=False)
        assert torch.equal(only_x[0], grads[0]) and only_x[1] is None and only_x[2] is None
        only_w = switch_low_rank_grads(grad, x, left, right, indices, x_grad=False)
        assert only_w[0] is None and torch.equal(only_w[1], grads[1]) and torch.equal(only_w[2], grads[2])


def test_gradients_against_differences(cuda):
    """Small integers keep every step exact; the product is linear in each of its three factors."""
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    gen = torch.Generator(device=cuda).manual_seed(4)
    def sparse(*shape):  # few ones: inner vectors and sums stay below 256
        return (torch.randint(-1, 2, shape, generator=gen, device=cuda) * (torch.rand(shape, generator=gen, device=cuda) < 0.4)).to(BF16)
    x, left, right, grad = sparse(20, 24), sparse(3, 16, 8), sparse(3, 8, 24), sparse(20, 2, 16)
    indices = torch.randint(-1, 3, (20, 2), generator=gen, device=cuda, dtype=torch.int32)
    dx, dleft, dright = switch_low_rank_grads(grad, x, left, right, indices, scale=0.5)
    y = lambda x, l, r: switch_low_rank(x, l, r, indices, scale=0.5).double()  # noqa: E731
    for _ in range(4):
        d, dl, dr = sparse(20, 24), sparse(3, 16, 8), sparse(3, 8, 24)
        along = lambda a, b: (grad.double() * (a - b) / 2).sum()  # noqa: E731
        assert along(y(x + d, left, right), y(x - d, left, right)) == (dx.double() * d.double()).sum()
        assert along(y(x, left + dl, right), y(x, left - dl, right)) == (dleft.double() * dl.double()).sum()
        assert along(y(x, left, right + dr), y(x, left, right - dr)) == (dright.double() * dr.double()).sum()


def test_autograd_records_the_same_gradients(cuda):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, 30, 3, 5, 128, 72, 12, base=BF16)
    want = switch_low_rank_grads(grad, x, left, right, indices, scale=0.25)
    leaves = [t.clone().requires_grad_() for t in (x, left, right, base)]
    switch_low_rank(leaves[0], leaves[1], leaves[2], indices, base=leaves[3], scale=0.25).backward(grad)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, (*want, grad)))
    only = base.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(switch_low_rank(x, left, right, indices, base=only), only, grad)[0], grad)


def test_captured_calls_follow_their_inputs(cuda):
    from keep_b200 import _lib
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    args = [t for t in make(cuda, 50, 2, 6, 128, 136, 16, dead=0.1, base=BF16)]
    x, left, right, indices, base, grad = args
    leaf = left.clone().requires_grad_()
    alive = switch_low_rank(x, leaf, right, indices, base=base)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            outs.append((switch_low_rank(x, left, right, indices, base=base), *switch_low_rank_grads(grad, x, left, right, indices)))
        graphs.append(graph)
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(_lib.KeepVQError, match="cannot be captured"):
            switch_low_rank(x, leaf, right, indices)
    torch.autograd.grad(alive, leaf, grad)
    for seed in (1, 2):
        for old, fresh in zip(args, make(cuda, 50, 2, 6, 128, 136, 16, dead=0.1, base=BF16, seed=seed)):
            old.copy_(fresh)
        want = (switch_low_rank(x, left, right, indices, base=base), *switch_low_rank_grads(grad, x, left, right, indices))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_an_adapter_on_an_expert_projection_as_a_routed_layer_uses_them(cuda):
    """Router, 16-bit gate projection, a low-rank correction per expert on top, and the gradients of both."""
    from keep_b200.dense_switch import switch_matmul
    from keep_b200.low_rank import switch_low_rank
    from keep_b200.router import routed_topk

    gen = torch.Generator(device=cuda).manual_seed(9)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=cuda).to(BF16)  # noqa: E731
    x, weight, left, right, gate = rand(33, 256), rand(8, 136, 256) / 16, rand(8, 136, 16) / 4, rand(8, 16, 256) / 16, rand(8, 256) / 50
    picks = routed_topk(x, gate, top_k=3).served_expert
    leaves = [t.clone().requires_grad_() for t in (x, weight, left, right)]
    y = switch_low_rank(leaves[0], leaves[2], leaves[3], picks, base=switch_matmul(leaves[0], leaves[1], picks))
    grad = rand(33, 3, 136) / 10
    y.backward(grad)
    want, bound = ref.matmul(x, weight, picks)
    more, more_bound = ref.low_rank(x, left, right, picks, None, 1.0)
    ref.close(y, (want + more, bound + more_bound + ref.rounding(want + more, BF16) + 2.0 ** -8 * bound))
    dense, low = ref.matmul_grads(grad, x, weight, picks), ref.low_rank_grads(grad, x, left, right, picks, 1.0)
    ref.close(leaves[1].grad, dense[1])
    ref.close(leaves[2].grad, low[1])
    ref.close(leaves[3].grad, low[2])
    both = dense[0][0] + low[0][0]
    ref.close(leaves[0].grad, (both, dense[0][1] + low[0][1] + ref.rounding(both, BF16) + 2.0 ** -8 * (dense[0][1] + low[0][1])))


def test_rows_beyond_32_bit_offsets(cuda):
    """2.2e9 values in x, base, grad and the results; a few rows at both ends that are not zero."""
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    tokens, width, rank = 270_000, 8192, 16
    gen = torch.Generator(device=cuda).manual_seed(3)
    ends = torch.cat([torch.arange(9, device=cuda), torch.arange(tokens - 9, tokens, device=cuda)])
    def rows():
        t = torch.zeros((tokens, width), dtype=BF16, device=cuda)
        t[ends] = torch.randn((18, width), generator=gen, device=cuda).to(BF16)
        return t
    left, right = (torch.randn((3, *shape), generator=gen, device=cuda).div(width ** 0.5).to(BF16) for shape in ((width, rank), (rank, width)))
    x, base = rows(), rows()
    indices = torch.arange(tokens, device=cuda, dtype=torch.int32) % 3
    want = ref.low_rank(x[ends], left, right, indices[ends], base[ends], 0.5)
    got = switch_low_rank(x, left, right, indices, base=base, scale=0.5)
    ref.close(got[ends], want)
    assert not got[9:tokens - 9].any()
    del got, base
    grad = rows()
    want = ref.low_rank_grads(grad[ends], x[ends], left, right, indices[ends], 0.5)
    dx, dleft, dright = switch_low_rank_grads(grad, x, left, right, indices, scale=0.5)
    ref.close(dx[ends], want[0])
    assert not dx[9:tokens - 9].any()
    ref.close(dleft, want[1])
    ref.close(dright, want[2])


def same_infinities(got, want_and_bound):
    """The definition's infinities and undefined values in their places, and everything else as near as ever."""
    want, bound = want_and_bound
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.double()[torch.isinf(want)], want[torch.isinf(want)])
    ref.close(got[finite], (want[finite], bound[finite]))


def with_infinities(t, step):
    """An infinity, of either sign in turn, in some of a matrix's rows, at one of their places each."""
    sets, n, width = t.shape
    t = t.clone()
    rows = torch.arange(0, n, step, device=t.device)
    t[:, rows, rows % width] = torch.where(rows // step % 2 == 0, float("inf"), float("-inf")).to(t.dtype)
    return t


# rows, sets, in, out, rank: a tile per row, and tiles of the plan
INFINITE = [(24, 2, 128, 72, 8), (24, 3, 264, 136, 40), (300, 2, 136, 200, 16), (180, 4, 136, 72, 100)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,sets,inp,out,rank", INFINITE)
def test_an_infinity_of_a_factor_is_one_of_the_result(cuda, rows, sets, inp, out, rank, dtype):
    """A vector that enters the second product in two parts meets it with both: zero, or of the other sign, times infinity is no value."""
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, rows, 1, sets, inp, out, rank, dtype=dtype, base=dtype, seed=rank)
    low = with_infinities(left, 5)
    want = ref.low_rank(x, low, right, indices, base, 0.5)
    assert torch.isinf(want[0]).any() and not torch.isnan(want[0]).any()
    same_infinities(switch_low_rank(x, low, right, indices, base=base, scale=0.5), want)
    high = with_infinities(right.transpose(1, 2), 7).transpose(1, 2)
    same_infinities(switch_low_rank_grads(grad, x, left, high, indices, weight_grad=False)[0], ref.low_rank_grads(grad, x, left, high, indices, 1.0)[0])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,sets,inp,out,rank", [*INFINITE[:3], (180, 4, 136, 72, 104), (200, 2, 72, 136, 24)])
def test_an_infinity_of_a_row_is_one_of_its_results(cuda, rows, sets, inp, out, rank, dtype):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, rows, 1, sets, inp, out, rank, dtype=dtype, base=dtype, seed=rank + 1)
    x[::3, 5], grad[1::4, 0, 9] = float("inf"), float("-inf")
    left[:, ::2], right[:, :, ::2] = left[:, ::2].abs(), right[:, :, ::2].abs()
    right[:, :, 5], left[:, 9] = right[:, :, 5].abs(), left[:, 9].abs()
    want = ref.low_rank(x, left, right, indices, base, 0.5)
    assert torch.isinf(want[0]).any()
    same_infinities(switch_low_rank(x, left, right, indices, base=base, scale=0.5), want)
    same_infinities(switch_low_rank_grads(grad, x, left, right, indices, weight_grad=False)[0], ref.low_rank_grads(grad, x, left, right, indices, 1.0)[0])


@pytest.mark.parametrize("rows", [24, 200])
def test_inner_vectors_beyond_the_range_of_fp16_beside_an_infinity(cuda, rows):
    """One inner value is infinite, the others are finite but beyond fp16: they do not become infinities of the other sign."""
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, _, grad = make(cuda, rows, 1, 2, 256, 72, 16, dtype=FP16)
    right, x, left = right * 16, 6000 * x.sign(), left * 2.0 ** -14
    x[:, 3], right[:, 5, 3] = 1, float("inf")
    inner = x.double() @ right[0].double().T
    assert (inner.abs() > 65504).sum(1).ge(2).any()
    want = ref.low_rank(x, left, right, indices, None, 1.0)
    assert torch.isinf(want[0]).all()
    same_infinities(switch_low_rank(x, left, right, indices), want)
    # the same on the way back: q = B^T grad with one infinite entry
    grad, left = 6000 * grad.sign(), left * 2.0 ** 18
    grad[:, :, 3], left[:, 3, 5], right = 1, float("inf"), right.nan_to_num(posinf=1.0) * 2.0 ** -18
    want = ref.low_rank_grads(grad, x, left, right, indices, 1.0)[0]
    assert torch.isinf(want[0]).any()
    same_infinities(switch_low_rank_grads(grad, x, left, right, indices, weight_grad=False)[0], want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,rank", [(24, 1), (24, 5), (180, 12), (180, 100)])
def test_ranks_that_fill_up_a_multiple_of_eight_stay_out_of_rows_that_are_not_finite(cuda, rows, rank, dtype):
    from keep_b200.low_rank import switch_low_rank, switch_low_rank_grads

    x, left, right, indices, base, grad = make(cuda, rows, 1, 3, 136, 72, rank, dtype=dtype, base=dtype, seed=rank)
    x[::3, 5], grad[1::4, 0, 9] = float("inf"), float("-inf")
    left[:, ::2], right[:, :, ::2] = left[:, ::2].abs(), right[:, :, ::2].abs()
    right[:, :, 5], left[:, 9] = right[:, :, 5].abs(), left[:, 9].abs()
    want = ref.low_rank(x, left, right, indices, base, 0.5)
    assert torch.isinf(want[0]).any()
    same_infinities(switch_low_rank(x, left, right, indices, base=base, scale=0.5), want)
    same_infinities(switch_low_rank_grads(grad, x, left, right, indices, weight_grad=False)[0], ref.low_rank_grads(grad, x, left, right, indices, 1.0)[0])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,sets,inp,out,rank", [(24, 2, 128, 72, 8), (70, 3, 264, 136, 40), (300, 2, 136, 200, 16), (180, 4, 136, 72, 100), (900, 3, 264, 100, 64), (600, 1, 72, 520, 128)])
def test_an_infinity_of_a_row_is_one_of_the_factors_gradients(cuda, rows, sets, inp, out, rank, dtype):
    """Inner vectors and, for fp16, the rows enter these products in two parts; so does what meets an infinity."""
    from keep_b200.low_rank import switch_low_rank_grads

    x, left, right, indices, _, grad = make(cuda, rows, 1, sets, inp, out, rank, dtype=dtype, seed=rank)
    indices[:sets, 0] = torch.arange(sets, device=cuda)
    inf = float("inf")
    for of_x, of_grad in (([(0, 5, inf)], []), ([], [(0, 9, -inf)]), ([(0, 5, inf), (sets, 5, -inf), (sets + 1, 7, inf)], []), ([(0, 5, inf)], [(sets - 1, 9, inf), (sets + 2, 9, -inf)])):
        a, g = x.clone(), grad.clone()
        for r, c, v in of_x:
            a[r, c] = v
        for r, c, v in of_grad:
            g[r, 0, c] = v
        got, want = switch_low_rank_grads(g, a, left, right, indices, scale=0.5), ref.low_rank_grads(g, a, left, right, indices, 0.5)
        assert torch.isinf(want[1][0]).any() or torch.isinf(want[2][0]).any()
        same_infinities(got[1], want[1])
        same_infinities(got[2], want[2])
