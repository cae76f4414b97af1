"""Products over 16-bit experts (switch_matmul and its gradients) against a plain 64-bit form."""

import pytest
import torch

import switch_reference as ref

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def make(cuda, tokens, k, experts, inp, out, dtype=BF16, per_route=False, dead=0.0, seed=0, one_expert=None):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=cuda)  # noqa: E731
    x = rand(*((tokens, k, inp) if per_route else (tokens, inp))).to(dtype)
    weight = (rand(experts, out, inp) * inp ** -0.5).to(dtype)
    indices = ref.picks(gen, tokens, k, experts, dead) if one_expert is None else torch.full((tokens, k), one_expert, dtype=torch.int32, device=cuda)
    return x, weight, indices, (0.1 * rand(tokens, k, out)).to(dtype)


# tokens, picks, experts, in, out: single tokens, sizes below and across the tiles, widths that fill no tile,
# one expert for all, more experts than routes, hundreds of routes an expert
SIZES = [(1, 6, 8, 256, 136), (1, 1, 1, 8, 8), (3, 2, 5, 72, 200), (17, 4, 6, 136, 72), (130, 1, 1, 128, 264), (5, 6, 300, 64, 40), (257, 6, 7, 520, 136),
         (700, 2, 3, 64, 1000), (64, 6, 48, 1024, 512), (1021, 6, 24, 392, 328)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("per_route", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(cuda, size, per_route, dtype):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, *size, dtype=dtype, per_route=per_route, dead=0.15 if size[0] > 2 else 0.0, seed=sum(size))
    ref.close(switch_matmul(x, weight, indices), ref.matmul(x, weight, indices))
    dx, dweight = switch_matmul_grads(grad, x, weight, indices)
    want_x, want_w = ref.matmul_grads(grad, x, weight, indices)
    ref.close(dx, want_x)
    ref.close(dweight, want_w)


@pytest.mark.parametrize("out", [1, 7, 100, 513])
def test_output_widths_that_are_no_multiple_of_eight(cuda, out):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 37, 3, 5, 264, out, dead=0.2, seed=out)
    ref.close(switch_matmul(x, weight, indices), ref.matmul(x, weight, indices))
    for got, want in zip(switch_matmul_grads(grad, x, weight, indices), ref.matmul_grads(grad, x, weight, indices)):
        ref.close(got, want)


def test_dead_routes_only_and_routes_of_one_expert_only(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    for k in (1, 3):
        x, weight, indices, grad = make(cuda, 19, k, 4, 128, 72, one_expert=-1)
        assert not switch_matmul(x, weight, indices).any()
        assert not any(g.any() for g in switch_matmul_grads(grad, x, weight, indices))
        x, weight, indices, grad = make(cuda, 190, k, 4, 128, 72, one_expert=2)  # the same index several times in a row of picks
        ref.close(switch_matmul(x, weight, indices), ref.matmul(x, weight, indices))
        dx, dweight = switch_matmul_grads(grad, x, weight, indices)
        ref.close(dx, ref.matmul_grads(grad, x, weight, indices)[0])
        assert not dweight[[0, 1, 3]].any()


def test_values_that_are_not_finite_stay_where_they_belong(cuda):
    """Neighbouring experts, tokens and rows share tiles with them."""
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 40, 1, 3, 136, 200, seed=3)
    indices[:] = torch.arange(40, device=cuda)[:, None] % 2
    want, want_grads = ref.matmul(x, weight, indices), ref.matmul_grads(grad, x, weight, indices)
    for bad in (float("nan"), float("inf")):
        w = weight.clone()
        w[2] = bad  # an expert without routes, right behind the last with some
        ref.close(switch_matmul(x, w, indices), want)
        ref.close(switch_matmul_grads(grad, x, w, indices)[0], want_grads[0])
        w = weight.clone()
        w[1] = bad
        keep = indices[:, 0] == 0
        ref.close(switch_matmul(x, w, indices)[keep], [t[keep] for t in want])
        ref.close(switch_matmul_grads(grad, x, w, indices)[0][keep], [t[keep] for t in want_grads[0]])
        rows = x.clone()
        rows[7] = bad  # expert 1's
        got = switch_matmul(rows, weight, indices)
        others = torch.arange(40, device=cuda) != 7
        ref.close(got[others], [t[others] for t in want])
        assert not torch.isfinite(got[7]).any()
        ref.close(switch_matmul_grads(grad, rows, weight, indices)[1][0], [t[0] for t in want_grads[1]])
        g = grad.clone()
        g[9] = bad
        dx, dweight = switch_matmul_grads(g, x, weight, indices)
        others = torch.arange(40, device=cuda) != 9
        ref.close(dx[others], [t[others] for t in want_grads[0]])
        ref.close(dweight[0], [t[0] for t in want_grads[1]])


@pytest.mark.parametrize("kind", [torch.int64, torch.uint32, torch.int16])
def test_index_types(cuda, kind):
    from keep_b200.dense_switch import switch_matmul

    x, weight, indices, _ = make(cuda, 9, 2, 4, 64, 48)
    want = switch_matmul(x, weight, indices)
    if kind == torch.uint32:
        indices[2, 1] = -1
        want[2, 1] = 0
        other = indices.view(torch.uint32)
    else:
        other = indices.to(kind)
    if kind == torch.int64:
        other[3, 0] += 1 << 32  # not an expert, whatever its low word says
        want[3, 0] = 0
    assert torch.equal(switch_matmul(x, weight, other), want)


def test_strides_alignment_and_leading_shapes(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 12, 2, 4, 64, 48)
    want, (want_x, want_w) = switch_matmul(x, weight, indices), switch_matmul_grads(grad, x, weight, indices)
    odd = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)  # noqa: E731 - starts 2 bytes into its allocation
    across = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    for change in (odd, across):
        assert torch.equal(switch_matmul(change(x), change(weight), indices.t().contiguous().t()), want)
        dx, dw = switch_matmul_grads(change(grad), change(x), change(weight), indices)
        assert torch.equal(dx, want_x) and torch.equal(dw, want_w)
    assert torch.equal(switch_matmul(x.view(3, 4, 64), weight, indices.view(3, 4, 2)), want.view(3, 4, 2, 48))
    assert torch.equal(switch_matmul(x[5], weight, indices[5]), want[5])


def test_no_routes(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 4, 2, 3, 64, 48)
    assert tuple(switch_matmul(x[:0], weight, indices[:0]).shape) == (0, 2, 48)
    assert tuple(switch_matmul(x, weight, indices[:, :0]).shape) == (4, 0, 48)
    dx, dw = switch_matmul_grads(grad[:, :0], x, weight, indices[:, :0])
    assert tuple(dx.shape) == (4, 64) and not dx.any() and not dw.any()


def test_a_call_repeats_bit_for_bit_and_does_not_depend_on_the_order_of_other_rows(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 777, 6, 10, 512, 264, seed=8)
    y, (dx, dw) = switch_matmul(x, weight, indices), switch_matmul_grads(grad, x, weight, indices)
    for _ in range(3):
        assert torch.equal(switch_matmul(x, weight, indices), y)
        again = switch_matmul_grads(grad, x, weight, indices)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    only_x, none = switch_matmul_grads(grad, x, weight, indices, weight_grad=False)
    assert none is None and torch.equal(only_x, dx)
    none, only_w = switch_matmul_grads(grad, x, weight, indices, x_grad=False)
    assert none is None and torch.equal(only_w, dw)


def test_gradients_against_differences(cuda):
    """Small integers: every product, sum and rounding is exact, and the product is linear in x and in the
    weights, so a central difference IS the derivative along its direction."""
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    gen = torch.Generator(device=cuda).manual_seed(4)
    ints = lambda *shape: torch.randint(-1, 2, shape, generator=gen, device=cuda).to(BF16)  # noqa: E731
    x, weight, grad = ints(20, 40), ints(3, 24, 40), ints(20, 2, 24)
    indices = ref.picks(gen, 20, 2, 3, dead=0.2)
    dx, dw = switch_matmul_grads(grad, x, weight, indices)
    for _ in range(4):
        d, e = ints(20, 40), ints(3, 24, 40)
        of_x = (switch_matmul(x + d, weight, indices).double() - switch_matmul(x - d, weight, indices).double()) / 2
        of_w = (switch_matmul(x, weight + e, indices).double() - switch_matmul(x, weight - e, indices).double()) / 2
        assert (grad.double() * of_x).sum() == (dx.double() * d.double()).sum()
        assert (grad.double() * of_w).sum() == (dw.double() * e.double()).sum()


def test_autograd_records_the_same_gradients(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 30, 3, 5, 128, 72)
    want = switch_matmul_grads(grad, x, weight, indices)
    xs, ws = x.clone().requires_grad_(), weight.clone().requires_grad_()
    switch_matmul(xs, ws, indices).backward(grad)
    assert torch.equal(xs.grad, want[0]) and torch.equal(ws.grad, want[1])
    frozen = x.clone().requires_grad_()
    y = switch_matmul(frozen, weight, indices)
    assert torch.equal(torch.autograd.grad(y, frozen, grad)[0], want[0])
    with torch.no_grad():
        assert not switch_matmul(xs, ws, indices).requires_grad


def test_captured_calls_follow_their_inputs(cuda):
    from keep_b200 import _lib
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 50, 2, 6, 128, 136, dead=0.1)
    leaf = x.clone().requires_grad_()
    alive = switch_matmul(leaf, weight, indices)  # an eager graph of a leaf, alive during the capture
    graphs, outs = [], []
    for _ in range(2):  # two graphs, replayed in turn: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            outs.append((switch_matmul(x, weight, indices), *switch_matmul_grads(grad, x, weight, indices)))
        graphs.append(graph)
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(_lib.KeepVQError, match="cannot be captured"):
            switch_matmul(leaf, weight, indices)
    torch.autograd.grad(alive, leaf, grad)
    for seed in (1, 2):
        new = make(cuda, 50, 2, 6, 128, 136, dead=0.1, seed=seed)
        for old, fresh in zip((x, weight, indices, grad), new):
            old.copy_(fresh)
        want = (switch_matmul(x, weight, indices), *switch_matmul_grads(grad, x, weight, indices))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_on_two_streams_at_once(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    problems = [make(cuda, 300, 3, 8, 512, 264, seed=s) for s in (1, 2)]
    want = [(switch_matmul(x, w, i), *switch_matmul_grads(g, x, w, i)) for x, w, i, g in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, (stream, (x, w, i, g)) in enumerate(zip(streams, problems)):
            with torch.cuda.stream(stream):
                got[n].append((switch_matmul(x, w, i), *switch_matmul_grads(g, x, w, i)))
    torch.cuda.synchronize()
    for n in range(2):
        for result in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(result, want[n]))


def test_many_tiles_of_a_block_and_calls_that_follow_one_another_at_once(cuda):
    """Several tiles of both gradients for every block, ragged experts, and calls enqueued without a wait between them."""
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    x, weight, indices, grad = make(cuda, 1500, 2, 5, 2048, 4096, dead=0.1, seed=5)
    indices[:900, 0] = 1  # one expert with most of the routes
    indices[:, 1][indices[:, 1] == 3] = 4  # one without any
    ref.close(switch_matmul(x, weight, indices), ref.matmul(x, weight, indices))
    want = ref.matmul_grads(grad, x, weight, indices)
    for got in [switch_matmul_grads(grad, x, weight, indices) for _ in range(40)][::13]:
        ref.close(got[0], want[0])
        ref.close(got[1], want[1])


def test_weights_beyond_32_bit_offsets(cuda):
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    experts, out, inp = 1100, 1024, 2048  # 2.3e9 values
    weight = torch.zeros((experts, out, inp), dtype=BF16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    for e in (0, experts - 1):
        weight[e] = torch.randn((out, inp), generator=gen, device=cuda).to(BF16)
    x = torch.randn((40, inp), generator=gen, device=cuda).to(BF16)
    grad = torch.randn((40, 2, out), generator=gen, device=cuda).to(BF16)
    indices = torch.tensor([[0, experts - 1]], dtype=torch.int32, device=cuda).repeat(40, 1)
    small = weight[[0, experts - 1]]
    few = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda).repeat(40, 1)
    ref.close(switch_matmul(x, weight, indices), ref.matmul(x, small, few))
    dx, dw = switch_matmul_grads(grad, x, weight, indices)
    want_x, want_w = ref.matmul_grads(grad, x, small, few)
    ref.close(dx, want_x)
    ref.close(dw[[0, experts - 1]], want_w)
    assert not dw[1:experts - 1].any()


def test_rows_beyond_32_bit_offsets(cuda):
    """2.2e9 values in the result and its gradient, 1.1e9 in x and the copies of rows; a few rows at both ends that are not zero."""
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads

    tokens, out, inp = 135_000, 8192, 4096
    gen = torch.Generator(device=cuda).manual_seed(3)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=cuda).to(BF16)  # noqa: E731
    ends = torch.cat([torch.arange(9, device=cuda), torch.arange(tokens - 9, tokens, device=cuda)])
    x, grad = torch.zeros((tokens, inp), dtype=BF16, device=cuda), torch.zeros((tokens, 2, out), dtype=BF16, device=cuda)
    x[ends], grad[ends] = rand(18, inp), rand(18, 2, out)
    weight = rand(4, out, inp) / 64
    first = torch.arange(tokens, device=cuda, dtype=torch.int32) % 4
    indices = torch.stack([first, 3 - first], dim=1)
    got = switch_matmul(x, weight, indices)
    ref.close(got[ends], ref.matmul(x[ends], weight, indices[ends]))
    assert not got[9:tokens - 9].any()
    del got
    want = ref.matmul_grads(grad[ends], x[ends], weight, indices[ends])
    dx, dweight = switch_matmul_grads(grad, x, weight, indices)
    ref.close(dx[ends], want[0])
    assert not dx[9:tokens - 9].any()
    ref.close(dweight, want[1])


@pytest.mark.parametrize("inp,out,experts", [(520, 300, 40), (1416, 520, 32)])
def test_weight_gradients_whose_last_columns_fill_no_tile(cuda, inp, out, experts):
    """Blocks take several tiles each, now inside the matrix, now across or behind its last columns, and experts without routes
    between them (whose zeros wait for nothing): no tile's values may end up in another's place.  Calls enqueued one after the other."""
    from keep_b200.dense_switch import switch_matmul_grads

    for used, tokens in ((experts, 300), (experts // 3, 90)):
        x, weight, _, grad = make(cuda, tokens, 2, experts, inp, out, seed=inp)
        indices = 3 * ref.picks(torch.Generator(device=cuda).manual_seed(4), tokens, 2, used) if used < experts else ref.picks(torch.Generator(device=cuda).manual_seed(4), tokens, 2, used)
        want = ref.matmul_grads(grad, x, weight, indices)[1]
        for got in [switch_matmul_grads(grad, x, weight, indices, x_grad=False)[1] for _ in range(20)]:
            ref.close(got, want)


@pytest.mark.parametrize("size", [(9, 2, 4, 256, 136), (700, 2, 3, 320, 520)])
def test_a_wait_that_runs_out_is_reported(cuda, size):
    """A call whose loaders of routes leave after their first tile: every other warp's wait runs into its limit of 2 ms, the blocks
    return, the device says so once, and the next calls are what they always are.  Both forms of the kernel, both directions."""
    import time

    from keep_b200 import _lib
    from keep_b200.dense_switch import switch_matmul, switch_matmul_grads, switch_matmul_wait_expired

    x, weight, indices, grad = make(cuda, *size)
    tokens, k, experts, inp, out = size
    want = (switch_matmul(x, weight, indices), *switch_matmul_grads(grad, x, weight, indices))
    assert not switch_matmul_wait_expired() and not switch_matmul_wait_expired(cuda)
    lib = _lib.load()
    result, dx, dweight = torch.empty_like(grad), torch.empty_like(x), torch.empty_like(weight)
    for grads in (0, 1):
        nbytes = int(lib.keepvq_switch_matmul_workspace_bytes(tokens * k, experts, out, inp, k, grads))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=cuda)
        args = _lib.SwitchMatmulArgs(x=x.data_ptr(), weight=weight.data_ptr(), grad=grad.data_ptr(), dtype=_lib.dtype_tag(BF16), indices=indices.data_ptr(), index_bits=32, x_div=k,
                                     routes=tokens * k, experts=experts, out_dim=out, in_dim=inp, grad_ld=out, out=result.data_ptr(), dx=dx.data_ptr(),
                                     dweight=dweight.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=nbytes)
        start = time.monotonic()
        _lib.check(lib.keepvq_switch_matmul_wait_selftest(args, grads, 2_000_000, _lib.stream_handle(cuda)), "keepvq_switch_matmul_wait_selftest")
        assert switch_matmul_wait_expired()
        assert time.monotonic() - start < 1.0
        assert int(ws[:4].view(torch.int32).item()) == 1
        assert not switch_matmul_wait_expired()  # told once
    for _ in range(3):
        again = (switch_matmul(x, weight, indices), *switch_matmul_grads(grad, x, weight, indices))
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    assert not switch_matmul_wait_expired()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        switch_matmul(x, weight, indices)
        with pytest.raises(_lib.KeepVQError, match="inside a graph capture"):
            switch_matmul_wait_expired()
