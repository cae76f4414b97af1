"""Plain 64-bit forms of the products over 16-bit experts and low-rank adapters, with the error that a
kernel with 16-bit operands and fp32 sums may make: test infrastructure."""

import torch


def routed_rows(x, indices):
    """One row of x per route, flat."""
    flat = x.reshape(-1, x.shape[-1])
    picks = indices.numel() // max(1, flat.shape[0])
    return flat.repeat_interleave(picks, 0)


def live_sets(indices, sets):
    flat = indices.reshape(-1).to(torch.int64)
    return [(e, torch.nonzero(flat == e).flatten()) for e in range(sets)]


def per_row(routes, x):
    """Routes' rows summed over the picks of x's rows."""
    rows = x.reshape(-1, x.shape[-1]).shape[0]
    return routes.reshape(rows, -1, x.shape[-1]).sum(1).reshape(x.shape)


def sum_error(depth):
    """How far an fp32 sum of `depth` products may be off, relative to the sum of their magnitudes: an
    instruction adds 16 products to the sum so far and may cut what it aligns (2^-22 with its own
    rounding), and a handful of parts are added in the end."""
    return (depth / 16 + 16) * 2.0 ** -22


def rounding(want, dtype):
    """Half a step of `dtype` at every value; fp16 steps stop shrinking at 2^-24."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return want.abs() * (torch.finfo(dtype).eps / 2) + tiny


def matmul(x, weight, indices):
    """(want, bound) of the forward product."""
    rows, sets = routed_rows(x, indices).double(), weight.shape[0]
    want = torch.zeros((rows.shape[0], weight.shape[1]), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(want)
    for e, r in live_sets(indices, sets):
        if r.numel():
            want[r], size[r] = rows[r] @ weight[e].double().T, rows[r].abs() @ weight[e].double().abs().T
    shape = (*indices.shape, weight.shape[1])
    return want.reshape(shape), (rounding(want, x.dtype) + sum_error(x.shape[-1]) * size).reshape(shape)


def matmul_grads(grad, x, weight, indices):
    """((dx, bound), (dweight, bound))."""
    rows, sets = routed_rows(x, indices).double(), weight.shape[0]
    g = grad.reshape(-1, grad.shape[-1]).double()
    dx, dx_size = torch.zeros_like(rows), torch.zeros_like(rows)
    dw = torch.zeros(weight.shape, dtype=torch.float64, device=x.device)
    dw_bound = torch.zeros_like(dw)
    for e, r in live_sets(indices, sets):
        if r.numel():
            w = weight[e].double()
            dx[r], dx_size[r] = g[r] @ w, g[r].abs() @ w.abs()
            dw[e] = g[r].T @ rows[r]
            dw_bound[e] = rounding(dw[e], x.dtype) + sum_error(r.numel()) * (g[r].abs().T @ rows[r].abs())
    dx, dx_size = per_row(dx, x), per_row(dx_size, x)
    return (dx, rounding(dx, x.dtype) + sum_error(weight.shape[1]) * dx_size), (dw, dw_bound)


def split_error(dtype):
    """What is left of a value that enters a product as the sum of two 16-bit ones."""
    return 2.0 ** -17 if dtype == torch.bfloat16 else 2.0 ** -21


def low_rank(x, left, right, indices, base, scale):
    rows, sets = routed_rows(x, indices).double(), left.shape[0]
    out_dtype = x.dtype if base is None else base.dtype
    want = torch.zeros((rows.shape[0], left.shape[1]), dtype=torch.float64, device=x.device)
    if base is not None:
        want += base.reshape(want.shape).double()
    bound = torch.zeros_like(want)
    for e, r in live_sets(indices, sets):
        if r.numel():
            a, b = right[e].double(), left[e].double()
            p, p_size = rows[r] @ a.T, rows[r].abs() @ a.abs().T
            p_error = split_error(x.dtype) * p.abs() + sum_error(x.shape[-1]) * p_size
            want[r] += scale * (p @ b.T)
            bound[r] += abs(scale) * ((p_error + sum_error(left.shape[2]) * p.abs()) @ b.abs().T)
    shape = (*indices.shape, left.shape[1])
    return want.reshape(shape), (rounding(want, out_dtype) + bound + 2.0 ** -23 * want.abs()).reshape(shape)


def low_rank_grads(grad, x, left, right, indices, scale):
    rows, sets = routed_rows(x, indices).double(), left.shape[0]
    g = grad.reshape(-1, grad.shape[-1]).double()
    dx, dx_bound = torch.zeros_like(rows), torch.zeros_like(rows)
    out = [(torch.zeros(w.shape, dtype=torch.float64, device=x.device), torch.zeros(w.shape, dtype=torch.float64, device=x.device)) for w in (left, right)]
    for e, r in live_sets(indices, sets):
        if r.numel():
            a, b = right[e].double(), left[e].double()
            p, p_size = rows[r] @ a.T, rows[r].abs() @ a.abs().T
            q, q_size = scale * (g[r] @ b), abs(scale) * (g[r].abs() @ b.abs())
            split = split_error(x.dtype)
            p_error, q_error = split * p.abs() + sum_error(x.shape[-1]) * p_size, split * q.abs() + sum_error(left.shape[1]) * q_size
            dx[r] = q @ a
            dx_bound[r] = (q_error + sum_error(left.shape[2]) * q.abs()) @ a.abs()
            many = sum_error(r.numel())
            for (want, bound), value, error in ((out[0], scale * (g[r].T @ p), abs(scale) * (g[r].abs().T @ (p_error + many * p.abs()))),
                                                (out[1], q.T @ rows[r], (q_error + many * q.abs()).T @ rows[r].abs())):
                want[e] = value
                bound[e] = error + rounding(value, x.dtype)
    dx, dx_bound = per_row(dx, x), per_row(dx_bound, x)
    return (dx, dx_bound + rounding(dx, x.dtype)), *out


def close(got, want_and_bound):
    want, bound = want_and_bound
    assert tuple(got.shape) == tuple(want.shape), (got.shape, want.shape)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item() if off.numel() else 0.0
    assert worst <= 0, f"off by {off.max().item()} where {bound.flatten()[(off - bound).argmax()].item()} is allowed"


def picks(gen, tokens, k, sets, dead=0.0):
    """k different sets per token, with some of the picks dead: -1, or beyond the last set."""
    idx = torch.rand((tokens, sets), generator=gen, device=gen.device).topk(k, dim=1).indices.to(torch.int32)
    if dead:
        gone = torch.rand(idx.shape, generator=gen, device=gen.device)
        idx = torch.where(gone < dead / 2, -1, torch.where(gone < dead, sets + 5, idx))
    return idx
