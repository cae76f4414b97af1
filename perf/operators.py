"""Switch products over 16-bit experts and over low-rank adapters: the cases they are timed on.

Every route (a token's pick, or a row of its own) names one of many weight sets.  ``experts`` cases
are products against 16-bit expert matrices, ``adapters`` cases a low-rank product added onto a
base; the ``_grad`` kinds are the gradients a training step asks for.  Tokens are N(0, 1), weights
N(0, 1 / width), picks of a router without or with a Zipf(1.1) preference.
"""

from __future__ import annotations

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # single-stream decode: one token's gate projections, an expert layer kept in 16 bits
        {"name": "experts_token", "kind": "experts", "tokens": 1, "picks": 6, "per_route": False, "experts": 384, "in": 4096, "out": 2048, "zipf": False, "dtype": "bf16"},
        # the down projection of a three-token draft on layers of the shipped shape: a row per route
        {"name": "experts_draft_down", "kind": "experts", "tokens": 3, "picks": 6, "per_route": True, "experts": 192, "in": 2304, "out": 5120, "zipf": False, "dtype": "fp16"},
        # the benchmark's batch of 64: more than half the pool is read for a route or two each
        {"name": "experts_batch", "kind": "experts", "tokens": 64, "picks": 6, "per_route": False, "experts": 384, "in": 4096, "out": 2048, "zipf": False, "dtype": "bf16"},
        # a prefill chunk of odd length, popular and idle experts side by side
        {"name": "experts_prefill_zipf", "kind": "experts", "tokens": 1021, "picks": 6, "per_route": False, "experts": 192, "in": 5120, "out": 2304, "zipf": True, "dtype": "fp16"},
        # a long prefill chunk over the experts of one rank: hundreds of routes each
        {"name": "experts_prefill", "kind": "experts", "tokens": 4096, "picks": 6, "per_route": False, "experts": 32, "in": 4096, "out": 2048, "zipf": False, "dtype": "bf16"},
        # a training step's gate projection: about a hundred routes an expert
        {"name": "experts_grad_1000", "kind": "experts_grad", "tokens": 1000, "picks": 6, "per_route": False, "experts": 64, "in": 4096, "out": 2048, "zipf": False, "dtype": "bf16"},
        # a training step's down projection, a row per route, hundreds of routes an expert
        {"name": "experts_grad_down", "kind": "experts_grad", "tokens": 4096, "picks": 6, "per_route": True, "experts": 32, "in": 2048, "out": 4096, "zipf": False, "dtype": "fp16"},
        # one request with its adapter, one decode step
        {"name": "adapters_token", "kind": "adapters", "tokens": 1, "picks": 1, "per_route": True, "experts": 64, "in": 4096, "out": 4096, "rank": 16, "runs": 1, "dtype": "bf16"},
        # a decode batch of many requests, some of them without an adapter
        {"name": "adapters_batch", "kind": "adapters", "tokens": 61, "picks": 1, "per_route": True, "experts": 128, "in": 4096, "out": 4096, "rank": 32, "runs": 1, "dtype": "fp16"},
        # low-rank sidecars of the experts of a routed layer, a continuous batch of odd size
        {"name": "adapters_sidecar", "kind": "adapters", "tokens": 251, "picks": 6, "per_route": False, "experts": 384, "in": 4096, "out": 2048, "rank": 8, "runs": 1, "dtype": "bf16"},
        # prompts of several requests in one chunk: runs of rows with the same adapter
        {"name": "adapters_prefill", "kind": "adapters", "tokens": 4096, "picks": 1, "per_route": True, "experts": 32, "in": 4096, "out": 4096, "rank": 64, "runs": 512, "dtype": "bf16"},
        # a training step over a batch of sequences, few adapters
        {"name": "adapters_grad", "kind": "adapters_grad", "tokens": 8192, "picks": 1, "per_route": True, "experts": 4, "in": 5120, "out": 2304, "rank": 16, "runs": 1024, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return min(high, int(low * (high / low) ** rng.random() + 0.5))


def draw(rng):
    kind = rng.choice(("experts", "experts", "experts_grad", "adapters", "adapters", "adapters_grad"))
    wide = rng.choice(((4096, 2048), (2048, 4096), (5120, 2304), (2304, 5120), (1000, 1416), (1416, 520)))
    case = {"kind": kind, "tokens": _log_int(rng, 1, 4096), "picks": rng.choice((1, 2, 6)), "per_route": rng.random() < 0.5, "in": wide[0], "out": wide[1],
            "dtype": rng.choice(("bf16", "fp16"))}
    if kind == "experts":
        return {**case, "experts": rng.choice((8, 32, 64, 192)), "zipf": rng.random() < 0.3}
    if kind == "experts_grad":
        return {**case, "tokens": _log_int(rng, 1, 2048), "experts": rng.choice((8, 16, 32)), "zipf": rng.random() < 0.3}
    return {**case, "experts": _log_int(rng, 1, 384), "rank": rng.choice((4, 8, 16, 24, 32, 64)), "runs": rng.choice((1, 1, 64, 512))}


# ---- inputs ------------------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens, picks, experts = DTYPES[case["dtype"]], case["tokens"], case["picks"], case["experts"]
    inp, out = case["in"], case["out"]
    state = {"kind": case["kind"], "x": _normal(gen, (tokens, picks, inp) if case["per_route"] else (tokens, inp), dtype)}
    if "rank" in case:
        # one adapter per run of rows; index -1, one in eight, is a request without one
        runs = -(-tokens // case["runs"])
        chosen = torch.randint(0, experts, (runs, picks), generator=gen, device="cuda", dtype=torch.int32)
        chosen[torch.rand((runs, picks), generator=gen, device="cuda") < (0.125 if runs > 1 else 0.0)] = -1
        state["indices"] = chosen.repeat_interleave(case["runs"], 0)[:tokens].contiguous()
        state["left"] = _normal(gen, (experts, out, case["rank"]), dtype, case["rank"] ** -0.5)
        state["right"] = _normal(gen, (experts, case["rank"], inp), dtype, inp ** -0.5)
        state["scale"] = 0.5
        state["base" if case["kind"] == "adapters" else "grad"] = _normal(gen, (tokens, picks, out), dtype)
    else:
        score = torch.rand((tokens, experts), generator=gen, device="cuda").log_().neg_().log_().neg_()  # Gumbel noise: picks without repetition
        if case["zipf"]:
            score = score - 1.1 * torch.arange(1, experts + 1, device="cuda").log()[torch.randperm(experts, generator=gen, device="cuda")]
        state["indices"] = score.topk(picks, dim=1).indices.to(torch.int32)
        state["weight"] = _normal(gen, (experts, out, inp), dtype, inp ** -0.5)
        if case["kind"] == "experts_grad":
            state["grad"] = _normal(gen, (tokens, picks, out), dtype, 0.05)
    return state


# ---- the plain forms -----------------------------------------------------------------------------

def _grouped(state):
    """The weight sets in use, and where every route stands in ``[sets, most, width]``; routes without a set last."""
    flat = state["indices"].reshape(-1).long()
    sets, which = torch.unique(flat, return_inverse=True)
    counts = torch.bincount(which, minlength=sets.numel())
    order = torch.argsort(which, stable=True)
    place = torch.empty_like(which)
    place[order] = torch.arange(which.numel(), device=which.device) - (counts.cumsum(0) - counts)[which[order]]
    return sets, sets >= 0, which, place, int(counts.max())


def _pad(rows, sets, which, place, most):
    padded = torch.zeros((sets.numel(), most, rows.shape[-1]), dtype=torch.float32, device=rows.device)
    padded[which, place] = rows.float()
    return padded


def _rows(state):
    x, picks = state["x"], state["indices"].shape[1]
    return x.reshape(-1, x.shape[-1]) if x.ndim == 3 else x.repeat_interleave(picks, 0)


def _of(weights, sets, live):
    return weights[sets.clamp(min=0)].float() * live[:, None, None]


def _over_all(grads, weights, sets, live):
    whole = torch.zeros_like(weights)
    whole[sets[live]] = grads[live].to(weights.dtype)
    return whole


def _input_grad(state, routes):
    x = state["x"]
    return (routes.reshape(x.shape) if x.ndim == 3 else routes.reshape(x.shape[0], -1, x.shape[1]).sum(1)).to(x.dtype)


def _plain(state):
    sets, live, which, place, most = _grouped(state)
    x = _pad(_rows(state), sets, which, place, most)
    if "weight" in state:
        weight = _of(state["weight"], sets, live)
        if "grad" not in state:
            y = torch.bmm(x, weight.transpose(1, 2))[which, place]
            return y.reshape(*state["indices"].shape, -1).to(state["x"].dtype)
        grad = _pad(state["grad"].flatten(0, 1), sets, which, place, most)
        dx = torch.bmm(grad, weight)[which, place]
        return {"x": _input_grad(state, dx), "weight": _over_all(torch.bmm(grad.transpose(1, 2), x), state["weight"], sets, live)}
    left, right = _of(state["left"], sets, live), _of(state["right"], sets, live)
    inner = torch.bmm(x, right.transpose(1, 2))
    if "grad" not in state:
        y = torch.bmm(inner, left.transpose(1, 2))[which, place].reshape(state["base"].shape)
        return (state["base"].float() + state["scale"] * y).to(state["base"].dtype)
    grad = _pad(state["grad"].flatten(0, 1), sets, which, place, most) * state["scale"]
    back = torch.bmm(grad, left)
    dx = torch.bmm(back, right)[which, place]
    return {"x": _input_grad(state, dx), "left": _over_all(torch.bmm(grad.transpose(1, 2), inner), state["left"], sets, live),
            "right": _over_all(torch.bmm(back.transpose(1, 2), x), state["right"], sets, live)}


def run(state):
    if not own:
        return _plain(state)
    from keep_b200 import dense_switch, low_rank

    x, indices = state["x"], state["indices"]
    if state["kind"] == "experts":
        return dense_switch.switch_matmul(x, state["weight"], indices)
    if state["kind"] == "experts_grad":
        dx, dw = dense_switch.switch_matmul_grads(state["grad"], x, state["weight"], indices)
        return {"x": dx, "weight": dw}
    if state["kind"] == "adapters":
        return low_rank.switch_low_rank(x, state["left"], state["right"], indices, base=state["base"], scale=state["scale"])
    dx, dleft, dright = low_rank.switch_low_rank_grads(state["grad"], x, state["left"], state["right"], indices, scale=state["scale"])
    return {"x": dx, "left": dleft, "right": dright}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    indices, picks = state["indices"].long(), state["indices"].shape[1]
    x, grad, base = state["x"], state.get("grad"), state.get("base")
    names = [n for n in ("weight", "left", "right") if n in state]
    y = torch.zeros((*indices.shape, case["out"]), dtype=torch.float64, device="cuda") if base is None else base.double()
    dx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    sums = {n: torch.zeros(state[n].shape, dtype=torch.float64, device="cuda") for n in names} if grad is not None else {}
    for e in range(case["experts"]):
        token, pick = torch.nonzero(indices == e, as_tuple=True)
        if token.numel() == 0:
            continue
        rows = (x[token, pick] if case["per_route"] else x[token]).double()
        w = {n: state[n][e].double() for n in names}
        if grad is None:
            y[token, pick] += rows @ w["weight"].T if "weight" in w else state["scale"] * ((rows @ w["right"].T) @ w["left"].T)
            continue
        g = grad[token, pick].double()
        if "weight" in w:
            back, sums["weight"][e] = g @ w["weight"], g.T @ rows
        else:
            g = state["scale"] * g
            inner = g @ w["left"]
            back, sums["right"][e], sums["left"][e] = inner @ w["right"], inner.T @ rows, g.T @ (rows @ w["right"].T)
        if case["per_route"]:
            dx[token, pick] = back
        else:
            dx.index_put_((token,), back, accumulate=True)
    return y if grad is None else {"x": dx, **sums}


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    tokens, experts, inp, out = case["tokens"], case["experts"], case["in"], case["out"]
    routes = tokens * case["picks"]
    rows_x = 2 * inp * (routes if case["per_route"] else tokens)
    rows_y = 2 * out * routes
    if "rank" in case:
        runs = -(-tokens // case["runs"])
        live = 0.875 if runs > 1 else 1.0
        used = experts * (1.0 - (1.0 - 1.0 / experts) ** (runs * case["picks"] * live))
        pair, flops = 2 * case["rank"] * (inp + out), 2 * routes * live * case["rank"] * (inp + out)
        if case["kind"] == "adapters":
            return {"bytes": used * pair + rows_x + 2 * rows_y + 4 * routes, "flops": flops}
        return {"bytes": (used + experts) * pair + 2 * rows_x + rows_y + 4 * routes, "flops": 3 * flops}
    matrix, flops = 2 * inp * out, 2 * routes * inp * out
    # experts that a router touches (without a preference; with one, fewer)
    used = experts * (1.0 - (1.0 - case["picks"] / experts) ** tokens)
    if case["zipf"]:
        mass = [(i + 1) ** -1.1 for i in range(experts)]
        used = sum(1.0 - (1.0 - min(1.0, case["picks"] * m / sum(mass))) ** tokens for m in mass)
    if case["kind"] == "experts":
        return {"bytes": used * matrix + rows_x + rows_y + 4 * routes, "flops": flops}
    return {"bytes": (used + experts) * matrix + 2 * rows_x + rows_y + 4 * routes, "flops": 2 * flops}
