"""Operators of an MoE layer step beside the int4 path: what is measured of them.

Four families that a program runs together (norm -> router -> experts -> norm):

  sort     token rows sorted by expert (`ops.dispatch_tokens`) and back with the routed weights
           applied (`ops.combine_tokens`), forward or with the gradients of a training step
  linear   activations quantised per token and multiplied by int8 weights with a scale per channel
           (`ops.int8_linear`)
  experts  the routed experts of a layer on those products (`ops.int8_experts`)
  norm     a block's output normed, gated, scaled and added to the scaled residual, and the next
           block's pre-norm (`ops.block_norm`), forward or with its gradients

A case is a dict of plain values. `prepare` makes what a program holds before the call, `run` makes
one pass, `work` states the bytes and operations that the pass cannot do without, and `exact` gives
the same outputs in 64 bits. Where `own` is false `run` computes the operators in elementary torch
operations in 32 bits.

Definitions the three computations share:
  - slot f = token * top_k + i; rows are ordered by (expert, slot); a slot whose id is outside
    [0, experts) is dropped: it takes a zero row behind the last expert's, and slot_row holds that
    row's bitwise complement;
  - quantised x: q = rint(127 x / a), scale = a / 127, a = the row's largest magnitude;
  - the experts' hidden rows and output rows are rounded to the activations' type, as they are
    where the products are called one by one; so is the residual stream that the pre-norm reads.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------------------ cases
def _sort(tokens, top_k=8, experts=256, hidden=2048, dtype="bf16", dropped=False, train=False):
    return {"op": "sort", "tokens": tokens, "top_k": top_k, "experts": experts, "hidden": hidden,
            "dtype": dtype, "dropped": dropped, "train": train}


def _linear(tokens, k, n, dtype="bf16", bias=False):
    return {"op": "linear", "tokens": tokens, "in": k, "out": n, "dtype": dtype, "bias": bias}


def _experts(tokens, top_k=8, experts=256, hidden=2048, inter=512, dtype="bf16"):
    return {"op": "experts", "tokens": tokens, "top_k": top_k, "experts": experts,
            "hidden": hidden, "inter": inter, "dtype": dtype}


def _norm(tokens, hidden=2048, dtype="bf16", post=True, gate="none", pre=True, train=False):
    return {"op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "post": post,
            "gate": gate, "pre": pre, "train": train}


def listed() -> list[dict]:
    cases = {
        # a small decode batch handed to a caller's own experts: all latency
        "sort_decode": _sort(8),
        # a prefill chunk
        "sort_prefill": _sort(4096),
        # a training step's micro-batch, with gradients
        "sort_train": _sort(8192, train=True),
        # full-precision training of a small model, some slots over their expert's capacity
        "sort_train_odd": _sort(1501, 5, 60, 1000, "fp32", dropped=True, train=True),
        # one user's decode step through a projection: weight streaming
        "linear_decode": _linear(1, 2048, 4096),
        # a serving batch, ragged on every side
        "linear_ragged": _linear(203, 1040, 2001, "fp16", bias=True),
        # a prefill chunk through a large projection: the largest case
        "linear_prefill": _linear(8192, 4096, 8192),
        # decode batch through the experts of a layer
        "experts_decode": _experts(16),
        # a prefill chunk through the experts of a layer
        "experts_prefill": _experts(4096),
        # one decode step between two blocks
        "norm_decode": _norm(4),
        # a prefill chunk, gated element by element
        "norm_prefill": _norm(8192, gate="full"),
        # a training step's micro-batch with a per-channel gate (layer scale)
        "norm_train": _norm(16384, gate="channel", train=True),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log(rng, lo, hi, step=1):
    """An integer of [lo, hi], even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng) -> dict:
    op = rng.choice(("sort", "linear", "experts", "norm"))
    if op == "sort":
        experts = rng.choice((8, 16, 60, 64, 128, 256, 512))
        hidden = rng.choice((_log(rng, 64, 2048, 8), _log(rng, 33, 2047), 2048))
        train = rng.random() < 0.5
        return _sort(_log(rng, 1, 8192 if train else 16384), rng.randint(1, 8), experts, hidden,
                     rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.4, train)
    if op == "linear":
        return _linear(_log(rng, 1, 8192), _log(rng, 64, 4096, 16),
                       rng.choice((_log(rng, 64, 8192, 64), _log(rng, 33, 8191))),
                       rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.3)
    if op == "experts":
        return _experts(_log(rng, 1, 4096), rng.randint(1, 8),
                        rng.choice((8, 16, 60, 64, 128, 256)), _log(rng, 256, 2048, 16),
                        _log(rng, 128, 1024, 16), rng.choice(("bf16", "bf16", "fp16")))
    train = rng.random() < 0.5
    hidden = rng.choice((_log(rng, 64, 8192, 8), _log(rng, 33, 4095), 2048))
    tokens = _log(rng, 1, max(1, min(16384, (1 << 25) // hidden)))
    post = rng.random() < 0.7
    return _norm(tokens, hidden, rng.choice(("bf16", "bf16", "fp16", "fp32")), post,
                 rng.choice(("none", "token", "channel", "full")),
                 not post or rng.random() < 0.8, train)


# ------------------------------------------------------------------------------ inputs
def _routing(case, gen):
    """Routed ids and weights with some experts much more in use than others."""
    T, k, E = case["tokens"], case["top_k"], case["experts"]
    popular = -0.5 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    popular = popular[torch.randperm(E, generator=gen, device="cuda")]
    logits = torch.randn(T, E, generator=gen, device="cuda") + popular
    top, ids = logits.topk(k, dim=-1)
    ids = ids.to(torch.int32)
    if case.get("dropped"):
        ids = torch.where(torch.rand(T, k, generator=gen, device="cuda") < 0.1, -1, ids)
    return ids.contiguous(), torch.softmax(top, dim=-1).contiguous()


def _int8(shape, gen):
    """int8 weights as a symmetric quantisation of normal ones leaves them, scales per channel."""
    q = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float16)
    q = q.mul_(32.0).round_().clamp_(-127, 127).to(torch.int8)
    rows = torch.rand(*shape[:-1], generator=gen, device="cuda")
    return q, (0.5 + rows) / (32.0 * math.sqrt(shape[-1]))


def _activations(rows, cols, dtype, gen):
    """Normal activations with a few channels much larger than the rest."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.005, 8.0, 1.0)
    return x.to(dtype)


def prepare(case: dict, seed: int):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
    state = {"case": case}
    T = case["tokens"]
    if case["op"] == "sort":
        S, H = T * case["top_k"], case["hidden"]
        state["ids"], state["weights"] = _routing(case, gen)
        state["x"], state["y"] = randn(T, H), randn(S, H)
        if case["train"]:
            state["drows"], state["dout"] = randn(S, H), randn(T, H)
            for name in ("x", "y", "weights"):
                state[name].requires_grad_()
        return state
    if case["op"] == "linear":
        state["x"] = _activations(T, case["in"], dtype, gen)
        state["w"], state["ws"] = _int8((case["out"], case["in"]), gen)
        state["bias"] = randn(case["out"]) if case["bias"] else None
        return state
    if case["op"] == "experts":
        E, H, I = case["experts"], case["hidden"], case["inter"]
        state["ids"], state["weights"] = _routing(case, gen)
        state["x"] = _activations(T, H, dtype, gen)
        for name, shape in (("gate", (E, I, H)), ("up", (E, I, H)), ("down", (E, H, I))):
            state[name], state[name + "_scale"] = _int8(shape, gen)
        if own:
            from mtp_amd.weights import Int8Experts
            state["experts"] = Int8Experts(*(state[n + s] for n in ("gate", "up", "down")
                                             for s in ("", "_scale")))
        return state
    H = case["hidden"]
    state["y"], state["res"] = randn(T, H), randn(T, H)
    state["post"] = 0.1 * randn(H) if case["post"] else None
    state["pre"] = 0.1 * randn(H) if case["pre"] else None
    shape = {"none": None, "token": (T, 1), "channel": (H,), "full": (T, H)}[case["gate"]]
    state["gate"] = None if shape is None else 0.5 + 0.2 * randn(*shape)
    if case["train"]:
        state["dr"] = randn(T, H)
        state["dx"] = randn(T, H) if case["pre"] else None
        for name in ("y", "res", "post", "pre", "gate"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# Residual and branch scales of the norm cases.
RES_SCALE, BRANCH_SCALE = 0.875, 1.25


# ------------------------------------------------------------------------------ the framework's
def _run_own(s):
    from mtp_amd import ops

    case = s["case"]
    if case["op"] == "sort":
        d = ops.dispatch_tokens(s["x"], s["ids"], case["experts"])
        out = ops.combine_tokens(s["y"], d.slot_row, s["weights"])
        res = {"rows": d.rows, "offsets": d.offsets, "row_slot": d.row_slot,
               "slot_row": d.slot_row, "out": out}
        if case["train"]:
            res["dx"], res["dy"], res["dweights"] = torch.autograd.grad(
                (d.rows, out), (s["x"], s["y"], s["weights"]), (s["drows"], s["dout"]))
        return res
    if case["op"] == "linear":
        return ops.int8_linear(s["x"], s["w"], s["ws"], bias=s["bias"])
    if case["op"] == "experts":
        return ops.int8_experts(s["x"], s["ids"], s["weights"], s["experts"])
    r, x = ops.block_norm(s["y"], s["res"], post_w=s["post"], gate=s["gate"], pre_w=s["pre"],
                          res_scale=RES_SCALE, branch_scale=BRANCH_SCALE, eps=EPS)
    res = {"res": r, "x": x}
    if case["train"]:
        outs, grads = ((r,), (s["dr"],)) if x is None else ((r, x), (s["dr"], s["dx"]))
        names = [n for n in ("y", "res", "post", "gate", "pre") if s[n] is not None]
        got = torch.autograd.grad(outs, [s[n] for n in names], grads)
        res.update({"d" + n: g for n, g in zip(names, got)})
    return res


# ------------------------------------------------------------------------------ plain forms
def _plain_quantize(x):
    x = x.float()
    a = x.abs().amax(dim=-1, keepdim=True)
    q = (x * 127.0 / a).round().nan_to_num(0.0, 0.0, 0.0)
    return q, a / 127.0


def _plain_product(q, w):
    """Exact sums of int8 products in float32 (64-bit sums of pieces below 2^24)."""
    acc = torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    for k in range(0, q.shape[1], 1024):
        acc += q[:, k:k + 1024] @ w[:, k:k + 1024].float().T
    return acc.float()


def _plain_sort(ids, experts):
    key = torch.where((ids >= 0) & (ids < experts), ids, experts).reshape(-1)
    row_slot = torch.sort(key, stable=True).indices
    edges = torch.arange(experts + 1, device=ids.device, dtype=key.dtype)
    offsets = torch.searchsorted(key[row_slot].contiguous(), edges).to(torch.int32)
    place = torch.empty_like(row_slot)
    place[row_slot] = torch.arange(row_slot.numel(), device=ids.device)
    slot_row = torch.where(key < experts, place, ~place).to(torch.int32)
    return row_slot.to(torch.int32), slot_row.view(ids.shape), offsets


def _plain_combine(rows, slot_row, weights):
    kept = slot_row >= 0
    picked = rows[torch.where(kept, slot_row, 0).long()].float()
    return ((weights * kept)[..., None] * picked).sum(dim=1)


def _plain_run_sort(s):
    case, dtype = s["case"], s["x"].dtype
    k = case["top_k"]
    row_slot, slot_row, offsets = _plain_sort(s["ids"], case["experts"])
    kept = slot_row >= 0
    x, y, w = s["x"].detach(), s["y"].detach(), s["weights"].detach()
    live = kept.reshape(-1)[row_slot.long()]
    rows = x[row_slot.long() // k] * live[:, None]
    res = {"rows": rows, "offsets": offsets, "row_slot": row_slot, "slot_row": slot_row,
           "out": _plain_combine(y, slot_row, w).to(dtype)}
    if case["train"]:
        res["dx"] = _plain_combine(s["drows"], slot_row, torch.ones_like(w)).to(dtype)
        wr = (w * kept).reshape(-1)[row_slot.long()]
        dout = s["dout"][row_slot.long() // k].float()
        res["dy"] = (wr[:, None] * dout).to(dtype)
        dw = torch.zeros(w.numel(), device=w.device)
        dw[row_slot.long()] = (dout * y.float()).sum(dim=-1) * live
        res["dweights"] = dw.view(w.shape)
    return res


def _plain_run_linear(s):
    q, scale = _plain_quantize(s["x"])
    y = _plain_product(q, s["w"]) * scale * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_run_experts(s):
    case, x = s["case"], s["x"]
    row_slot, slot_row, offsets = _plain_sort(s["ids"], case["experts"])
    q, scale = _plain_quantize(x)
    y = torch.zeros(row_slot.numel(), case["hidden"], dtype=x.dtype, device=x.device)
    ends = offsets.tolist()
    for e in range(case["experts"]):
        if ends[e] == ends[e + 1]:
            continue
        t = row_slot[ends[e]:ends[e + 1]].long() // case["top_k"]
        qe, se = q[t], scale[t]
        g = _plain_product(qe, s["gate"][e]) * se * s["gate_scale"][e]
        u = _plain_product(qe, s["up"][e]) * se * s["up_scale"][e]
        h = (g / (1.0 + torch.exp(-g)) * u).to(x.dtype)
        qh, sh = _plain_quantize(h)
        y[ends[e]:ends[e + 1]] = (_plain_product(qh, s["down"][e]) * sh
                                  * s["down_scale"][e]).to(x.dtype)
    return _plain_combine(y, slot_row, s["weights"]).to(x.dtype)


def _sum_to(t, shape):
    for dim, n in enumerate((1,) * (t.dim() - len(shape)) + tuple(shape)):
        if n == 1 and t.shape[dim] != 1:
            t = t.sum(dim=dim, keepdim=True)
    return t.reshape(shape)


def _plain_run_norm(s):
    case, dtype = s["case"], s["y"].dtype
    f = {n: None if s[n] is None else s[n].detach().float()
         for n in ("y", "res", "post", "gate", "pre")}
    y = f["y"]
    gate = 1.0 if f["gate"] is None else f["gate"]
    if case["post"]:
        ry = torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + EPS)
        p = y * ry * (1.0 + f["post"])
    else:
        p = y
    r = (RES_SCALE * f["res"] + BRANCH_SCALE * gate * p).to(dtype)
    u = r.float()
    x = None
    if case["pre"]:
        rr = torch.rsqrt((u * u).mean(dim=-1, keepdim=True) + EPS)
        x = (u * rr * (1.0 + f["pre"])).to(dtype)
    res = {"res": r, "x": x}
    if case["train"]:
        du = s["dr"].float()
        if case["pre"]:
            dx, uh = s["dx"].float(), u * rr
            g = dx * (1.0 + f["pre"])
            du = du + rr * (g - uh * (g * uh).mean(dim=-1, keepdim=True))
        db = BRANCH_SCALE * du
        dp = db * gate
        if case["post"]:
            yh, g = y * ry, dp * (1.0 + f["post"])
            res["dy"] = (ry * (g - yh * (g * yh).mean(dim=-1, keepdim=True))).to(dtype)
        else:
            res["dy"] = dp.to(dtype)
        res["dres"] = (RES_SCALE * du).to(dtype)
        if case["post"]:
            res["dpost"] = (dp * yh).sum(dim=0).to(dtype)
        if f["gate"] is not None:
            res["dgate"] = _sum_to(db * p, s["gate"].shape).to(dtype)
        if case["pre"]:
            res["dpre"] = (dx * uh).sum(dim=0).to(dtype)
    return res


def run(state):
    if own:
        return _run_own(state)
    return {"sort": _plain_run_sort, "linear": _plain_run_linear, "experts": _plain_run_experts,
            "norm": _plain_run_norm}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ work
def work(case: dict) -> dict:
    T, es = case["tokens"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "sort":
        k, H, S = case["top_k"], case["hidden"], case["tokens"] * case["top_k"]
        # x -> rows, y -> out; ids, weights and the three tables
        b = 2 * (T + S) * H * es + S * 16 + 4 * (case["experts"] + 1)
        f = 2 * S * H
        if case["train"]:
            # drows -> dx; dout and y -> dy; weights' gradient (y is read once for both passes)
            b += (S + T) * H * es + (T + S) * H * es + S * 4
            f += S * H + 3 * S * H
        return {"bytes": b, "flops": f}
    if case["op"] == "linear":
        K, N = case["in"], case["out"]
        return {"bytes": T * K * es + N * K + 4 * N + T * N * es + (N * es if case["bias"] else 0),
                "flops": 2 * T * K * N}
    if case["op"] == "experts":
        E, k, H, I = case["experts"], case["top_k"], case["hidden"], case["inter"]
        # experts that at least one token is expected to reach
        touched = E * (1.0 - (1.0 - k / E) ** T)
        return {"bytes": int(2 * T * H * es + T * k * 8 + touched * (3 * H * I + 8 * I + 4 * H)),
                "flops": 6 * T * k * H * I}
    H = case["hidden"]
    rows = 2 + 1 + (1 if case["pre"] else 0) + (1 if case["gate"] == "full" else 0)
    f = 12 * T * H
    if case["train"]:
        rows += 1 + (1 if case["pre"] else 0) + 2 + (1 if case["gate"] == "full" else 0)
        f += 30 * T * H
    small = (1 if case["post"] else 0) + (1 if case["pre"] else 0) + (case["gate"] == "channel")
    return {"bytes": (rows * T * H + small * H * (2 if case["train"] else 1)
                      + (T * (2 if case["train"] else 1) if case["gate"] == "token" else 0)) * es,
            "flops": f}


# ------------------------------------------------------------------------------ 64 bits
def _exact_quantize(x):
    x = x.double()
    peak = x.abs().max(dim=-1).values[:, None]
    q = torch.where(peak > 0, torch.round(127.0 * x / peak.clamp_min(1e-300)), 0.0)
    return q, peak / 127.0


def _exact_order(ids, experts):
    """(slots of each expert in order, dropped slots last), on the host."""
    flat = ids.reshape(-1).tolist()
    groups = [[] for _ in range(experts + 1)]
    for slot, e in enumerate(flat):
        groups[e if 0 <= e < experts else experts].append(slot)
    return groups


def _exact_sort(case, s):
    T, k, H, E = case["tokens"], case["top_k"], case["hidden"], case["experts"]
    x, y, w = (s[n].detach().double() for n in ("x", "y", "weights"))
    groups = _exact_order(s["ids"], E)
    order = torch.tensor([f for g in groups for f in g])
    offsets = torch.tensor([0] + [len(g) for g in groups[:E]]).cumsum(0).to(torch.int32)
    n = int(offsets[-1])
    row = torch.empty(T * k, dtype=torch.long)
    row[order] = torch.arange(T * k)
    slot_row = row.clone()
    slot_row[order[n:]] = ~row[order[n:]]
    dev = x.device
    kept_slots, order_d = order[:n].to(dev), order.to(dev)
    token = kept_slots // k
    rows = torch.zeros(T * k, H, dtype=torch.float64, device=dev)
    rows[:n] = x[token]
    wk = w.reshape(-1)[kept_slots][:, None]
    out = torch.zeros(T, H, dtype=torch.float64, device=dev).index_add_(0, token, wk * y[:n])
    res = {"rows": rows, "offsets": offsets.to(dev), "row_slot": order_d.to(torch.int32),
           "slot_row": slot_row.to(torch.int32).view(T, k).to(dev), "out": out}
    if case["train"]:
        drows, dout = s["drows"].double(), s["dout"].double()
        res["dx"] = torch.zeros_like(out).index_add_(0, token, drows[:n])
        res["dy"] = torch.zeros_like(rows)
        res["dy"][:n] = wk * dout[token]
        dw = torch.zeros(T * k, dtype=torch.float64, device=dev)
        dw[kept_slots] = torch.linalg.vecdot(dout[token], y[:n])
        res["dweights"] = dw.view(T, k)
    return res


def _exact_experts(case, s):
    k, dtype = case["top_k"], s["x"].dtype
    q, scale = _exact_quantize(s["x"])
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=q.device)
    weights = s["weights"].double().reshape(-1)
    flat = s["ids"].reshape(-1)
    for e in flat.unique().tolist():
        slots = (flat == e).nonzero()[:, 0]
        t = slots // k

        def part(name, a, a_scale):
            return (a @ s[name][e].double().T) * a_scale * s[name + "_scale"][e].double()

        g = part("gate", q[t], scale[t])
        h = (torch.sigmoid(g) * g * part("up", q[t], scale[t])).to(dtype)
        y = part("down", *_exact_quantize(h)).to(dtype).double()
        out.index_add_(0, t, weights[slots, None] * y)
    return out


def _exact_norm(case, s):
    d = lambda n: s[n].detach().double()  # noqa: E731
    one = torch.ones((), dtype=torch.float64, device="cuda")
    H, dtype = case["hidden"], s["y"].dtype
    # (t * inv(t)) has a mean square of one but for eps
    inv = lambda t: (t.pow(2).sum(-1, keepdim=True) / H + EPS) ** -0.5  # noqa: E731
    gate = one if s["gate"] is None else d("gate")
    wpost = one + d("post") if case["post"] else None
    branch = d("y") * inv(d("y")) * wpost if case["post"] else d("y")
    stream = (RES_SCALE * d("res") + gate * branch * BRANCH_SCALE).to(dtype).double()
    res = {"res": stream, "x": stream * inv(stream) * (one + d("pre")) if case["pre"] else None}
    if case["train"]:
        # d(t * inv(t)) . v  =  inv(t) v - t inv(t)^3 <t, v> / H
        pull = lambda t, v: inv(t) * v - t * inv(t) ** 3 * (t * v).sum(-1, keepdim=True) / H  # noqa: E731
        ds = s["dr"].double()
        if case["pre"]:
            ds = ds + pull(stream, s["dx"].double() * (one + d("pre")))
            dpre = (s["dx"].double() * stream * inv(stream)).sum(0)
        dbranch = BRANCH_SCALE * gate * ds
        res["dy"] = pull(d("y"), dbranch * wpost) if case["post"] else dbranch
        res["dres"] = RES_SCALE * ds
        if case["post"]:
            res["dpost"] = (dbranch * d("y") * inv(d("y"))).sum(0)
        if s["gate"] is not None:
            full = BRANCH_SCALE * ds * branch
            res["dgate"] = {"token": lambda: full.sum(1, keepdim=True),
                            "channel": lambda: full.sum(0), "full": lambda: full}[case["gate"]]()
        if case["pre"]:
            res["dpre"] = dpre
    return res


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "sort":
        return _exact_sort(case, s)
    if case["op"] == "linear":
        q, scale = _exact_quantize(s["x"])
        y = (q @ s["w"].double().T) * scale * s["ws"].double()
        return y if s["bias"] is None else y + s["bias"].double()
    return _exact_experts(case, s) if case["op"] == "experts" else _exact_norm(case, s)
