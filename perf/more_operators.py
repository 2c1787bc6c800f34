"""Operators around an MoE layer's experts: what is measured of them.

Three families that a decoder layer runs together (norm -> router -> experts, and the dense int4
projections of the same checkpoints beside them):

  int4    a linear layer on int4 weights with a scale and a zero point per group (`ops.int4_linear`),
          from the matrix-vector product of one token to a prefill chunk
  route   router logits to routed ids and weights, tokens per expert, the balance and the z loss
          (`ops.route_tokens`), forward or with the logits' gradient
  norm    layer norm (`ops.layer_norm`), forward or with the gradients of its input, weight and bias

A case is a dict of plain values. `prepare` makes what a program holds before the call, `run` makes
one pass, `work` states the bytes and operations that the pass cannot do without, and `exact` gives
the same outputs in 64 bits. Where `own` is false `run` computes the operators in elementary torch
operations in 32 bits.

Definitions the three computations share:
  - int4: w[k, n] = (q[k, n] - z[k // G, n]) * s[k // G, n] with nibble j of qweight[r, n] as
    q[8 r + j, n] and nibble j of qzeros[g, c] as z[g, 8 c + j]; w is not rounded;
  - route: p = softmax(logits) over a token's experts. The top_k largest logits are chosen, equal ones
    by the lower id; an expert whose logit is -inf is not chosen: its place takes the id -1 and the
    weight 0, behind the chosen ones. A token that the mask leaves out, or that has no expert left, is
    not counted: its ids are -1, its weights and gradient 0. Over the n tokens that count, with c[e]
    slots for expert e,
        balance = E * sum_e (c[e] / (n * top_k)) * mean_t p[t, e],   z = mean_t logsumexp(logits[t])^2
    (both 0 for n = 0); c is not differentiated. Weights are p, divided by their sum over the chosen
    experts where they are renormalised;
  - norm: y = (x - mean) * rsqrt(var + eps) * weight + bias with the biased variance.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5
# Coefficients of the two losses in a training step.
BALANCE_COEF, Z_COEF = 1e-2, 1e-3


# ------------------------------------------------------------------------------ cases
def _int4(tokens, k, n, group=128, dtype="bf16", bias=False):
    return {"op": "int4", "tokens": tokens, "in": k, "out": n, "group": group, "dtype": dtype,
            "bias": bias}


def _route(tokens, experts=256, top_k=8, dtype="fp32", renorm=True, padded=False, blocked=False,
           train=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "renorm": renorm, "padded": padded, "blocked": blocked, "train": train}


def _norm(tokens, hidden=2048, dtype="bf16", bias=True, train=False):
    return {"op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "bias": bias,
            "train": train}


def listed() -> list[dict]:
    cases = {
        # one user's decode step through a projection: weight streaming and latency
        "int4_decode": _int4(1, 2048, 4096),
        # a decode batch through a wide projection
        "int4_batch": _int4(16, 4096, 8192),
        # a serving batch between decode and prefill, ragged sizes and small groups
        "int4_ragged": _int4(203, 1056, 2008, 32, "fp16", bias=True),
        # a prefill chunk through a large projection: the largest case
        "int4_prefill": _int4(4096, 4096, 8192),
        # a decode batch's routing: all latency
        "route_decode": _route(8),
        # a prefill chunk's routing with its load statistics
        "route_prefill": _route(8192, dtype="bf16"),
        # a training step's micro-batch with both losses and the gradient
        "route_train": _route(16384, train=True),
        # padded sequences, experts that some tokens may not use, weights as they come
        "route_train_odd": _route(1501, 60, 5, "fp16", renorm=False, padded=True, blocked=True,
                                  train=True),
        # a few tokens between two blocks
        "norm_decode": _norm(4),
        # a prefill chunk of a wide model
        "norm_prefill": _norm(8192, 4096, "fp16"),
        # a training step's micro-batch
        "norm_train": _norm(16384, train=True),
        # full-precision training of a small model, without a bias
        "norm_train_odd": _norm(2001, 1000, "fp32", bias=False, train=True),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def _log(rng, lo, hi, step=1):
    """An integer of [lo, hi], even over its logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng) -> dict:
    op = rng.choice(("int4", "int4", "route", "norm"))
    train = rng.random() < 0.5
    if op == "int4":
        group = rng.choice((32, 64, 128, 128))
        k = _log(rng, group, 8192, group)
        n = rng.choice((_log(rng, 64, 16384, 64), _log(rng, 40, 8192, 8)))
        most = max(1, (1 << 37) // (k * n))
        return _int4(_log(rng, 1, min(4096, most)), k, n, group,
                     rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.3)
    if op == "route":
        experts = rng.choice((8, 16, 60, 64, 128, 256, 512, rng.randint(3, 511)))
        return _route(_log(rng, 1, 32768), experts, rng.randint(1, min(10, experts)),
                      rng.choice(("fp32", "fp32", "bf16", "fp16")), rng.random() < 0.6,
                      rng.random() < 0.4, rng.random() < 0.3, train)
    hidden = rng.choice((_log(rng, 64, 8192, 8), _log(rng, 33, 4095), 2048))
    tokens = _log(rng, 1, max(1, min(16384, (1 << 25) // hidden)))
    return _norm(tokens, hidden, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.7,
                 train)


# ------------------------------------------------------------------------------ inputs
def _nibbles(rows, cols, mean, spread, gen):
    q = torch.randn(rows, cols, generator=gen, device="cuda")
    return q.mul_(spread).add_(mean).round_().clamp_(0, 15).to(torch.int32)


def _pack(values):
    """Eight neighbours of the first dimension into a word, the first in the lowest bits."""
    v = values.view(values.shape[0] // 8, 8, values.shape[1])
    word = v[:, 0].clone()
    for j in range(1, 8):
        word |= v[:, j] << (4 * j)
    return word


def _activations(rows, cols, dtype, gen):
    """Normal activations with a few channels much larger than the rest."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.005, 8.0, 1.0)
    return x.to(dtype)


def prepare(case: dict, seed: int):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
    state = {"case": case}
    T = case["tokens"]
    if case["op"] == "int4":
        K, N, G = case["in"], case["out"], case["group"]
        state["x"] = _activations(T, K, dtype, gen)
        state["qweight"] = _pack(_nibbles(K, N, 7.5, 2.5, gen))
        state["qzeros"] = _pack(_nibbles(N, K // G, 7.5, 1.0, gen)).T.contiguous()
        state["scales"] = ((0.5 + rand(K // G, N)) / (2.5 * math.sqrt(K))).half()
        state["bias"] = randn(N).to(dtype) if case["bias"] else None
        return state
    if case["op"] == "route":
        E = case["experts"]
        # some experts much more in use than others
        popular = -0.5 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
        logits = randn(T, E) + popular[torch.randperm(E, generator=gen, device="cuda")]
        if case["blocked"]:
            logits.masked_fill_(rand(T, E) < 0.25, -math.inf)
        state["logits"] = logits.to(dtype)
        state["mask"] = None
        if case["padded"]:  # sequences of 128 tokens, each with a padded end
            at = torch.arange(T, device="cuda")
            length = 1 + (rand(T // 128 + 1) * 128).long()
            state["mask"] = at % 128 < length[at // 128]
        if case["train"]:
            state["logits"].requires_grad_()
            # a mean over the tokens; gradients of fp16 are scaled out of its subnormal range
            scale = 1024.0 if case["dtype"] == "fp16" else 1.0
            state["dweights"] = randn(T, case["top_k"]) * (scale / T)
            state["dbalance"] = torch.full((), scale * BALANCE_COEF, device="cuda")
            state["dz"] = torch.full((), scale * Z_COEF, device="cuda")
        return state
    H = case["hidden"]
    state["x"] = (_activations(T, H, torch.float32, gen) + 0.5 * randn(T, 1)).to(dtype)
    state["weight"] = (1.0 + 0.1 * randn(H)).to(dtype)
    state["bias"] = (0.1 * randn(H)).to(dtype) if case["bias"] else None
    if case["train"]:
        state["dy"] = randn(T, H).to(dtype)
        for name in ("x", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------------------ the framework's
def _run_own(s):
    from mtp_amd import ops

    case = s["case"]
    if case["op"] == "int4":
        return ops.int4_linear(s["x"], s["qweight"], s["qzeros"], s["scales"],
                               group_size=case["group"], bias=s["bias"])
    if case["op"] == "route":
        r = ops.route_tokens(s["logits"], case["top_k"], mask=s["mask"], renormalize=case["renorm"])
        res = {"ids": r.topk_ids, "weights": r.topk_weights, "counts": r.counts,
               "balance": r.balance_loss, "z": r.z_loss}
        if case["train"]:
            res["dlogits"], = torch.autograd.grad(
                (r.topk_weights, r.balance_loss, r.z_loss), (s["logits"],),
                (s["dweights"], s["dbalance"], s["dz"]))
        return res
    y = ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    res = {"y": y}
    if case["train"]:
        names = [n for n in ("x", "weight", "bias") if s[n] is not None]
        got = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        res.update({"d" + n: g for n, g in zip(names, got)})
    return res


# ------------------------------------------------------------------------------ plain forms
def _plain_run_int4(s):
    case, x = s["case"], s["x"]
    K, N, G = case["in"], case["out"], case["group"]
    shift = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    q = (s["qweight"][:, None, :] >> shift[:, None]) & 15
    z = (s["qzeros"][:, :, None] >> shift) & 15
    w = (q.view(K // G, G, N) - z.view(K // G, 1, N)).float() * s["scales"].float()[:, None, :]
    y = x.float() @ w.view(K, N)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def _plain_run_route(s):
    case, dtype = s["case"], s["logits"].dtype
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    l = s["logits"].detach().float()
    top, ids = torch.sort(l, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    live = top[:, :1] > -math.inf
    if s["mask"] is not None:
        live = live & s["mask"][:, None]
    chosen = live & (top > -math.inf)
    peak = torch.where(live, top[:, :1], 0.0)
    ex = torch.where(live, torch.exp(l - peak), 0.0)
    total = torch.where(live, ex.sum(dim=1, keepdim=True), 1.0)
    p = ex / total
    lse = torch.where(live, peak + torch.log(total), 0.0)
    picked = torch.where(chosen, torch.exp(top - peak), 0.0)
    over = picked.sum(dim=1, keepdim=True) if case["renorm"] else total
    weights = picked / torch.where(live, over, 1.0)
    n = live.sum()
    inv_n = torch.where(n > 0, 1.0 / n.clamp(min=1), 0.0)
    ids = torch.where(chosen, ids, -1)
    counts = (torch.arange(E, device=l.device)[:, None] == ids.reshape(1, -1)).sum(dim=1)
    share = counts.float() * (inv_n / k)
    balance = E * (share * (p.sum(dim=0) * inv_n)).sum()
    z = (lse * lse).sum() * inv_n
    res = {"ids": ids.to(torch.int32), "weights": weights, "counts": counts.to(torch.int32),
           "balance": balance, "z": z}
    if case["train"]:
        dw = s["dweights"]
        dot = (weights * dw).sum(dim=1, keepdim=True)
        if case["renorm"]:
            d = torch.zeros_like(l)
        else:
            d = -p * dot
        d = d.scatter_add(1, ids.clamp(min=0), weights * (dw - dot if case["renorm"] else dw))
        mean_share = (p * share).sum(dim=1, keepdim=True)
        d = d + (s["dbalance"] * E * inv_n) * p * (share - mean_share)
        d = d + (2.0 * s["dz"] * inv_n) * lse * p
        res["dlogits"] = d.to(dtype)
    return res


def _plain_run_norm(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    centred = x - x.mean(dim=1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    h = centred * r
    y = h * w
    if s["bias"] is not None:
        y = y + s["bias"].detach().float()
    res = {"y": y.to(dtype)}
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - g.mean(dim=1, keepdim=True) - h * (g * h).mean(dim=1, keepdim=True))
        res["dx"] = dx.to(dtype)
        res["dweight"] = (dy * h).sum(dim=0).to(dtype)
        if s["bias"] is not None:
            res["dbias"] = dy.sum(dim=0).to(dtype)
    return res


def run(state):
    if own:
        return _run_own(state)
    return {"int4": _plain_run_int4, "route": _plain_run_route,
            "norm": _plain_run_norm}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------ work
def work(case: dict) -> dict:
    T, es = case["tokens"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "int4":
        K, N, G = case["in"], case["out"], case["group"]
        weights = K * N // 2 + (K // G) * (N // 2 + 2 * N)
        return {"bytes": weights + (T * K + T * N) * es + (N * es if case["bias"] else 0),
                "flops": 2 * T * K * N}
    if case["op"] == "route":
        E, k = case["experts"], case["top_k"]
        # logits; ids, weights and counts; the mask; with a gradient the weights' and the logits'
        b = T * E * es + 8 * T * k + 4 * E + (T if case["padded"] else 0)
        f = 6 * T * E
        if case["train"]:
            b += 4 * T * k + T * E * es
            f += 8 * T * E
        return {"bytes": b, "flops": f}
    H = case["hidden"]
    small = (2 if case["bias"] else 1) * (2 if case["train"] else 1)
    return {"bytes": ((4 if case["train"] else 2) * T + small) * H * es,
            "flops": (22 if case["train"] else 8) * T * H}


# ------------------------------------------------------------------------------ 64 bits
def _exact_int4(case, s):
    K, N, G = case["in"], case["out"], case["group"]
    y = torch.zeros(case["tokens"], N, dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for g in range(K // G):
        zero = torch.empty(N, dtype=torch.float64, device="cuda")
        for j in range(8):
            zero[j::8] = ((s["qzeros"][g] >> (4 * j)) & 15).double()
        step = s["scales"][g].double()
        for j in range(8):  # every eighth row of the group
            rows = (s["qweight"][g * G // 8:(g + 1) * G // 8] >> (4 * j)) & 15
            y += x[:, g * G + j:(g + 1) * G:8] @ ((rows.double() - zero) * step)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_route(case, s):
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    l = s["logits"].detach().double()
    mask = torch.ones(T, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    alive = mask & torch.isfinite(l).any(dim=1)
    n = int(alive.sum())
    # ranks by counting: how many experts come before e
    ids = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(E, device="cuda")
    for lo in range(0, T, 256):
        part = l[lo:lo + 256]
        ahead = part[:, None, :] > part[:, :, None]
        ahead |= (part[:, None, :] == part[:, :, None]) & (at[None, :] < at[:, None])
        rank = ahead.sum(dim=2)
        take = (rank < k) & torch.isfinite(part) & alive[lo:lo + 256, None]
        t, e = take.nonzero(as_tuple=True)
        ids[lo + t, rank[t, e]] = e.to(torch.int32)
    chosen = ids >= 0
    p = torch.zeros_like(l)
    p[alive] = torch.softmax(l[alive], dim=1)
    lse = torch.zeros(T, dtype=torch.float64, device="cuda")
    lse[alive] = torch.logsumexp(l[alive], dim=1)
    weights = torch.where(chosen, p.gather(1, ids.clamp(min=0).long()), 0.0)
    if case["renorm"]:
        weights = torch.where(chosen, weights / weights.sum(dim=1, keepdim=True), 0.0)
    counts = torch.bincount(ids[chosen].long(), minlength=E)
    share = counts.double() / max(1, n * k)
    balance = E * torch.dot(share, p.sum(dim=0)) / max(1, n)
    res = {"ids": ids, "weights": weights, "counts": counts.to(torch.int32), "balance": balance,
           "z": lse.square().sum() / max(1, n)}
    if case["train"]:
        # the gradient with respect to p, through the softmax; the z loss has it directly
        dw = torch.where(chosen, s["dweights"].double(), 0.0)
        if case["renorm"]:
            total = torch.where(chosen, p.gather(1, ids.clamp(min=0).long()), 0.0).sum(1, keepdim=True)
            dw = (dw - (dw * weights).sum(dim=1, keepdim=True)) / total
            dw = torch.where(chosen, dw, 0.0)
        dp = (float(s["dbalance"]) * E / max(1, n)) * share.expand(T, E).clone()
        dp.scatter_add_(1, ids.clamp(min=0).long(), dw)
        d = p * (dp - (p * dp).sum(dim=1, keepdim=True))
        d += (2.0 * float(s["dz"]) / max(1, n)) * lse[:, None] * p
        res["dlogits"] = d
    return res


def _exact_norm(case, s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    std = torch.sqrt(var + EPS)
    unit = (x - mean) / std
    res = {"y": unit * w if s["bias"] is None else unit * w + s["bias"].detach().double()}
    if case["train"]:
        dy = s["dy"].double()
        H = case["hidden"]
        g = dy * w
        res["dx"] = (H * g - g.sum(1, keepdim=True) - unit * (g * unit).sum(1, keepdim=True)) / (H * std)
        res["dweight"] = (dy * unit).sum(0)
        if s["bias"] is not None:
            res["dbias"] = dy.sum(0)
    return res


def exact(case: dict, seed: int):
    return {"int4": _exact_int4, "route": _exact_route,
            "norm": _exact_norm}[case["op"]](case, prepare(case, seed))
