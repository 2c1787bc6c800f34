"""Routing with its losses (route_tokens) and the logits' gradient against the formulas in 64 bits.

u = 2^-24 is fp32's half step. exp(l - top) is off by 3 u of itself for the function and |l - top| u for
the difference it is taken of, at most 16 u for logits within 16 of the largest; a token's sum of them adds
at most 36 roundings (32 registers, 4 exchanges). A weight is the quotient of such a term and such a sum: at
most 19 + 19 + 36 + 1 u of itself, 100 u taken; lse is off by 55 u absolutely plus u |lse|. Sums over
tokens: a rounding for each of a wave's tokens and of the workgroup's 16 waves, the rest in 64 bits. Ids and
counts are exact.
"""

from __future__ import annotations

import math

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -148}
INF = math.inf


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(T, E, dtype, blocked=0.0, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * T + E)
    l = (2.0 * torch.randn(T, E, generator=g)).to(dtype)
    return l.masked_fill(torch.rand(T, E, generator=g) < blocked, -INF) if blocked else l


def formulas(l, k, mask=None, renorm=True, grads=None):
    """A token at a time from the definition, in 64 bits; with grads (dw, db, dz) also the gradient and
    the sum of the magnitudes it is made of."""
    T, E = l.shape
    x = l.double()
    ids = torch.full((T, k), -1, dtype=torch.int32)
    w, p = torch.zeros(T, k, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
    lse, counts = torch.zeros(T, dtype=torch.float64), torch.zeros(E, dtype=torch.int32)
    live = torch.zeros(T, dtype=torch.bool)
    for t in range(T):
        if (mask is not None and not mask[t]) or not bool((x[t] > -INF).any()):
            continue
        live[t] = True
        p[t], lse[t] = torch.softmax(x[t], 0), torch.logsumexp(x[t], 0)
        best = sorted((e for e in range(E) if x[t, e] > -INF), key=lambda e: (-x[t, e].item(), e))[:k]
        for i, e in enumerate(best):
            ids[t, i], w[t, i] = e, p[t, e]
            counts[e] += 1
        if renorm:
            w[t] /= w[t].sum()
    n = int(live.sum())
    share = counts.double() / max(1, n * k)
    out = {"ids": ids, "w": w, "counts": counts, "balance": E * (share * p.sum(0)).sum() / max(1, n),
           "z": lse.square().sum() / max(1, n), "n": n, "lse": lse}
    if grads is not None:
        dw, db, dz = (None if v is None else v.double() for v in grads)
        d, size = torch.zeros(T, E, dtype=torch.float64), torch.zeros(T, E, dtype=torch.float64)
        cb = 0.0 if db is None else float(db) * E / max(1, n)
        cz = 0.0 if dz is None else 2 * float(dz) / max(1, n)
        for t in range(T):
            if not live[t]:
                continue
            pf = (p[t] * share).sum()
            d[t] = p[t] * (cb * (share - pf) + cz * lse[t])
            size[t] = p[t] * (abs(cb) * (share + pf) + abs(cz) * (1 + lse[t].abs()))
            if dw is not None:
                sel = ids[t] >= 0
                e, wt, g = ids[t][sel].long(), w[t][sel], dw[t][sel]
                dot, mag = (wt * g).sum(), (wt * g).abs().sum()
                if renorm:
                    d[t, e] += wt * (g - dot)
                    size[t, e] += wt * (g.abs() + mag)
                else:
                    d[t] -= p[t] * dot
                    size[t] += p[t] * mag
                    d[t, e] += wt * g
                    size[t, e] += wt * g.abs()
        out["d"], out["size"] = d, size
    return out


def check(got, want, T):
    assert torch.equal(got.topk_ids.cpu(), want["ids"]) and torch.equal(got.counts.cpu(), want["counts"])
    err = (got.topk_weights.detach().cpu().double() - want["w"]).abs()
    assert bool((err <= 100 * U * want["w"] + 2.0 ** -148).all()), float((err / want["w"]).max() / U)
    sums = T / 4096 + 18
    assert abs(float(got.balance_loss.detach()) - want["balance"]) <= (110 + sums) * U * want["balance"]
    scale = (want["lse"].square() + 100 * want["lse"].abs() + 50).sum() / max(1, want["n"])
    assert abs(float(got.z_loss.detach()) - want["z"]) <= (sums + 4) * U * want["z"] + U * scale


CASES = [  # T, E, k, dtype, masked, blocked, renormalised
    (1, 1, 1, torch.float32, False, 0.0, True), (1, 256, 8, torch.float32, False, 0.0, True),
    (8, 256, 8, torch.bfloat16, False, 0.0, True), (3, 7, 7, torch.float16, False, 0.5, False),
    (16, 64, 6, torch.float32, True, 0.0, False), (17, 60, 5, torch.float16, True, 0.3, True),
    (33, 512, 10, torch.bfloat16, False, 0.0, True), (70, 65, 3, torch.float32, True, 0.9, True),
    (300, 128, 8, torch.float32, True, 0.2, False), (65, 511, 64, torch.float32, False, 0.0, True),
    (900, 16, 2, torch.bfloat16, True, 0.97, True), (5000, 8, 2, torch.float32, True, 0.1, True),
    (129, 129, 1, torch.float16, False, 0.0, True),
    (40, 300, 17, torch.bfloat16, True, 0.3, False), (40, 300, 16, torch.bfloat16, True, 0.3, False),
    (2100, 64, 8, torch.float16, False, 0.0, True), (31, 512, 16, torch.float32, True, 0.95, True),
    (1100, 300, 16, torch.bfloat16, True, 0.3, False), (1030, 512, 10, torch.float16, True, 0.97, True),
    (1027, 7, 7, torch.bfloat16, False, 0.5, True), (1501, 60, 5, torch.float16, True, 0.25, False),
    (1024, 130, 1, torch.bfloat16, True, 0.0, True),
    (1025, 8, 2, torch.float32, True, 0.0, True), (1100, 64, 16, torch.float32, True, 0.6, False),
    (1030, 200, 10, torch.float32, False, 0.0, True), (1026, 256, 8, torch.float32, True, 0.97, True),
    (1090, 7, 7, torch.float32, False, 0.5, True), (1040, 300, 8, torch.float32, False, 0.0, True)]


@pytest.mark.parametrize("T,E,k,dtype,masked,blocked,renorm", CASES)
def test_forward_and_gradient(T, E, k, dtype, masked, blocked, renorm):
    l = make(T, E, dtype, blocked)
    g = torch.Generator().manual_seed(11)
    mask = torch.rand(T, generator=g) < 0.7 if masked else None
    dw, db, dz = torch.randn(T, k, generator=g), torch.tensor(3.0), torch.tensor(-0.5)
    want = formulas(l, k, mask, renorm, (dw, db, dz))
    x = l.cuda().requires_grad_()
    got = ops.route_tokens(x, k, mask=None if mask is None else mask.cuda(), renormalize=renorm)
    check(got, want, T)
    d, = torch.autograd.grad((got.topk_weights, got.balance_loss, got.z_loss), x,
                             (dw.cuda(), db.cuda(), dz.cuda()))
    err = (d.cpu().double() - want["d"]).abs()
    tol = 160 * U * want["size"] + half(dtype) * want["d"].abs() + TINY[dtype]
    assert bool((err <= tol).all()), float((err / tol).max())
    with torch.no_grad():
        plain = ops.route_tokens(x, k, mask=None if mask is None else mask.cuda(), renormalize=renorm)
    for a, b in zip(got, plain):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,E,dtype", [(60, 96, torch.float32), (1100, 40, torch.float16)])
def test_gradient_of_large_logits(T, E, dtype):
    """Logits about a common value of 1000 (steps of half a unit, exact in both types): log sum exp has a
    half step of 512 u there, which neither the probabilities nor the gradient may be off by."""
    g = torch.Generator().manual_seed(21)
    l = (1000 + torch.randint(-12, 13, (T, E), generator=g) * 0.5).to(dtype)
    dw, db = torch.randn(T, 6, generator=g), torch.tensor(3.0)
    want = formulas(l, 6, None, False, (dw, db, None))
    x = l.cuda().requires_grad_()
    r = ops.route_tokens(x, 6, renormalize=False)
    d, = torch.autograd.grad((r.topk_weights, r.balance_loss), x, (dw.cuda(), db.cuda()))
    tol = 160 * U * want["size"] + half(dtype) * want["d"].abs() + TINY[dtype]
    err = (d.cpu().double() - want["d"]).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("parts", ["w", "b", "z", "wz"])
def test_gradient_of_some_results(parts):
    l = make(50, 40, torch.float32)
    g = torch.Generator().manual_seed(12)
    grads = (torch.randn(50, 4, generator=g) if "w" in parts else None,
             torch.tensor(2.0) if "b" in parts else None, torch.tensor(0.7) if "z" in parts else None)
    want = formulas(l, 4, grads=grads)
    x = l.cuda().requires_grad_()
    r = ops.route_tokens(x, 4)
    pick = [(o, v.cuda()) for o, v in zip((r.topk_weights, r.balance_loss, r.z_loss), grads) if v is not None]
    d, = torch.autograd.grad([o for o, _ in pick], x, [v for _, v in pick])
    tol = 160 * U * want["size"] + U * want["d"].abs() + TINY[torch.float32]
    assert bool(((d.cpu().double() - want["d"]).abs() <= tol).all())


@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_against_differences(renorm):
    """Central differences over a step of 2^-6 of a scalar of about 10: rounding 10 * 100 u * 2^6,
    truncation of about step^2 times its third derivative (below 10). Logits half a unit apart: no
    step reaches another selection."""
    g = torch.Generator().manual_seed(13)
    l = torch.stack([torch.randperm(12, generator=g) * 0.5 for _ in range(5)]).cuda().requires_grad_()
    v = torch.randn(5, 3, generator=g).double().cuda()

    def value(x):
        r = ops.route_tokens(x, 3, renormalize=renorm)
        return (r.topk_weights.double() * v).sum() + 2.0 * r.balance_loss + 0.1 * r.z_loss

    grad, = torch.autograd.grad(value(l), l)
    for i in range(l.numel()):
        step = torch.zeros(l.numel(), device="cuda")
        step[i] = 2.0 ** -6
        step = step.view(l.shape)
        with torch.no_grad():
            diff = (value(l + step) - value(l - step)) * 2.0 ** 5
        assert abs(float(diff) - float(grad.flatten()[i])) < 10 * 100 * U * 2 ** 6 + 10 * 2.0 ** -12, i


def test_ties_take_the_lower_id():
    l = torch.zeros(20, 300)
    l[:, 250], l[:, 7] = 1.0, -0.0
    r = ops.route_tokens(l.cuda(), 5)
    assert torch.equal(r.topk_ids.cpu(), torch.tensor([250, 0, 1, 2, 3], dtype=torch.int32).expand(20, 5))
    assert int(r.counts.sum()) == 100


@pytest.mark.parametrize("again", [1, 17])
@pytest.mark.parametrize("E,k", [(12, 3), (60, 8), (256, 16), (500, 10), (500, 20)])
def test_logits_closer_than_the_keys(E, k, again):
    """fp32 logits that agree in their upper bits, equal ones among them, next to ordinary tokens: the
    order is that of the values."""
    g = torch.Generator().manual_seed(E)
    l = torch.randn(64, E, generator=g)
    l[::2] = 3.0 + torch.randint(0, 40, (32, E), generator=g) * 2.0 ** -20
    l[1::8] = (2.0 * torch.randn(8, E, generator=g)).bfloat16().float()  # many equal values
    l[4::16, ::3] = -INF
    l[6::16] = -1e-30 * torch.randint(0, 9, (4, E), generator=g)
    l[8::16, E // 2:] = -INF
    l = l.repeat(again, 1)
    check(ops.route_tokens(l.cuda(), k), formulas(l, k), 64 * again)


def test_tokens_without_an_expert():
    """Rows of -inf, of the type's lowest value, and padding that holds NaN and infinities."""
    for dtype, more in ((torch.float32, 0), (torch.float32, 1100), (torch.bfloat16, 0), (torch.float16, 0), (torch.bfloat16, 1100),
                        (torch.float16, 2048)):
        low = torch.finfo(dtype).min
        l = make(6 + more, 32, dtype)
        l[0], l[1] = -INF, low
        l[2, :30] = -INF
        l[3], l[4, 5], l[4, 6] = float("nan"), INF, -INF
        mask = torch.tensor([True, True, True, False, False, True] + [False] * more)
        x = l.cuda().requires_grad_()
        r = ops.route_tokens(x, 4, mask=mask.cuda())
        ids, w = r.topk_ids.cpu(), r.topk_weights.detach().cpu()
        assert bool((ids[[0, 3, 4]] == -1).all()) and not w[[0, 3, 4]].any()
        assert ids[1].tolist() == [0, 1, 2, 3] and w[1].tolist() == [0.25] * 4  # all equal: even
        assert ids[2].tolist()[2:] == [-1, -1] and sorted(ids[2].tolist()[:2]) == [30, 31]
        assert abs(float(w[2].sum()) - 1) < 8 * U and int(r.counts.sum()) == 4 + 2 + 4
        dw = torch.full((6 + more, 4), float("nan"))
        dw[[1, 5]], dw[2, :2] = 1.0, 1.0  # what stands at places without an expert is not looked at
        d, = torch.autograd.grad((r.topk_weights, r.balance_loss), x,
                                 (dw.cuda(), torch.tensor(1.0, device="cuda")))
        assert bool(d.isfinite().all()) and not d[[0, 3, 4]].any()


@pytest.mark.parametrize("T,dtype", [(40, torch.float32), (40, torch.bfloat16), (1040, torch.float16),
                                     (1040, torch.float32)])
def test_a_counted_nan_shows(T, dtype):
    for bad in (float("nan"), INF):
        l = make(T, 24, dtype)
        l[7, 3] = bad
        x = l.cuda().requires_grad_()
        r = ops.route_tokens(x, 2)
        w = r.topk_weights.detach()
        assert bool(w[7].isnan().all()) and bool(w[[6, 8]].isfinite().all())
        assert bool(r.balance_loss.isnan()) and bool(r.z_loss.isnan())
        d, = torch.autograd.grad(r.topk_weights, x, torch.ones_like(w))
        assert bool(d[7].isnan().all()) and bool(d[[6, 8]].isfinite().all())
    l = torch.full((T, 24), float("nan"), dtype=dtype)
    r = ops.route_tokens(l.cuda(), 2)
    assert bool((r.topk_ids == -1).all()) and math.isnan(float(r.z_loss))


def test_no_tokens_and_none_that_count():
    for T in (0, 5, 500):
        x = torch.zeros(T, 48, device="cuda", requires_grad=True)
        r = ops.route_tokens(x, 2, mask=torch.zeros(T, dtype=torch.bool, device="cuda"))
        assert not r.counts.any() and float(r.balance_loss.detach()) == 0.0 and not bool(r.z_loss)
        d, = torch.autograd.grad((r.topk_weights, r.balance_loss, r.z_loss), x,
                                 (torch.ones(T, 2, device="cuda"),) + (torch.tensor(1.0, device="cuda"),) * 2)
        assert d.shape == (T, 48) and not d.any()


def test_same_bits_every_run_and_even_routing():
    l = make(20000, 64, torch.float32).cuda()
    first = ops.route_tokens(l, 4)
    for _ in range(3):
        for a, b in zip(first, ops.route_tokens(l, 4)):
            assert torch.equal(a, b)
    even = torch.zeros(64, 64)
    even[torch.arange(64), torch.arange(64)] = 1e-3
    assert abs(float(ops.route_tokens(even.cuda(), 1).balance_loss) - 1.0) < 200 * U


def test_unaligned_rows():
    l = make(30, 130, torch.bfloat16)
    flat = torch.empty(30 * 130 + 1, dtype=torch.bfloat16, device="cuda")
    x = flat[1:].view(30, 130).copy_(l)
    check(ops.route_tokens(x, 6), formulas(l, 6), 30)


def test_captured_steps_share_nothing():
    """Two captured training steps replayed in turn, with eager calls between."""
    graphs = []
    for T in (40, 700):
        x = torch.zeros(T, 96, device="cuda", requires_grad=True)
        dw, one = torch.ones(T, 4, device="cuda") / T, torch.ones((), device="cuda")
        dw[:, 0] = 2.0 / T

        def step(x=x, dw=dw, one=one):
            r = ops.route_tokens(x, 4)
            d, = torch.autograd.grad((r.topk_weights, r.balance_loss, r.z_loss), x, (dw, one, one))
            return r, d

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        graphs.append((T, x, dw, graph, out, one))  # a replay reads them: they stay alive
    for seed in range(3):
        for T, x, *_ in graphs:
            with torch.no_grad():
                x.copy_(make(T, 96, torch.float32, seed=seed))
        for *_, graph, _, _ in graphs:
            graph.replay()
        ops.route_tokens(make(333, 96, torch.float32).cuda(), 4)
        torch.cuda.synchronize()
        for T, x, dw, _, (r, d), _ in graphs:
            want = formulas(x.detach().cpu(), 4, grads=(dw.cpu(), torch.tensor(1.0), torch.tensor(1.0)))
            check(r, want, T)
            tol = 160 * U * want["size"] + U * want["d"].abs() + TINY[torch.float32]
            assert bool(((d.cpu().double() - want["d"]).abs() <= tol).all())


def test_a_router_in_training():
    """layer_norm -> router -> route_tokens -> dispatch -> experts -> combine with both losses, forward and
    backward, against 64-bit autograd on the host over the same selection. Everything is fp32: sums of up
    to 64 terms through five operators, gradients below 2^-10 of their largest."""
    T, H, E, k = 90, 64, 12, 3
    g = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    host = {"x": r(T, H), "nw": 1 + 0.1 * r(H), "nb": 0.1 * r(H), "router": r(H, E) / 8, "w": r(E, H, H) / 8}
    mask = torch.arange(T) % 9 != 8
    dout = r(T, H)
    dev = {n: t.cuda().requires_grad_() for n, t in host.items()}
    xn = ops.layer_norm(dev["x"], dev["nw"], dev["nb"])
    route = ops.route_tokens(xn @ dev["router"], k, mask=mask.cuda())
    d = ops.dispatch_tokens(xn, route.topk_ids, E)
    ends = d.offsets.tolist()
    rows = torch.cat([d.rows[a:b] @ dev["w"][e] for e, (a, b) in enumerate(zip(ends, ends[1:]))]
                     + [d.rows[ends[E]:]])
    out = ops.combine_tokens(rows, d.slot_row, route.topk_weights)
    total = (out * dout.cuda()).sum() + 0.5 * route.balance_loss + 0.1 * route.z_loss
    got = torch.autograd.grad(total, list(dev.values()))

    ref = {n: t.double().requires_grad_() for n, t in host.items()}
    xn = torch.nn.functional.layer_norm(ref["x"], (H,), ref["nw"], ref["nb"])
    logits = xn @ ref["router"]
    p = torch.softmax(logits, 1)
    ids = route.topk_ids.cpu().long()
    kept = mask[:, None].expand(T, k)
    assert torch.equal(ids >= 0, kept)
    assert torch.equal(ids[mask], torch.sort(logits[mask], dim=1, descending=True, stable=True)[1][:, :k])
    safe = ids.clamp(min=0)
    w = p.gather(1, safe) * kept
    w = w / torch.where(mask[:, None], w.sum(1, keepdim=True), 1.0)
    ref_out = (w[..., None] * (xn[:, None, None] @ ref["w"][safe])[:, :, 0]).sum(1)
    n = int(mask.sum())
    counts = torch.bincount(ids[kept], minlength=E)
    balance = E * (counts.double() / (n * k) * p[mask].mean(0)).sum()
    ref_total = ((ref_out * dout.double()).sum() + 0.5 * balance
                 + 0.1 * torch.logsumexp(logits[mask], 1).square().mean())
    assert torch.equal(route.counts.cpu().long(), counts)
    assert abs(float(total.detach()) - float(ref_total.detach())) < 2.0 ** -10 * float((ref_out.detach() * dout).abs().sum())
    for (name, _), a, b in zip(host.items(), got, torch.autograd.grad(ref_total, list(ref.values()))):
        assert float((a.cpu().double() - b).abs().max()) < 2.0 ** -10 * float(b.abs().max()), name
