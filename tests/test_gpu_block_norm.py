"""The fused norms around a block (block_norm) and their gradients against the formulas in 64 bits.

u = 2^-24 is fp32's half step, h the type's. The sums run over 8 columns a thread, 6 butterfly steps
and up to 16 waves: 30 roundings, so a norm's factor is off by at most (30 / 2 + 3) u and a normed
value by 24 u; with the scales and the residual sum 32 u of the terms' magnitudes. Gradients: each of
the two reductions and the products around them, 64 u of the terms' magnitudes for du, 160 u behind
the second; sums over tokens add a rounding a token. Each result is rounded once to its type. x and
the gradients are checked against formulas of the residual stream that the kernel returned (itself
checked), as they are defined on the rounded stream.
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops, synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -148}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(T, H, dtype, post, gate, pre, seed=0):
    g = torch.Generator().manual_seed(seed + T + H)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    shape = {"none": None, "token": (T, 1), "channel": (H,), "full": (T, H)}[gate]
    return {"y": r(T, H), "res": r(T, H), "post_w": 0.1 * r(H) if post else None,
            "gate": None if shape is None else 0.5 + 0.3 * r(*shape),
            "pre_w": 0.1 * r(H) if pre else None}


def near(got, want, slack, dtype):
    err = (got.detach().cpu().double() - want).abs()
    tol = slack * (1 + half(dtype)) + half(dtype) * want.abs() + TINY[dtype]
    assert bool((err <= tol).all()), float((err / tol).max())


CASES = [  # T, H, dtype, post, gate, pre
    (1, 1, torch.float32, True, "full", True), (4, 2048, torch.bfloat16, True, "none", True),
    (3, 7, torch.float16, True, "channel", True), (13, 512, torch.bfloat16, True, "token", True),
    (9, 513, torch.float32, False, "full", True), (5, 2048, torch.float16, True, "full", False),
    (6, 2056, torch.bfloat16, False, "none", True), (7, 1000, torch.float32, True, "channel", True),
    (2, 8192, torch.bfloat16, True, "channel", True), (3, 8191, torch.float16, True, "token", True),
    (70, 64, torch.bfloat16, True, "channel", True), (1100, 96, torch.float32, True, "channel", True),
    (4, 4096, torch.bfloat16, False, "token", False), (2500, 33, torch.bfloat16, True, "full", True)]
A, B = 0.875, 1.25


@pytest.mark.parametrize("T,H,dtype,post,gate,pre", CASES)
def test_forward_and_gradients(T, H, dtype, post, gate, pre):
    s = make(T, H, dtype, post, gate, pre)
    dev = {n: None if t is None else t.cuda().requires_grad_() for n, t in s.items()}
    r, x = ops.block_norm(dev["y"], dev["res"], post_w=dev["post_w"], gate=dev["gate"],
                          pre_w=dev["pre_w"], res_scale=A, branch_scale=B, eps=EPS)
    assert (x is None) == (not pre)
    d = {n: None if t is None else t.double() for n, t in s.items()}
    gt = 1.0 if d["gate"] is None else d["gate"]
    y = d["y"]
    qy = (y.square().mean(1, keepdim=True) + EPS).rsqrt() if post else 1.0
    w1 = 1 + d["post_w"] if post else 1.0
    yh = y * qy
    p = yh * w1
    near(r, A * d["res"] + B * gt * p, 32 * U * (A * d["res"].abs() + (B * gt * p).abs()), dtype)
    st = r.detach().cpu().double()
    qr = (st.square().mean(1, keepdim=True) + EPS).rsqrt()
    w2 = 1 + d["pre_w"] if pre else 1.0
    if pre:
        near(x, st * qr * w2, 32 * U * (st * qr * w2).abs(), dtype)

    gen = torch.Generator().manual_seed(99)
    dr = torch.randn(T, H, generator=gen).to(dtype)
    dx = torch.randn(T, H, generator=gen).to(dtype)
    names = [n for n, t in dev.items() if t is not None]
    outs, gs = ((r, x), (dr.cuda(), dx.cuda())) if pre else ((r,), (dr.cuda(),))
    grads = dict(zip(names, torch.autograd.grad(outs, [dev[n] for n in names], gs)))
    du, size = dr.double(), dr.double().abs()
    if pre:
        g, rh = dx.double() * w2, st * qr
        du = du + qr * (g - rh * (g * rh).mean(1, keepdim=True))
        size = size + qr * (g.abs() + rh.abs() * (g * rh).abs().mean(1, keepdim=True))
        near(grads["pre_w"], (dx.double() * rh).sum(0),
             (T + 100) * U * (dx.double() * rh).abs().sum(0), dtype)
    near(grads["res"], A * du, 66 * U * A * size, dtype)
    db, dbs = B * du, B * size
    if gate != "none":
        dims = {"token": 1, "channel": 0, "full": None}[gate]
        full, fs = db * p, 128 * U * dbs * p.abs()
        if gate == "channel":
            full, fs = full.sum(0), fs.sum(0) + T * U * (dbs * p.abs()).sum(0)
        elif gate == "token":
            full = full.sum(1, keepdim=True)
            fs = fs.sum(1, keepdim=True) + 30 * U * (dbs * p.abs()).sum(1, keepdim=True)
        near(grads["gate"], full, fs, dtype)
        del dims
    dp, dps = db * gt, dbs * (gt.abs() if gate != "none" else 1.0)
    if post:
        near(grads["post_w"], (dp * yh).sum(0), (T + 200) * U * (dps * yh.abs()).sum(0), dtype)
        hh, hs = dp * w1, dps * w1.abs()
        dy = qy * (hh - yh * (hh * yh).mean(1, keepdim=True))
        dys = qy * (hs + yh.abs() * (hs * yh.abs()).mean(1, keepdim=True))
        near(grads["y"], dy, 160 * U * dys, dtype)
    else:
        near(grads["y"], dp, 70 * U * dps, dtype)


@pytest.mark.parametrize("gate", ["none", "token", "channel", "full"])
def test_gradients_against_differences(gate):
    """Central differences of a smooth scalar in fp32: rounding (values of about 30 over a step of
    2^-5) below 30 * 2^-22 * 2^5 and third-order truncation of about step^2 = 2^-10."""
    s = {n: None if t is None else t.cuda().requires_grad_()
         for n, t in make(3, 24, torch.float32, True, gate, True, 5).items()}
    g = torch.Generator().manual_seed(6)
    v1, v2 = torch.randn(3, 24, generator=g).cuda(), torch.randn(3, 24, generator=g).cuda()

    def value(d):
        r, x = ops.block_norm(d["y"], d["res"], post_w=d["post_w"], gate=d["gate"],
                              pre_w=d["pre_w"], res_scale=A, branch_scale=B)
        return (r * v1).double().sum() + (x * v2).double().sum()

    names = [n for n, t in s.items() if t is not None]
    grads = torch.autograd.grad(value(s), [s[n] for n in names])
    step = 2.0 ** -5
    with torch.no_grad():
        for n, grad in zip(names, grads):
            for i in range(0, s[n].numel(), 7):
                ends = []
                for sign in (1, -1):
                    t = s[n].clone()
                    t.view(-1)[i] += sign * step
                    ends.append(value({**s, n: t}))
                diff = float((ends[0] - ends[1]) / (2 * step))
                assert abs(diff - float(grad.view(-1)[i])) < 2.0 ** -7 * (1 + abs(diff)), (n, i)


def test_partial_gradients_and_unused_outputs():
    """Gradients of one input, of the stream alone (x unused) and of x alone, and expanded ones."""
    s = make(11, 264, torch.float32, True, "channel", True)
    dev = {n: t.cuda().requires_grad_() for n, t in s.items()}
    call = lambda d: ops.block_norm(d["y"], d["res"], post_w=d["post_w"], gate=d["gate"],  # noqa: E731
                                    pre_w=d["pre_w"])
    r, x = call(dev)
    gr, gx = torch.ones_like(r), torch.randn_like(r)
    names = list(dev)
    both = torch.autograd.grad((r, x), [dev[n] for n in names], (gr, gx), retain_graph=True)
    only_x = torch.autograd.grad(x, [dev[n] for n in names], gx, retain_graph=True)
    only_r = torch.autograd.grad(r.sum(), [dev[n] for n in names], allow_unused=True)
    zero = torch.zeros_like(r)
    r, x = call(dev)
    with_zero = torch.autograd.grad((r, x), [dev[n] for n in names], (zero, gx), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(only_x, with_zero))
    with_zero = torch.autograd.grad((r, x), [dev[n] for n in names], (gr, zero))
    for n, a, b in zip(names, only_r, with_zero):
        assert torch.equal(a, b), n
    for n, want in zip(names, both):
        one = {m: (t if m == n else t.detach()) for m, t in dev.items()}
        r, x = call(one)
        assert torch.equal(torch.autograd.grad((r, x), one[n], (gr, gx))[0], want)


def test_not_finite_rows_stay_in_their_rows():
    s = make(6, 40, torch.bfloat16, True, "token", True)
    s["y"][2, 3] = float("nan")
    s["gate"][4, 0] = float("inf")
    d = {n: t.cuda() for n, t in s.items()}
    r, x = ops.block_norm(d["y"], d["res"], post_w=d["post_w"], gate=d["gate"], pre_w=d["pre_w"])
    assert bool(torch.isnan(r[2]).all()) and bool(torch.isnan(x[2]).all())
    assert not bool(torch.isfinite(r[4]).any())
    ok = [0, 1, 3, 5]
    clean = {n: (t if t.dim() == 1 else t[ok].contiguous()) for n, t in d.items()}
    r2, x2 = ops.block_norm(clean["y"], clean["res"], post_w=clean["post_w"], gate=clean["gate"],
                            pre_w=clean["pre_w"])
    assert torch.equal(r[ok], r2) and torch.equal(x[ok], x2)


def test_no_tokens_unaligned_bases_and_graph():
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.zeros(64, device="cuda", requires_grad=True)
    r, x = ops.block_norm(e, e, post_w=w, gate=w, pre_w=w)
    assert r.shape == x.shape == (0, 64)
    (r.sum() + x.sum()).backward()
    assert float(w.grad.abs().sum()) == 0.0

    s = {n: t.cuda() for n, t in make(50, 64, torch.bfloat16, True, "full", True).items()}
    want = ops.block_norm(**s)
    off = {}
    for n, t in s.items():
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        off[n] = buf[1:].view(t.shape)
        off[n].copy_(t)
    # the narrow form adds its columns in another order: at most a step of the type apart
    for a, b in zip(ops.block_norm(**off), want):
        assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 1e-30).all())

    leaf = {n: t.clone().requires_grad_() for n, t in s.items()}
    gr = torch.randn(50, 64).to(torch.bfloat16).cuda()

    def step():
        r, x = ops.block_norm(**leaf)
        return (r.detach(), x.detach(), *torch.autograd.grad((r, x), list(leaf.values()), (gr, gr)))

    with torch.cuda.stream(torch.cuda.Stream()):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        with torch.no_grad():
            leaf["y"].add_(0.5 * i)
        graph.replay()
        torch.cuda.synchronize()
        held = [t.detach().clone() for t in static]
        assert all(torch.equal(a, b.detach()) for a, b in zip(held, step()))


def test_layer_step_of_the_operators():
    """A layer step as they are used together: block_norm -> router -> int8 experts -> block_norm, and
    the same with rows dispatched to the caller's own experts, trained: gradients reach every input
    and equal those of the plain composition in fp32 (a chain of six stages, each within 200 u of its
    terms; 2^-12 of the largest gradient leaves a factor of four)."""
    from mtp_amd.weights import Int8Experts

    T, H, E, I, k = 24, 128, 8, 64, 2
    g = torch.Generator().manual_seed(8)
    layer = synth.layer_to(synth.make_layer(2, num_experts=16, hidden=512, intermediate=256), "cuda")
    ex8 = Int8Experts.from_gptq(layer.experts)
    y0 = synth.make_tokens(T, 512, seed=1).cuda()
    res = synth.make_tokens(T, 512, seed=2).cuda()
    w = (0.1 * torch.randn(512, generator=g)).to(torch.bfloat16).cuda()
    r, x = ops.block_norm(y0, res, post_w=w, pre_w=w)
    ids, wt, _, _ = ops.router_topk(x, layer.router_w, 4)
    y = ops.int8_experts(x, ids, wt, ex8)
    r2, x2 = ops.block_norm(y, r, post_w=w, pre_w=w, branch_scale=0.5)
    assert bool(torch.isfinite(x2.float()).all()) and r2.shape == (T, 512)

    ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    ids[3, 1] = -1
    leaves = [torch.randn(*s, generator=g) for s in
              ((T, H), (T, H), (H,), (E, I, H), (E, H, I), (T, k))]
    v = torch.randn(T, H, generator=g)

    def ours(y, res, w, up, down, wt):
        r, x = ops.block_norm(y, res, post_w=w, pre_w=w)
        d = ops.dispatch_tokens(x, ids.cuda(), E)
        ends = d.offsets.tolist()
        parts = [torch.relu(d.rows[a:b] @ up[e].T) @ down[e].T
                 for e, (a, b) in enumerate(zip(ends, ends[1:]))] + [d.rows[ends[-1]:]]
        out = ops.combine_tokens(torch.cat(parts), d.slot_row, wt)
        return ops.block_norm(out, r, post_w=w, pre_w=w)[1]

    def plain(y, res, w, up, down, wt):
        n = lambda t: t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt() * (1 + w)  # noqa: E731
        r = res + n(y)
        x, out = n(r), torch.zeros_like(r)
        for t in range(T):
            for i in range(k):
                if ids[t, i] >= 0:
                    e = int(ids[t, i])
                    out[t] += wt[t, i] * (torch.relu(x[t] @ up[e].T) @ down[e].T)
        return n(r + n(out))

    mine = [t.cuda().requires_grad_() for t in leaves]
    ref = [t.double().requires_grad_() for t in leaves]
    got = torch.autograd.grad(ours(*mine), mine, v.cuda())
    want = torch.autograd.grad(plain(*ref), ref, v.double())
    for a, b in zip(got, want):
        assert float((a.cpu().double() - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max())


def test_tensors_beyond_4_gib():
    """Rows do not depend on each other: the last rows of tensors of more than 2^32 bytes (4.3 GB of
    bf16), and their gradients, are those of a call on these rows alone."""
    T, H, last = (1 << 21) + 5, 1032, 700
    gen = torch.Generator(device="cuda").manual_seed(5)
    y = torch.randn(T, H, generator=gen, dtype=torch.bfloat16, device="cuda").requires_grad_()
    assert y.numel() * 2 > 1 << 32
    w = (torch.randn(H, generator=gen, device="cuda") / 8).to(torch.bfloat16)

    def run(t):
        res, gate = t.detach() * 0.5, t.detach()[:, :1].contiguous()
        r, x = ops.block_norm(t, res, post_w=w, pre_w=w, gate=gate)
        return (r.detach(), x.detach(), *torch.autograd.grad((r, x), t, (res, res)))

    full = [t[-last:].clone() for t in run(y)]
    part = run(y.detach()[-last:].clone().requires_grad_())
    assert all(torch.equal(a, b) for a, b in zip(full, part))
