"""Layer norm and its gradients against the formulas in 64 bits.

u = 2^-24 is fp32's half step. The mean is a sum in 64 bits. x - m = (x - m_hi) - m_lo is off by 2 u of
itself; a square of it by 4 u and its product's rounding, 8 of them in a tree of fp32 by 3 more, the rest in
64 bits: the variance by 8 u, r by 4 u and its rounding, so h by 2 + 5 + 1 = 8 u |h|, and y = fma(h, w, b) by
8 u |h w| + u |y|. The means of g and g h are fp32 sums over 8 columns a thread, 6 butterfly steps and up to 16 waves: 30
roundings and their division, 33 u of the mean of the magnitudes, and 9 u more where h stands in them.
Sums over tokens add a rounding a token. Each result is rounded once to its type.
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -148}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, slack, dtype):
    err = (got.detach().cpu().double() - want).abs()
    tol = slack * (1 + half(dtype)) + half(dtype) * want.abs() + TINY[dtype]
    assert bool((err <= tol).all()), float((err / tol).max())


def make(T, H, dtype, weight, bias, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + H)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"x": (r(T, H) + 0.5 * r(T, 1)).to(dtype), "weight": (1 + 0.2 * r(H)).to(dtype) if weight else None,
            "bias": (0.2 * r(H)).to(dtype) if bias else None, "dy": r(T, H).to(dtype)}


def formulas(s):
    """(y, its slack, gradients with their slacks) in 64 bits."""
    x, dy = s["x"].double(), s["dy"].double()
    T, H = x.shape
    w = s["weight"].double() if s["weight"] is not None else torch.ones(H, dtype=torch.float64)
    b = s["bias"].double() if s["bias"] is not None else torch.zeros(H, dtype=torch.float64)
    d = x - x.mean(1, keepdim=True)
    r = (d.square().mean(1, keepdim=True) + EPS).rsqrt()
    h = d * r
    y = h * w + b
    g = dy * w
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    dx = r * (g - mean(g) - h * mean(g * h))
    slack = r * U * (8 * g.abs() + 40 * mean(g.abs()) + h.abs() * 56 * mean((g * h).abs()))
    return y, U * (8 * (h * w).abs() + y.abs()), {
        "x": (dx, slack),
        "weight": ((dy * h).sum(0), (T + 44) * U * (dy * h).abs().sum(0)),
        "bias": (dy.sum(0), (T + 40) * U * dy.abs().sum(0))}


CASES = [  # T, H, dtype, weight, bias
    (1, 1, torch.float32, True, True), (1, 2048, torch.bfloat16, True, True),
    (3, 7, torch.float16, True, False), (13, 512, torch.bfloat16, True, True),
    (9, 513, torch.float32, False, True), (5, 2048, torch.float16, False, False),
    (6, 2056, torch.bfloat16, True, True), (7, 1000, torch.float32, True, False),
    (2, 8192, torch.bfloat16, True, True), (3, 8191, torch.float16, True, True),
    (2, 8192, torch.float32, True, True), (70, 64, torch.bfloat16, True, True),
    (1700, 96, torch.float32, True, True), (2500, 33, torch.bfloat16, True, True),
    (4, 4096, torch.bfloat16, True, False), (1601, 2048, torch.bfloat16, True, True),
    (1100, 4100, torch.float16, True, True)]
CASES += [  # several rows a wave: 8, 4 and 2 of them, the last ones behind the tensor
    (1, 8, torch.bfloat16, True, True), (770, 24, torch.bfloat16, True, True), (9, 64, torch.float32, True, True),
    (50001, 16, torch.bfloat16, True, True), (67, 128, torch.float16, True, False), (50, 65, torch.float32, True, True),
    (26003, 100, torch.float16, False, True), (13, 256, torch.bfloat16, True, True), (1001, 200, torch.float32, True, True),
    (12511, 250, torch.bfloat16, True, True), (3, 129, torch.bfloat16, True, True), (2, 257, torch.float32, True, True)]


@pytest.mark.parametrize("T,H,dtype,weight,bias", CASES)
def test_forward_and_gradients(T, H, dtype, weight, bias):
    s = make(T, H, dtype, weight, bias)
    y, slack, want = formulas(s)
    dev = {n: None if s[n] is None else s[n].cuda().requires_grad_() for n in ("x", "weight", "bias")}
    got = ops.layer_norm(dev["x"], dev["weight"], dev["bias"], eps=EPS)
    near(got, y, slack, dtype)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(dev["x"], dev["weight"], dev["bias"], eps=EPS), got)
    names = [n for n, t in dev.items() if t is not None]
    grads = torch.autograd.grad(got, [dev[n] for n in names], s["dy"].cuda())
    for n, g in zip(names, grads):
        near(g, *want[n], dtype)


@pytest.mark.parametrize("wanted", ["x", "weight", "bias"])
def test_one_gradient_alone(wanted):
    s = make(37, 260, torch.float32, True, True)
    dev = {n: s[n].cuda() for n in ("x", "weight", "bias")}
    dev[wanted].requires_grad_()
    ops.layer_norm(dev["x"], dev["weight"], dev["bias"], eps=EPS).backward(s["dy"].cuda())
    near(dev[wanted].grad, *formulas(s)[2][wanted], torch.float32)


@pytest.mark.parametrize("mean,spread,H", [(1e4, 1.0, 2048), (-300.0, 1e-3, 1000), (0.0, 1e-20, 640),
                                           (3e18, 1e15, 96), (2.0 ** 20, 1.0, 8192)])
def test_rows_far_from_zero(mean, spread, H):
    """The variance of rows whose mean is up to 10^6 times their spread, and of very small and large
    ones: moments of fp32 sums of the raw values would have no digit left. The slack is the values' own."""
    g = torch.Generator().manual_seed(3)
    x = (mean + spread * torch.randn(4, H, generator=g)).float()
    x[1, 0] = mean + 1000 * spread  # the value that the sums are taken from is an outlier
    d = x.double() - x.double().mean(1, keepdim=True)
    want = d * (d.square().mean(1, keepdim=True) + EPS).rsqrt()
    near(ops.layer_norm(x.cuda(), eps=EPS), want, 9 * U * want.abs(), torch.float32)


def test_constant_rows():
    x = torch.tensor([[3.0], [-7.5], [0.0], [1e30]]).expand(4, 600).contiguous()
    x = x.cuda().requires_grad_()
    y = ops.layer_norm(x, bias=torch.full((600,), 0.5, device="cuda"))
    assert torch.equal(y, torch.full_like(y, 0.5))
    dy = torch.randn(4, 600, generator=torch.Generator().manual_seed(1))
    dx, = torch.autograd.grad(y, x, dy.cuda())
    want = (dy.double() - dy.double().mean(1, keepdim=True)) * EPS ** -0.5
    near(dx, want, EPS ** -0.5 * U * (4 * dy.abs() + 36 * dy.abs().mean(1, keepdim=True)).double(),
         torch.float32)


def test_rows_with_infinities_and_nan_are_nan_alone():
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(2)).cuda()
    clean = ops.layer_norm(x)
    bad = x.clone()
    bad[1, 7], bad[3, 0], bad[4, 299] = float("inf"), float("nan"), float("-inf")
    y = ops.layer_norm(bad)
    assert bool(y[[1, 3, 4]].isnan().all()) and torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])


@pytest.mark.parametrize("H", [40, 64, 101, 128, 200, 256])
def test_rows_of_one_wave_do_not_touch_each_other(H):
    x = torch.randn(11, H, generator=torch.Generator().manual_seed(4)).cuda()
    dy = torch.randn(11, H, generator=torch.Generator().manual_seed(5)).cuda()
    rows = [[], []]
    for i, x in enumerate((x, x.clone())):
        if i:
            x[2, 3], x[10, H - 1] = float("nan"), float("inf")
        x.requires_grad_()
        y = ops.layer_norm(x)
        rows[i] = [y.detach(), *torch.autograd.grad(y, x, dy)]
    keep = [t for t in range(11) if t not in (2, 10)]
    for clean, got in zip(*rows):
        assert torch.equal(clean[keep], got[keep]) and bool(got[[2, 10]].isnan().all())


def test_no_tokens():
    x = torch.empty(0, 96, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = (torch.ones(96, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 96) and not dw.any() and not db.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unaligned_rows_give_the_same(dtype):
    """Tensors that start between two 16-byte boundaries take the element-wise loads."""
    s = make(40, 520, dtype, True, True)

    def off(t):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        v = flat[1:].view(t.shape)
        return v.copy_(t).requires_grad_()

    y, slack, want = formulas(s)
    x, w, b = off(s["x"]), off(s["weight"]), off(s["bias"])
    got = ops.layer_norm(x, w, b, eps=EPS)
    near(got, y, slack, dtype)
    for n, g in zip(("x", "weight", "bias"), torch.autograd.grad(got, (x, w, b), off(s["dy"]).detach())):
        near(g, *want[n], dtype)


def test_gradients_against_differences():
    """Central differences of a smooth scalar in fp32: values of about 30 over a step of 2^-5: rounding
    below 30 * 2^-22 * 2^5, third-order truncation of about step^2."""
    s = make(3, 24, torch.float32, True, True, 5)
    dev = {n: s[n].cuda().requires_grad_() for n in ("x", "weight", "bias")}
    v = s["dy"].cuda()

    def value(**kw):
        at = {**dev, **kw}
        return (ops.layer_norm(at["x"], at["weight"], at["bias"], eps=EPS).double() * v.double()).sum()

    grads = torch.autograd.grad(value(), list(dev.values()))
    for (name, t), g in zip(dev.items(), grads):
        for i in range(0, t.numel(), 5):
            step = torch.zeros_like(t).flatten()
            step[i] = 2.0 ** -5
            step = step.view(t.shape)
            with torch.no_grad():
                diff = (value(**{name: t + step}) - value(**{name: t - step})) / 2.0 ** -4
            assert abs(float(diff) - float(g.flatten()[i])) < 30 * 2.0 ** -17 + 0.02, (name, i)


def test_captured_step_on_another_stream():
    """A training step captured with leaves of its own and replayed on changing inputs."""
    s = make(300, 2048, torch.bfloat16, True, True)
    dev = {n: s[n].cuda().requires_grad_() for n in ("x", "weight", "bias")}
    dy = s["dy"].cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(ops.layer_norm(*dev.values(), eps=EPS), list(dev.values()), dy)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = ops.layer_norm(*dev.values(), eps=EPS)
        grads = torch.autograd.grad(y, list(dev.values()), dy)
    for seed in (1, 2, 3):
        n = make(300, 2048, torch.bfloat16, True, True, seed)
        with torch.no_grad():
            for k, t in dev.items():
                t.copy_(n[k])
            dy.copy_(n["dy"])
        graph.replay()
        torch.cuda.synchronize()
        want_y, slack, want = formulas(n)
        near(y, want_y, slack, torch.bfloat16)
        for k, g in zip(dev, grads):
            near(g, *want[k], torch.bfloat16)
