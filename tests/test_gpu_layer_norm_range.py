"""Layer norm of rows whose squares leave fp32's range, against the formulas in 64 bits, and the weights'
gradients of many rows, exactly.

Such a row is taken in units of a power of two, which rounds nothing, so the bounds are those of any row
(u = 2^-24): x - m off by 2 u of itself, r by 4 u, h by 8 u |h|, y by 8 u |h w| + u |y|; dx by
r u (8 |g| + 40 mean|g| + 56 |h| mean|g h|); the weights' gradients by a rounding for each token and 44 more.
Each result is rounded once to its type.
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = {torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -148}
# a width of each kernel: several rows a wave, a wave a row, a workgroup a row; element-wise loads
WIDTHS = [40, 100, 129, 200, 400, 1000, 2000, 2001, 4000, 4097, 8192]


def near(got, want, slack, dtype, what):
    half = torch.finfo(dtype).eps / 2
    err = (got.detach().cpu().double() - want).abs()
    tol = slack * (1 + half) + half * want.abs() + TINY[dtype]
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


def check(x, dy, eps, dtype):
    g = torch.Generator().manual_seed(x.shape[1])
    T, H = x.shape
    w, b = (1 + 0.2 * torch.randn(H, generator=g)).to(dtype), (0.2 * torch.randn(H, generator=g)).to(dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.cuda())
    x, dy, wd = x.double(), dy.double(), w.double()
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    d = x - mean(x)
    r = (mean(d.square()) + eps).rsqrt()
    h, gr = d * r, dy * wd
    want = h * wd + b.double()
    near(y, want, U * (8 * (h * wd).abs() + want.abs()), dtype, "y")
    near(dx, r * (gr - mean(gr) - h * mean(gr * h)),
         r * U * (8 * gr.abs() + 40 * mean(gr.abs()) + 56 * h.abs() * mean((gr * h).abs())), dtype, "dx")
    near(dw, (dy * h).sum(0), (T + 44) * U * (dy * h).abs().sum(0), dtype, "dw")
    near(db, dy.sum(0), (T + 40) * U * dy.abs().sum(0), dtype, "db")
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", WIDTHS)
def test_large_rows(H, dtype):
    """Deviations from 10^19 on, where fp32's squares overflow, up to the largest finite values of both
    signs (whose difference from the mean may itself pass fp32), between ordinary rows."""
    g = torch.Generator().manual_seed(H)
    x = torch.randn(12, H, generator=g)
    x[1] *= 1e20
    x[2] *= 3e19
    x[4] = 3.3e38 * (2 * torch.rand(H, generator=g) - 1)
    x[5] = 3e38
    x[5, :H // 8] = -3e38
    x[7] = 1e25 + 1e24 * x[7]
    x[8, 3] = 2e38
    x[11] *= 1e30
    y = check(x.to(dtype), torch.randn(12, H, generator=g).to(dtype), 1e-5, dtype)
    ordinary = torch.randn(12, H, generator=torch.Generator().manual_seed(H))
    at = [0, 3, 6, 9, 10]
    w = (1 + 0.2 * torch.randn(H, generator=torch.Generator().manual_seed(H))).to(dtype)
    clean = x.clone()
    clean[[1, 2, 4, 5, 7, 8, 11]] = ordinary[[1, 2, 4, 5, 7, 8, 11]]
    assert torch.equal(ops.layer_norm(clean.to(dtype).cuda(), w.cuda())[at],
                       ops.layer_norm(x.to(dtype).cuda(), w.cuda())[at])
    assert bool(y.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", WIDTHS)
def test_small_rows_without_eps(H, dtype):
    """With eps = 0 a row keeps its shape down to subnormal values, whose squares fp32 rounds to zero. The
    incoming gradient is as small as keeps dx finite."""
    g = torch.Generator().manual_seed(H + 1)
    x, dy = torch.randn(9, H, generator=g), torch.randn(9, H, generator=g)
    x[1] *= 1e-24
    x[2] = 1e-30 + 1e-31 * x[2]
    x[4] *= 1e-13
    x[5] *= 1e-40
    dy[5] *= 1e-10
    x[7] *= 1e-37
    dy[7] *= 1e-5
    check(x.to(dtype), dy.to(dtype), 0.0, dtype)


def test_constant_rows_and_a_tiny_eps():
    """var = 0 and eps far below the squares' range: the bias, whatever the rows' values."""
    for eps in (1e-30, 1e-40, 1e37, 3e38):
        x = torch.tensor([[3.0], [-7.5], [0.0], [1e30], [1e-30], [3e38]]).expand(6, 600).contiguous().cuda()
        y = ops.layer_norm(x, bias=torch.full((600,), 0.5, device="cuda"), eps=eps)
        assert torch.equal(y, torch.full_like(y, 0.5))


@pytest.mark.parametrize("H", [60, 1000, 5000])
def test_eps_that_outweighs_the_row(H):
    """An eps of 10^38: y = (x - m) 10^-19."""
    x = torch.randn(5, H, generator=torch.Generator().manual_seed(6))
    eps = float(torch.tensor(1e38))
    d = x.double() - x.double().mean(1, keepdim=True)
    want = d * (d.square().mean(1, keepdim=True) + eps).rsqrt()
    near(ops.layer_norm(x.cuda(), eps=eps), want, 9 * U * want.abs(), torch.float32, "y")


# Rows of +-1, as many of either: mean 0, variance 1, and with eps = 0 h = x exactly. With incoming gradients of
# small integers the weights' gradients are integers below 2^24, exact in fp32 in any order: equality, to the
# last row. T lies behind one, two and more passes of all workgroups (768 or 256 of 32, 16, 8, 4 or 1 rows), with ragged
# ends: a workgroup, a wave, a row more, a row less.
PASSES = [(8, 32), (64, 32), (66, 16), (100, 16), (128, 16), (130, 8), (256, 8), (258, 4), (512, 4), (514, 1), (2000, 1),
          (2050, 1), (8192, 1), (8190, 1)]


@pytest.mark.parametrize("H,rows", PASSES)
def test_every_row_counts_once_in_the_weights_gradients(H, rows):
    groups = 768 if H <= 2048 else 256
    for T in (rows, rows + 1, groups * rows - 1, groups * rows, groups * rows + 1, 2 * groups * rows - 1,
              2 * groups * rows + 3, (3 if H < 600 else 2) * groups * rows + rows // 2 + 1):
        g = torch.Generator(device="cuda").manual_seed(T + H)
        x = torch.ones(T, H, device="cuda")
        x[:, ::2] = -1.0
        x *= 1.0 - 2.0 * torch.randint(0, 2, (T, 1), generator=g, device="cuda")
        dy = torch.randint(1, 8, (T, H), generator=g, device="cuda").float()
        w, b = (torch.ones(H, device="cuda", requires_grad=True) for _ in range(2))
        y = ops.layer_norm(x, w, b, eps=0.0)
        assert torch.equal(y, x + 1.0)
        dw, db = torch.autograd.grad(y, (w, b), dy)
        assert torch.equal(db, dy.double().sum(0).float()), T
        assert torch.equal(dw, (dy.double() * x).sum(0).float()), T
        only, = torch.autograd.grad(ops.layer_norm(x, w, b, eps=0.0), (b,), dy)
        assert torch.equal(only, db)
