"""Tensors whose elements or bytes pass 32 bits: the int4 linear layer, routing and layer norm at rows and
channels on both sides of the 32-bit boundaries, against the formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF = torch.bfloat16


def nibbles(words, rows, cols):
    """int32 [R, C] words of `rows` x `cols` (8 rows or 8 columns a word) as their nibbles, 64 bits."""
    v = torch.stack([(words >> (4 * j)) & 15 for j in range(8)])
    v = v.permute(1, 0, 2) if rows else v.permute(1, 2, 0)
    return v.reshape(words.shape[0] * (8 if rows else 1), words.shape[1] * (1 if rows else 8)).double()


@pytest.mark.parametrize("T,K,N", [(31, 64, 40_000_008), (300, 64, 9_000_008), (66_000, 64, 66_056),
                                   (66_000, 32, 66_056)])
def test_int4_linear(T, K, N):
    """Few, more and many rows (K = 64), and groups that end inside a step: integers and scales that are
    powers of two, exact in fp32."""
    g = torch.Generator(device="cuda").manual_seed(1)
    G = K
    qw = torch.randint(-2 ** 31, 2 ** 31 - 1, (K // 8, N), generator=g, device="cuda", dtype=torch.int32)
    qz = torch.randint(-2 ** 31, 2 ** 31 - 1, (1, N // 8), generator=g, device="cuda", dtype=torch.int32)
    s = torch.randint(1, 3, (1, N), generator=g, device="cuda").half() / 4
    x = torch.randint(-2, 3, (T, K), generator=g, device="cuda").to(BF)
    out = ops.int4_linear(x, qw, qz, s, group_size=G)
    assert out.numel() * 2 > 1 << 31
    flat = [0, (1 << 31) // N, (1 << 32) // N, (1 << 30) // N, T - 1]  # rows about the boundaries
    rows = torch.tensor(sorted({min(max(r + d, 0), T - 1) for r in flat for d in (-1, 0, 1)}))
    for c0 in (0, N // 16 * 8, N - 512):
        w = nibbles(qw[:, c0:c0 + 512].cpu(), True, False) - nibbles(qz[:, c0 // 8:c0 // 8 + 64].cpu(), False, True)
        want = (x[rows.cuda()].cpu().double() @ (w * s[:, c0:c0 + 512].cpu().double())).float().to(BF)
        assert torch.equal(out[rows.cuda(), c0:c0 + 512].cpu(), want)


@pytest.mark.parametrize("T", [3, 64, 130, 450])
@pytest.mark.parametrize("G", [32, 64, 128, 65536])
def test_int4_linear_of_the_longest_rows(T, G):
    """K = 65536 with from one group to 2048, a tenth of x in use: sums below 2^24 / 4."""
    K, N = 65536, 10_368
    g = torch.Generator(device="cuda").manual_seed(3)
    qw = torch.randint(-2 ** 31, 2 ** 31 - 1, (K // 8, N), generator=g, device="cuda", dtype=torch.int32)
    qz = torch.randint(-2 ** 31, 2 ** 31 - 1, (K // G, N // 8), generator=g, device="cuda", dtype=torch.int32)
    s = torch.randint(1, 3, (K // G, N), generator=g, device="cuda").half() / 4
    x = torch.randint(-1, 2, (T, K), generator=g, device="cuda").to(BF)
    x *= torch.rand(T, K, generator=g, device="cuda") < 0.1
    out = ops.int4_linear(x, qw, qz, s, group_size=G)
    for c0 in (0, N - 64):
        z = nibbles(qz[:, c0 // 8:c0 // 8 + 8].cpu(), False, True).repeat_interleave(G, 0)
        w = (nibbles(qw[:, c0:c0 + 64].cpu(), True, False) - z) * s[:, c0:c0 + 64].cpu().double().repeat_interleave(G, 0)
        assert torch.equal(out[:, c0:c0 + 64].cpu(), (x.cpu().double() @ w).float().to(BF))


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_route_tokens(dtype):
    """2^22 tokens of 512 experts, the most slots; each prefers its number modulo 512."""
    T, E = 1 << 22, 512
    l = torch.zeros(T, E, dtype=dtype, device="cuda")
    at = torch.arange(T, device="cuda") % E
    l.scatter_(1, at[:, None], 5.0)
    l.requires_grad_()
    r = ops.route_tokens(l, 1, renormalize=False)
    assert torch.equal(r.topk_ids[:, 0], at.int()) and bool((r.counts == T // E).all())
    p = torch.softmax(torch.tensor([5.0] + [0.0] * 511, dtype=torch.float64), 0)
    assert bool(((r.topk_weights.double() - p[0]).abs() <= 100 * U * p[0]).all())
    # T / 4096 + 18 roundings of a sum over tokens
    assert abs(float(r.balance_loss.detach()) - 1) <= (110 + T / 4096 + 18) * U
    dw = torch.ones(T, 1, device="cuda")
    d, = torch.autograd.grad(r.topk_weights, l, dw)
    half = torch.finfo(dtype).eps / 2
    # d = p_j (-p0) + [j chosen] p0: 160 u of the terms, and of bf16 half a step of the result itself (the
    # result p0 (1 - p0) = 0.174 is off by up to 2^-8 * 0.174 = 6.8e-4 then, more than 2^-8 p0^2 = 2.0e-4)
    for t in (0, (1 << 20) - 1, 1 << 20, (1 << 21) - 1, 1 << 21, T - 1):
        chosen = torch.arange(E) == t % E
        pt = torch.where(chosen, p[0], p[1])
        want = torch.where(chosen, p[0], 0.0) - pt * p[0]
        tol = 160 * U * (pt * p[0] + torch.where(chosen, p[0], 0.0)) + half * want.abs()
        assert bool(((d[t].cpu().double() - want).abs() <= tol).all())


def test_layer_norm():
    """4.4e9 elements; zeros but for the rows that are looked at."""
    T, H = 2_150_000, 2048
    rows = torch.tensor([0, (1 << 30) // H, (1 << 31) // H - 1, (1 << 31) // H, (1 << 32) // H - 1, (1 << 32) // H,
                         T - 1], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    some, dsome = (torch.randn(len(rows), H, generator=g, device="cuda").to(BF) for _ in range(2))
    x, dy = torch.zeros(T, H, dtype=BF, device="cuda"), torch.zeros(T, H, dtype=BF, device="cuda")
    x[rows], dy[rows] = some, dsome
    w = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(BF).requires_grad_()
    x.requires_grad_()
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xs = some.double().requires_grad_()
    ws = w.detach().double().requires_grad_()
    want = torch.nn.functional.layer_norm(xs, (H,), ws, None, 1e-5)
    want_dx, want_dw = torch.autograd.grad(want, (xs, ws), dsome.double())
    half = 2.0 ** -8
    want, size = want.detach(), dsome.double().abs() * w.detach().double().abs()
    assert bool(((y[rows].detach().double() - want).abs() <= (half + 16 * U) * want.abs() + 2.0 ** -126).all())
    # dx of a row: 64 u of the three terms it is made of
    r = xs.detach().var(1, unbiased=False).add(1e-5).rsqrt()[:, None]
    h = (xs.detach() - xs.detach().mean(1, keepdim=True)) * r
    terms = r * (size + size.mean(1, keepdim=True) + h.abs() * (size * h.abs()).mean(1, keepdim=True))
    assert bool(((dx[rows].double() - want_dx).abs() <= half * want_dx.abs() + 64 * U * terms).all())
    of_w = (dsome.double() * h).abs().sum(0)
    assert bool(((dw.double() - want_dw).abs() <= half * want_dw.abs() + 64 * U * of_w).all())
    assert not bool(dx[1:1000].any()) and not bool(y[T - 1000:T - 1].any())
