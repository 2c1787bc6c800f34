"""The int4 linear layer at the ends of its range, and that its weights are not rounded.

At the ends scales lie between fp16's smallest and largest values (powers of two: the ratios between groups are exact), x
goes up to 2^64. u = 2^-24. Whatever the form, a product is rounded into a sum of magnitudes of at most 62 (bf16:
x (16 + q) and (16 + z) x) or 158 (fp16: 64) |x|, K of them at most, and a group's sum is scaled and added with
three roundings more: (K + 3 K / 32 + 16) u 158 sum_k s |x| bounds them all, rounded once to the type.

With scales of 11 bits and x of small integers in one group of at most 128 (k, q and z random) a group's sum is an
integer below 128 * 3 * 79 < 2^15 on the way and, checked, below 2^13 in the end: its product with the scale has
24 bits, exact in fp32, and the result is the formula's, rounded once: equality. Where that group is not the last
one, the form for many rows rounds it at each group's end: two roundings a group (u each).
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops
from tests.test_gpu_int4_linear import BF, FP, U, exact, make

pytestmark = pytest.mark.gpu

# T, K, N, G of every form: few rows in their tiles; x shared in four, two and one share of K; tiles of integers
# with groups of 128, 64 and 32
FORMS = [(1, 256, 72, 128), (7, 512, 520, 32), (20, 256, 4104, 64), (40, 256, 4104, 32), (100, 384, 5256, 128),
         (130, 256, 8200, 64), (300, 512, 8200, 128), (3000, 512, 1544, 128), (4400, 256, 4104, 64),
         (9000, 96, 1032, 32)]


def on(*ts):
    return tuple(t.cuda() for t in ts)


@pytest.mark.parametrize("T,K,N,G", FORMS)
def test_large_activations_and_all_scales(T, K, N, G):
    q, z, qw, qz, g = make(K, N, G, 21)
    x = (torch.randint(-4, 5, (T, K), generator=g) * 2.0 ** 62).to(BF)
    s = torch.exp2(torch.randint(-24, 16, (K // G, N), generator=g).float()).half()
    x, q, z, s, qw, qz = on(x, q, z, s, qw, qz)
    want = exact(x, q, z, s, G)
    size = x.double().abs().view(T, -1, G).sum(2) @ s.double()
    err = (ops.int4_linear(x, qw, qz, s, group_size=G).double() - want).abs()
    tol = 1.01 * (K + 3 * K / 32 + 16) * U * 158 * size + 2.0 ** -8 * want.abs()
    assert bool((err <= tol).all())


@pytest.mark.parametrize("T,K,N,G", FORMS)
@pytest.mark.parametrize("dtype,step", [(BF, 2.0 ** -133), (FP, 2.0 ** -24)])
def test_subnormal_activations(T, K, N, G, dtype, step):
    """x among its type's smallest numbers, a scale that lifts the result out of them: sums of small integers."""
    q, z, qw, qz, g = make(K, N, G, 22)
    k = torch.randint(-2, 3, (T, K), generator=g)
    x = (k * step).to(dtype)
    s = torch.full((K // G, N), 1024.0).half()
    x, q, z, s, qw, qz = on(x, q, z, s, qw, qz)
    want = exact(x, q, z, s, G)
    assert torch.equal(ops.int4_linear(x, qw, qz, s, group_size=G), want.float().to(dtype))


def odd_scales(K, N, G, g):
    """1 + j / 1024 with odd j: all of fp16's 11 bits, times 2^-8 .. 2^-2."""
    j = 2 * torch.randint(0, 512, (K // G, N), generator=g) + 1
    return ((1 + j / 1024) * torch.exp2(torch.randint(-8, -1, (K // G, N), generator=g).float())).half()


def one_group(T, K, N, G, dtype, at, seed):
    """x in group `at` alone, the formula's result, and what weights rounded to the type would give."""
    q, z, qw, qz, g = make(K, N, G, seed)
    s = odd_scales(K, N, G, g)
    x = torch.zeros(T, K)
    x[:, at * G:(at + 1) * G] = torch.randint(-3, 4, (T, G), generator=g).float()
    x, q, z, s, qw, qz = on(x.to(dtype), q, z, s, qw, qz)
    want = exact(x, q, z, s, G)
    k = slice(at * G, (at + 1) * G)
    assert float((x[:, k].double() @ (q[k] - z[at]).double()).abs().max()) < 2 ** 13
    w = ((q.view(-1, G, N) - z[:, None]).double() * s[:, None].double()).to(dtype).double().view(K, N)
    return x, qw, qz, s, want, x.double() @ w


UNROUNDED = FORMS + [(16, 128, 16392, 128), (64, 128, 4104, 128)]


@pytest.mark.parametrize("T,K,N,G", UNROUNDED)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_weights_are_not_rounded(T, K, N, G, dtype):
    x, qw, qz, s, want, rounded = one_group(T, K, N, G, dtype, K // G - 1, 23)
    want = want.float().to(dtype)
    assert int((rounded.float().to(dtype) != want).sum()) > want.numel() // 100  # rounded ones would show
    assert torch.equal(ops.int4_linear(x, qw, qz, s, group_size=G), want)


@pytest.mark.parametrize("T,K,N,G", FORMS)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_weights_of_the_first_group_are_not_rounded(T, K, N, G, dtype):
    x, qw, qz, s, want, _ = one_group(T, K, N, G, dtype, 0, 24)
    got = ops.int4_linear(x, qw, qz, s, group_size=G).double()
    slack = (2 * K / G + 2) * U * want.abs()
    assert bool(((got - want).abs() <= 1.01 * slack + torch.finfo(dtype).eps / 2 * want.abs()
                 + (2.0 ** -25 if dtype == FP else 0)).all())


def test_weights_are_not_rounded_off_a_boundary():
    """Tensors between two 16-byte boundaries."""
    def off(t):
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    for dtype in (BF, FP):
        x, qw, qz, s, want, _ = one_group(19, 256, 136, 64, dtype, 2, 25)
        got = ops.int4_linear(off(x), off(qw), off(qz), off(s), group_size=64)
        assert torch.equal(got, want.float().to(dtype))


@pytest.mark.parametrize("T,K,N,G", [(1, 2048, 512, 128), (13, 1056, 200, 32), (40, 512, 264, 64), (150, 2048, 328, 128),
                                     (100, 2048, 5448, 128), (200, 1088, 8200, 64), (700, 1024, 4104, 128)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_random_values_of_the_packed_forms(T, K, N, G, dtype):
    """Few and more rows: sums of at most 128 products of magnitude 31 (fp16: 79) |x|, as much again taken off, then
    a rounding of 15 |x| s for each of the K / 32 parts at most that are added up, and 8 for the shares of K:
    ((128 + 1) 62 + 15 (K / 32 + 8)) u sum_k s |x| in bf16, 158 for 62 in fp16."""
    q, z, qw, qz, g = make(K, N, G, 26)
    x = torch.randn(T, K, generator=g)
    x = (x * torch.where(torch.rand(K, generator=g) < 0.02, 20.0, 1.0)).to(dtype)
    s = (0.01 * (0.5 + torch.rand(K // G, N, generator=g))).half()
    x, q, z, s, qw, qz = on(x, q, z, s, qw, qz)
    want = exact(x, q, z, s, G)
    size = x.double().abs().view(T, -1, G).sum(2) @ s.double()
    err = (ops.int4_linear(x, qw, qz, s, group_size=G).double() - want).abs()
    eps = torch.finfo(dtype).eps
    sums = (129 * (62 if dtype == BF else 158) + 15 * (K / 32 + 8)) * U * size
    assert bool((err <= (1 + eps) * sums + eps / 2 * want.abs() + 2.0 ** -25).all())
