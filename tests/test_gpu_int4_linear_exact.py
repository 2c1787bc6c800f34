"""The int4 linear layer at the ends of its range.

Scales lie between fp16's smallest and largest values (powers of two: the ratios between groups are exact), x
goes up to 2^64. u = 2^-24. Whatever the form, a product is rounded into a sum of magnitudes of at most 62 (bf16:
x (16 + q) and (16 + z) x) or 158 (fp16: 64) |x|, K of them at most, and a group's sum is scaled and added with
three roundings more: (K + 3 K / 32 + 16) u 158 sum_k s |x| bounds them all, rounded once to the type.
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
