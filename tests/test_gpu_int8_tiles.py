"""int8 experts at each tile size that their plan gives, in the 16-bit types, with gates and scales that
differ by channel and expert; a shared expert as one more expert; and their place
in a graph of gradients."""

from __future__ import annotations

import pytest
import torch

from mtp_amd import ops
from mtp_amd.weights import Int8Experts
from tests.test_gpu_int8 import U, expected_experts, half, make_experts

pytestmark = pytest.mark.gpu


def tile_rows(T, k, E, H, I, dtype, workspace_bytes):
    """The rows of a tile, which the workspace's size tells: it holds 16 bytes for each tile there may
    be (slots / rows + one an expert), behind rows, scales and tables of sizes that do not depend on it."""
    def up(n):
        return -(-n // 256) * 256

    S, es, chunks = T * k, dtype.itemsize, -(-T * k // 1024)
    scratch = 0 if S <= 4096 else chunks * (E + 1) * 4 + chunks * 1024 * 2
    rest = sum(map(up, (T * H, T * 4, (E + 1) * 4, S * 4, S * 4, scratch, S * I * es, S * I, S * 4,
                        S * H * es)))
    fits = [bm for bm in (32, 64, 128, 256)
            if rest + up((S // bm + min(S, E)) * 16) == workspace_bytes]
    assert len(fits) == 1, (fits, workspace_bytes - rest)
    return fits[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,T,k,E,H,I", [
    (32, 400, 3, 40, 272, 208), (32, 300, 4, 150, 144, 80), (64, 900, 2, 7, 272, 1008),
    (64, 700, 6, 90, 144, 208), (128, 1024, 4, 64, 144, 528), (128, 1500, 3, 40, 336, 1552),
    (256, 1500, 3, 5, 272, 1008), (256, 2600, 2, 11, 528, 656)])
def test_experts_of_every_tile(rows, T, k, E, H, I, dtype):
    """Sampled tokens against 64 bits, within what expected_experts allows; and bit for bit against a
    call of their own, which has other tiles (of 32 rows) and neighbours."""
    gen = torch.Generator().manual_seed(T + I)
    x = torch.randn(T, H, generator=gen).to(dtype)
    # uneven: a third of the slots at one expert, another tenth dropped
    ids = torch.randint(0, E, (T, k), generator=gen, dtype=torch.int32)
    ids[torch.rand(T, k, generator=gen) < 0.3] = E - 2
    ids[torch.rand(T, k, generator=gen) < 0.1] = -1
    w = torch.rand(T, k, generator=gen)
    ex = make_experts(E, H, I, T)
    dev = ex.to("cuda")
    assert tile_rows(T, k, E, H, I, dtype, ops.int8_experts_workspace_bytes(T, k, dev, dtype)) == rows
    got = ops.int8_experts(x.cuda(), ids.cuda(), w.cuda(), dev).cpu()
    for n in (3, 41):  # tokens that sit at all places of the tiles
        some = torch.randperm(T, generator=gen)[:n]
        own = ops.int8_experts(x[some].cuda(), ids[some].cuda(), w[some].cuda(), dev).cpu()
        assert torch.equal(got[some], own)
    want, tol = expected_experts(x[some], ids[some], w[some], ex)
    err = (got[some].double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert float(got[(ids < 0).all(1)].abs().sum()) == 0.0


@pytest.mark.parametrize("T", [1, 50])
def test_shared_expert_as_one_more_expert(T):
    """A gated shared expert as one more expert of the stacks, its id and gate one more slot: what the
    routed experts and the shared one give apart, each rounded to the type (half a step of each), and
    k + 1 fp32 sums."""
    E, H, I, k, dtype = 24, 256, 96, 4, torch.bfloat16
    gen = torch.Generator().manual_seed(T)
    routed, shared = make_experts(E, H, I, 1).to("cuda"), make_experts(1, H, I, 2).to("cuda")
    both = Int8Experts(*(torch.cat([getattr(routed, n), getattr(shared, n)]) for n in (
        "gate", "gate_scale", "up", "up_scale", "down", "down_scale")))
    x = torch.randn(T, H, generator=gen).to(dtype).cuda()
    ids = torch.randint(0, E, (T, k), generator=gen, dtype=torch.int32).cuda()
    w = torch.rand(T, k, generator=gen).cuda()
    gate = torch.sigmoid(x.float() @ torch.randn(H, 1, generator=gen).cuda() / 16)
    out = ops.int8_experts(x, torch.cat([ids, torch.full_like(ids[:, :1], E)], 1),
                           torch.cat([w, gate], 1), both)
    a = ops.int8_experts(x, ids, w, routed).double()
    one = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    b = ops.int8_experts(x, one, torch.ones(T, 1, device="cuda"), shared).double()
    rows = [ops.int8_experts(x, ids[:, i:i + 1].contiguous(), torch.ones(T, 1, device="cuda"), routed)
            for i in range(k)]
    size = sum(w[:, i:i + 1].double() * r.double().abs() for i, r in enumerate(rows)) + gate * b.abs()
    want, h = a + gate.double() * b, half(dtype)
    tol = h * a.abs() * (1 + h) + h * want.abs() * (1 + h) + 2 * (k + 1) * U * size
    assert bool(((out.double() - want).abs() <= tol).all())


def test_gradients_end_with_an_error():
    """An input that requires a gradient changes no value, and a backward pass raises."""
    ex = make_experts(4, 64, 32, 1).to("cuda")
    x = torch.randn(9, 64).to(torch.bfloat16).cuda()
    ids, w = torch.zeros(9, 2, dtype=torch.int32).cuda(), torch.ones(9, 2).cuda()
    leaf = x.clone().requires_grad_()
    for call in (lambda t: ops.int8_experts(t, ids, w, ex),
                 lambda t: ops.int8_linear(t, ex.gate[0].contiguous(), ex.gate_scale[0].contiguous())):
        out = call(leaf * 1)
        assert torch.equal(out, call(x))
        with pytest.raises(NotImplementedError, match="no gradient"):
            out.sum().backward()
    assert leaf.grad is None
