"""int8 quantisation, products and experts against exact integers and 64-bit computations.

Quantised values equal those of exact arithmetic (integers: round half to even of 127 x / a, which for
bf16 and fp16 inputs is what an IEEE division of exact operands gives); fp32 inputs equal the same
operations in fp32 on the host. The products' sums are exact, and sum -> * token scale -> * channel
scale are IEEE fp32 operations, so outputs without a bias equal the host's bit for bit; with a bias
the compiler may fuse the last product into the sum: off by half a step of the product (2^-24).
"""

from __future__ import annotations

from fractions import Fraction

import pytest
import torch

from mtp_amd import ops, synth
from mtp_amd.moe import MoeBlock
from mtp_amd.weights import Int8Experts

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def host_quantize(x):
    """fp32 host form (IEEE operations)."""
    x = x.float()
    a = x.abs().amax(dim=1, keepdim=True)
    q = (x * 127.0 / a).round()
    return torch.where(a > 0, q, 0.0).to(torch.int8), (a / 127.0)[:, 0]


def exact_quantize_row(row):
    a = max(abs(Fraction(float(v))) for v in row)
    return [0 if a == 0 else round(127 * Fraction(float(v)) / a) for v in row]  # half to even


@pytest.mark.parametrize("T,K,dtype", [(1, 1, torch.bfloat16), (5, 16, torch.float16),
                                       (9, 513, torch.bfloat16), (33, 512, torch.float32),
                                       (7, 2048, torch.bfloat16), (6, 2049, torch.float16),
                                       (3, 8192, torch.bfloat16), (2, 8200, torch.float32),
                                       (2, 65536, torch.bfloat16), (2, 65535, torch.float16)])
def test_quantize(T, K, dtype):
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    q, s = ops.quantize_tokens(x.cuda())
    want_q, want_s = host_quantize(x)
    assert torch.equal(q.cpu(), want_q)
    assert torch.equal(s.cpu(), want_s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_ties_and_extremes(dtype):
    """Exact halves (64 equally spaced values of an 8-bit significand make many), rows near the
    type's largest and smallest values, zeros, signed zeros, and every value against fractions."""
    top = float(torch.finfo(dtype).max)
    low = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133  # smallest subnormal
    grid = torch.arange(-128, 128, dtype=torch.float64)
    rows = torch.stack([grid / 128, grid / 127 * 100, grid * 2.0 ** -14, grid / 128 * top,
                        grid * low, torch.zeros(256, dtype=torch.float64),
                        torch.where(grid == 3, 254.0, grid)])
    x = rows.to(dtype)
    x[5, ::2] = -0.0
    q, s = ops.quantize_tokens(x.cuda())
    for i in range(x.shape[0]):
        assert q[i].cpu().tolist() == exact_quantize_row(x[i].tolist()), i
    assert torch.equal(s.cpu(), x.float().abs().amax(1) / 127.0)
    assert float(s[5]) == 0.0


def test_quantize_not_finite():
    x = torch.randn(4, 40).to(torch.bfloat16)
    x[0, 3], x[1, 39], x[2, 0] = float("inf"), float("nan"), float("-inf")
    q, s = ops.quantize_tokens(x.cuda())
    assert int(q[:3].abs().sum()) == 0 and bool(q[3].any())
    assert torch.isinf(s[0]) and torch.isnan(s[1]) and torch.isinf(s[2]) and torch.isfinite(s[3])
    y = ops.int8_linear(torch.nn.functional.pad(x, (0, 8)).cuda(),
                        torch.ones(5, 48, dtype=torch.int8).cuda(), torch.ones(5).cuda())
    assert bool(torch.isnan(y[:3]).all()) and bool(torch.isfinite(y[3]).all())


def make_weight(N, K, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    return w, torch.rand(N, generator=g) / 127


def host_product(q, qs, w, ws):
    acc = q.double() @ w.double().T  # integers below 2^53: exact
    return (acc.float() * qs[:, None]) * ws[None, :]


SHAPES = [  # T, K, N, dtype, bias
    (1, 16, 1, torch.bfloat16, False), (1, 2048, 4096, torch.bfloat16, False),
    (8, 4096, 8200, torch.float16, True), (5, 8192, 96, torch.float32, False),
    (7, 4224, 24, torch.bfloat16, True), (8, 6160, 40, torch.bfloat16, False),
    (9, 320, 8193, torch.float32, False), (3, 272, 19, torch.float32, False),
    (2, 48, 33, torch.float16, True), (15, 1040, 100, torch.bfloat16, True),
    (16, 64, 64, torch.float32, False), (17, 16, 1, torch.bfloat16, False),
    (20, 32, 7, torch.float16, True), (80, 16, 3, torch.float32, False), (17, 80, 65, torch.float16, False),
    (31, 2048, 96, torch.float32, True), (33, 144, 200, torch.bfloat16, False),
    (64, 4096, 130, torch.bfloat16, False), (65, 272, 257, torch.float16, True),
    (130, 512, 511, torch.bfloat16, True), (203, 1040, 2001, torch.float16, True),
    (257, 128, 256, torch.bfloat16, False), (300, 2064, 640, torch.float32, False),
    (513, 1552, 1000, torch.bfloat16, True), (1030, 256, 514, torch.float16, False),
    (2048, 2048, 2048, torch.bfloat16, False), (1100, 1168, 2500, torch.bfloat16, False),
    (400, 272, 3001, torch.float32, True), (513, 144, 2504, torch.bfloat16, False),
    (300, 96, 1200, torch.float32, False), (450, 400, 900, torch.float16, True),
    (3000, 272, 3001, torch.float32, True), (2990, 80, 3000, torch.bfloat16, False),
    (4099, 272, 3001, torch.float16, True), (5001, 144, 2500, torch.bfloat16, False)]


@pytest.mark.parametrize("T,K,N,dtype,bias", SHAPES)
def test_matmul_and_linear(T, K, N, dtype, bias):
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(N)).to(dtype)
    w, ws = make_weight(N, K, T)
    b = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(dtype) if bias else None
    q, qs = host_quantize(x)
    got = ops.int8_linear(x.cuda(), w.cuda(), ws.cuda(), bias=None if b is None else b.cuda()).cpu()
    again = ops.int8_matmul(q.cuda(), qs.cuda(), w.cuda(), ws.cuda(), dtype=dtype,
                            bias=None if b is None else b.cuda()).cpu()
    assert torch.equal(got, again)
    want = host_product(q, qs, w, ws)
    if b is None:
        assert torch.equal(got, want.to(dtype))
    else:
        full = want.double() + b.double()
        err = (got.double() - full).abs()
        slack = 2 * U * (want.double().abs() + b.double().abs())
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
        assert bool((err <= half(dtype) * (full.abs() + slack) + slack + tiny).all())


@pytest.mark.parametrize("T", [3, 40])
def test_linear_of_unaligned_rows(T):
    x = torch.randn(T, 96).to(torch.bfloat16).cuda()
    buf = torch.empty(T * 96 + 1, dtype=torch.bfloat16, device="cuda")
    xo = buf[1:].view(T, 96)
    xo.copy_(x)
    w, ws = make_weight(50, 96, 4)
    assert torch.equal(ops.int8_linear(xo, w.cuda(), ws.cuda()),
                       ops.int8_linear(x, w.cuda(), ws.cuda()))


def test_extreme_sums():
    """The largest sums: -128 * -128 over the largest K (2^30), and both signs of 127 * 128."""
    K = 65536
    q = torch.full((3, K), -128, dtype=torch.int8)
    q[1], q[2] = 127, -128
    w = torch.full((20, K), -128, dtype=torch.int8)
    w[1] = 127
    qs, ws = torch.ones(3), torch.ones(20)
    got = ops.int8_matmul(q.cuda(), qs.cuda(), w.cuda(), ws.cuda(), dtype=torch.float32).cpu()
    assert torch.equal(got, host_product(q, qs, w, ws))


def test_misaligned_int8_is_refused():
    from mtp_amd._lib import MoeLibraryError
    buf = torch.zeros(8 * 64 + 3, dtype=torch.int8, device="cuda")
    w = buf[3:].view(8, 64)
    with pytest.raises(MoeLibraryError, match="16-byte"):
        ops.int8_linear(torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda"), w,
                        torch.zeros(8, device="cuda"))


# ------------------------------------------------------------------------------ experts
def make_experts(E, H, I, seed):
    g = torch.Generator().manual_seed(seed)
    parts = []
    for n, k in ((I, H), (I, H), (H, I)):
        parts += [torch.randint(-127, 128, (E, n, k), generator=g, dtype=torch.int8),
                  (0.5 + torch.rand(E, n, generator=g)) / (64 * k ** 0.5)]
    return Int8Experts(*parts)


def expected_experts(x, ids, w, ex):
    """64-bit outputs and how far the kernels' may lie from them. The hidden values are computed in
    fp32 (e^-g: |g| + 8 half steps and less than 2^-18 in all for |g| < 20), so near a tie of their
    rounding or of their quantisation they may fall either way: the interval of h is carried through
    both roundings, and what the ends differ by is allowed."""
    T, H = x.shape
    k, dtype, delta = ids.shape[1], x.dtype, 2.0 ** -18
    out = torch.zeros(T, H, dtype=torch.float64)
    slack, size = torch.zeros_like(out), torch.zeros_like(out)
    q, qs = host_quantize(x)
    for t in range(T):
        for i in range(k):
            e = int(ids[t, i])
            if not 0 <= e < ex.num_experts:
                continue
            g = (ex.gate[e].double() @ q[t].double()) * float(qs[t]) * ex.gate_scale[e].double()
            u = (ex.up[e].double() @ q[t].double()) * float(qs[t]) * ex.up_scale[e].double()
            assert float(g.abs().max()) < 20
            h = g * torch.sigmoid(g) * u
            lo, hi = (h * (1 - delta)).to(dtype).double(), (h * (1 + delta)).to(dtype).double()
            mid = h.to(dtype).double()

            def levels(v, a):
                return torch.round(127 * v / a).clamp(-127, 127)

            a, a_lo, a_hi = mid.abs().max(), torch.minimum(lo.abs(), hi.abs()).max(), \
                torch.maximum(lo.abs(), hi.abs()).max()
            if float(a) == 0:
                continue
            step = a / 127
            base = levels(mid, a)
            spread = torch.zeros_like(base)
            for v in (lo, hi):
                for peak in (a_lo, a_hi):
                    spread = torch.maximum(spread, (levels(v, peak) * peak / 127 - base * step).abs())
            wd = ex.down[e].double()
            scale = ex.down_scale[e].double()
            y = (wd @ base) * step * scale
            dy = (wd.abs() @ spread) * scale + 4 * U * y.abs()
            dy = dy + half(dtype) * (y.abs() + dy)  # rounded to the type
            wt = float(w[t, i])
            out[t] += wt * y
            slack[t] += abs(wt) * dy
            size[t] += abs(wt) * (y.abs() + dy)
    slack += (k + 1) * U * size
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return out, slack * (1 + half(dtype)) + half(dtype) * out.abs() + (k + 1) * tiny


@pytest.mark.parametrize("T,k,E,H,I,dtype", [
    (1, 1, 1, 16, 16, torch.bfloat16), (1, 8, 16, 256, 128, torch.bfloat16),
    (5, 3, 8, 272, 144, torch.float16), (37, 4, 8, 256, 128, torch.float32),
    (64, 8, 12, 128, 80, torch.bfloat16), (150, 2, 3, 144, 208, torch.bfloat16),
    (270, 2, 2, 96, 48, torch.float16), (420, 3, 2, 160, 272, torch.bfloat16)])
def test_experts(T, k, E, H, I, dtype):
    g = torch.Generator().manual_seed(T + E)
    x = torch.randn(T, H, generator=g).to(dtype)
    ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    ids[torch.rand(T, k, generator=g) < 0.1] = -1
    if T > 30:
        ids[7] = E  # a token none of whose slots is kept
    w = torch.rand(T, k, generator=g)
    ex = make_experts(E, H, I, 5)
    got = ops.int8_experts(x.cuda(), ids.cuda(), w.cuda(), ex.to("cuda")).cpu().double()
    want, tol = expected_experts(x, ids, w, ex)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
    dropped = ((ids < 0) | (ids >= E)).all(1)
    assert float(got[dropped].abs().sum()) == 0.0


@pytest.mark.parametrize("T,k,E,H,I", [
    (90, 4, 6, 64, 32), (11, 8, 70, 2064, 48), (600, 8, 5, 2064, 48), (1024, 4, 64, 144, 512),
    (1500, 3, 5, 272, 1008), (2048, 4, 4, 144, 512), (1300, 8, 40, 96, 1552)])
def test_experts_equal_their_parts(T, k, E, H, I):
    """Rows whose h is the same give what dispatch, int8_matmul over each expert's rows, and combine
    give: with gates so large that silu(g) = g exactly and up sums that make h exact in the type."""
    gen = torch.Generator().manual_seed(T)
    ex = make_experts(E, H, I, 9).to("cuda")
    ids = torch.randint(-1, E, (T, k), generator=gen, dtype=torch.int32).cuda()
    w = torch.rand(T, k, generator=gen).cuda()
    x = torch.zeros(T, H, dtype=torch.float32, device="cuda")
    x[:, 0] = 127.0  # q = (127, 0, ...): g = gate[e, :, 0] * 127 * scale
    x[:, H - 1] = torch.randint(-127, 128, (T,), generator=gen).float().cuda()
    gate, up = torch.zeros_like(ex.gate), torch.zeros_like(ex.up)
    gate[:, :, 0] = 64
    up[:, :, 0] = torch.randint(-127, 128, (E, I), generator=gen, dtype=torch.int8).cuda()
    up[:, :, H - 1] = torch.randint(-127, 128, (E, I), generator=gen, dtype=torch.int8).cuda()
    one = torch.ones(E, I, device="cuda")
    ex = Int8Experts(gate, one, up, one / 127, ex.down, ex.down_scale)
    got = ops.int8_experts(x, ids, w, ex)
    d = ops.dispatch_tokens(x, ids, E)
    y = torch.zeros(T * k, H, device="cuda")
    ends = d.offsets.tolist()
    for e in range(E):
        rows = d.rows[ends[e]:ends[e + 1]].contiguous()
        g = ops.int8_linear(rows, ex.gate[e].contiguous(), ex.gate_scale[e].contiguous())
        u = ops.int8_linear(rows, ex.up[e].contiguous(), ex.up_scale[e].contiguous())
        y[ends[e]:ends[e + 1]] = ops.int8_linear(g * u, ex.down[e].contiguous(),
                                                 ex.down_scale[e].contiguous())
    assert torch.equal(got, ops.combine_tokens(y, d.slot_row, w))


@pytest.mark.parametrize("T,k,E,dtype", [(130, 2, 300, torch.bfloat16), (90, 1, 64, torch.float32),
                                         (500, 3, 40, torch.float16)])
def test_experts_of_uneven_routing(T, k, E, dtype):
    """Most tokens at two experts of many (several tiles of an expert while the average is a few rows):
    a token's values are those of a call of its own."""
    ex = make_experts(E, 96, 144, 8).to("cuda")
    gen = torch.Generator().manual_seed(T)
    ids = torch.where(torch.rand(T, k, generator=gen) < 0.8, torch.randint(3, 5, (T, k), generator=gen),
                      torch.randint(0, E, (T, k), generator=gen)).to(torch.int32).cuda()
    w = torch.rand(T, k, generator=gen).cuda()
    x = torch.randn(T, 96, generator=gen).to(dtype).cuda()
    got = ops.int8_experts(x, ids, w, ex)
    for t in range(0, T, 7):
        assert torch.equal(got[t:t + 1], ops.int8_experts(x[t:t + 1], ids[t:t + 1], w[t:t + 1], ex)), t


@pytest.mark.parametrize("T", [3, 700])
def test_experts_graph_streams_and_workspace(T):
    """A captured call replayed on new inputs between eager calls, two calls on two streams, and a
    caller's workspace that holds NaN patterns from before give the eager results."""
    k, E, H, I = 8, 32, 256, 128
    ex = make_experts(E, H, I, 2).to("cuda")
    xs = [torch.randn(T, H).to(torch.bfloat16).cuda() for _ in range(2)]
    ids = [torch.randint(-1, E, (T, k), dtype=torch.int32).cuda() for _ in range(2)]
    w = torch.rand(T, k).cuda()
    want = [ops.int8_experts(x, i, w, ex) for x, i in zip(xs, ids)]
    ws = torch.full((ops.int8_experts_workspace_bytes(T, k, ex),), 255, dtype=torch.uint8,
                    device="cuda")
    assert torch.equal(ops.int8_experts(xs[0], ids[0], w, ex, workspace=ws), want[0])
    assert torch.equal(ops.int8_experts(xs[1], ids[1], w, ex, workspace=ws), want[1])
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(ops.int8_experts(xs[i], ids[i], w, ex))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x0, i0 = xs[0].clone(), ids[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.int8_experts(x0, i0, w, ex)
    for i in (1, 0, 1):
        x0.copy_(xs[i])
        i0.copy_(ids[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.equal(ops.int8_experts(xs[i], ids[i], w, ex), want[i])


@pytest.mark.parametrize("T", [3, 40, 300])
def test_linear_in_a_graph(T):
    """A captured linear layer replayed on new inputs between eager calls gives the eager results: the
    fused kernel, and the ones that keep quantised rows in a workspace."""
    w, ws = make_weight(130, 272, T)
    w, ws = w.cuda(), ws.cuda()
    xs = [torch.randn(T, 272).to(torch.bfloat16).cuda() for _ in range(2)]
    want = [ops.int8_linear(x, w, ws) for x in xs]
    x0 = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.int8_linear(x0, w, ws)
    for i in (1, 0, 1):
        x0.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        assert torch.equal(ops.int8_linear(xs[i], w, ws), want[i])


@pytest.mark.parametrize("T", [5, 700])
def test_experts_of_unaligned_rows(T):
    ex = make_experts(9, 96, 48, 3).to("cuda")
    x = torch.randn(T, 96).to(torch.float16).cuda()
    buf = torch.empty(T * 96 + 1, dtype=torch.float16, device="cuda")
    xo = buf[1:].view(T, 96)
    xo.copy_(x)
    ids = torch.randint(0, 9, (T, 8), dtype=torch.int32).cuda()
    w = torch.rand(T, 8).cuda()
    assert torch.equal(ops.int8_experts(xo, ids, w, ex), ops.int8_experts(x, ids, w, ex))


def test_no_tokens():
    ex = make_experts(4, 64, 32, 1).to("cuda")
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    out = ops.int8_experts(x, torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                           torch.empty(0, 2, device="cuda"), ex)
    assert out.shape == (0, 64)
    assert ops.int8_linear(x, ex.gate[0].contiguous(), ex.gate_scale[0].contiguous()).shape == (0, 32)
    assert ops.quantize_tokens(x)[0].shape == (0, 64)


def test_from_gptq_and_moe_block():
    """int4 experts requantised to int8 run in MoeBlock's forward and moe_tokens: the block's routing
    equals the int4 block's, its output is int8_experts over that routing, and it lies as near the
    int4 block as int8's half steps leave it: relative to the largest output, below 5 % (three
    quantisations of 1/254 of a row's largest value each, sums of random signs)."""
    layer = synth.layer_to(synth.make_layer(3, num_experts=16, hidden=512, intermediate=256), "cuda")
    ex8 = Int8Experts.from_gptq(layer.experts)
    w = ops.dequantize(layer.experts.up.qweight[5], layer.experts.up.qzeros[5],
                       layer.experts.up.scales[5], dtype=torch.float32)
    err = (ex8.up[5].float() * ex8.up_scale[5][:, None] - w).abs()
    assert bool((err <= 0.5 * (1 + 2.0 ** -10) * ex8.up_scale[5][:, None]).all())
    dense = [torch.stack([ops.dequantize(p.qweight[e], p.qzeros[e], p.scales[e],
                                         dtype=torch.float32) for e in range(16)])
             for p in (layer.experts.gate, layer.experts.up, layer.experts.down)]
    again = Int8Experts.from_dense(*dense)
    assert torch.equal(again.down, ex8.down) and torch.equal(again.gate_scale, ex8.gate_scale)
    x = synth.make_tokens(40, 512, seed=4).cuda().view(2, 20, 512)
    b4 = MoeBlock(layer.experts, layer.router_w, top_k=4)
    b8 = MoeBlock(ex8, layer.router_w, top_k=4)
    y4, ids4, w4 = b4(x, return_routing=True)
    y8, ids8, w8 = b8(x, return_routing=True)
    assert torch.equal(ids4, ids8) and torch.equal(w4, w8)
    flat = ops.int8_experts(x.view(40, 512), ids8, w8, ex8)
    assert torch.equal(y8.view(40, 512), flat)
    assert torch.equal(b8.moe_tokens(x, ids8.view(2, 20, 4), w8.view(2, 20, 4)), y8)
    assert float((y8.float() - y4.float()).abs().max() / y4.float().abs().max()) < 0.05


def test_weights_and_outputs_beyond_4_gib():
    """The last experts of stacks of more than 2^32 bytes give what they give as a set of their own,
    and the last rows of an output of more than 2^32 bytes what they give alone."""
    E, H, I, T, k = 300, 4096, 3584, 40, 3
    gen = torch.Generator(device="cuda").manual_seed(1)

    def weights(*shape):
        return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8, device="cuda")

    parts = []
    for n, K in ((I, H), (I, H), (H, I)):
        parts += [weights(E, n, K), torch.rand(E, n, generator=gen, device="cuda") / 8192]
    assert parts[0].numel() > 1 << 32
    last = Int8Experts(*(t[-4:].clone() for t in parts))
    x = torch.randn(T, H, generator=gen, dtype=torch.bfloat16, device="cuda")
    ids = torch.randint(0, 4, (T, k), generator=gen, dtype=torch.int32, device="cuda")
    w = torch.rand(T, k, generator=gen, device="cuda")
    assert torch.equal(ops.int8_experts(x, ids + (E - 4), w, Int8Experts(*parts)),
                       ops.int8_experts(x, ids, w, last))
    del parts
    T, K, N = 66000, 64, 32776
    x = torch.randn(T, K, generator=gen, dtype=torch.bfloat16, device="cuda")
    wq, ws = weights(N, K), torch.rand(N, generator=gen, device="cuda")
    out = ops.int8_linear(x, wq, ws)
    assert out.numel() * 2 > 1 << 32
    assert torch.equal(out[-300:], ops.int8_linear(x[-300:].clone(), wq, ws))
