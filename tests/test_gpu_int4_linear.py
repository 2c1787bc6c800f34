"""The int4 linear layer against its formula in 64 bits.

Two kinds of inputs. With activations that are small integers and scales that are powers of two every
product and sum is an integer multiple of 1/4 below 2^24 / 4, exact in fp32 in any order and with any
offset of the weights, so the result is the correctly rounded value: equality. With random ones a group's
sum may be formed from weights offset by 128 (x (128 + q) less (128 + z) x: magnitudes up to 286 |x|) over
G products and 4 more roundings, and K / G groups are added in up to K / G + 8 roundings:
(G + K / G + 12) u * 286 * sum_k s |x|, rounded once to the type.
"""

from __future__ import annotations

import pytest
import torch

from mtp_amd import awq, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, FP = torch.bfloat16, torch.float16


def pack(values):
    """Eight neighbours of the first dimension into an int32, the first in the lowest bits."""
    v = values.to(torch.int64).view(values.shape[0] // 8, 8, -1)
    word = sum(v[:, j] << (4 * j) for j in range(8))
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)


def make(K, N, G, seed=0):
    """(q, z) and the packed tensors of random nibbles."""
    g = torch.Generator().manual_seed(seed + K + N)
    q = torch.randint(0, 16, (K, N), generator=g)
    z = torch.randint(0, 16, (K // G, N), generator=g)
    return q, z, pack(q), pack(z.T.contiguous()).T.contiguous(), g


def exact(x, q, z, s, G, bias=None):
    w = ((q.double().view(-1, G, q.shape[1]) - z.double()[:, None]) * s.double()[:, None]).view(q.shape)
    y = x.double() @ w
    return y if bias is None else y + bias.double()


SIZES = [  # T, K, N, G
    (1, 32, 8, 32), (1, 128, 8, 128), (1, 2048, 4096, 128), (2, 256, 72, 64), (3, 1056, 2008, 32),
    (5, 4096, 512, 128), (8, 512, 1000, 256), (15, 768, 136, 768), (16, 2048, 264, 128), (17, 384, 96, 96),
    (31, 1024, 520, 64), (33, 640, 264, 32), (64, 2048, 1032, 128), (65, 128, 2056, 128),
    (100, 1152, 328, 64), (129, 2048, 776, 128), (203, 1056, 2008, 32), (257, 512, 264, 256),
    (300, 4096, 136, 128), (520, 1024, 1544, 64), (1000, 256, 520, 32), (513, 8192, 264, 128),
    (7, 8192, 24, 2048), (2050, 128, 264, 128), (1, 65536, 16, 128), (40, 65536, 8, 4096)]


@pytest.mark.parametrize("T,K,N,G", SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_exact_sums(T, K, N, G, dtype):
    q, z, qw, qz, g = make(K, N, G)
    top = 2 if K <= 8192 else 1
    x = torch.randint(-top, top + 1, (T, K), generator=g).to(dtype)
    if K > 8192:  # fewer terms: sums stay below 2^24 / 4
        x *= torch.rand(T, K, generator=g) < 0.1
    s = torch.tensor([0.25, 0.5, 1.0])[torch.randint(0, 3, (K // G, N), generator=g)].half()
    bias = torch.randint(-8, 9, (N,), generator=g).to(dtype) if N % 3 else None
    want = exact(x, q, z, s, G, bias).float().to(dtype)
    got = ops.int4_linear(x.cuda(), qw.cuda(), qz.cuda(), s.cuda(), group_size=G,
                          bias=None if bias is None else bias.cuda())
    assert torch.equal(got.cpu(), want), int((got.cpu() != want).sum())


TILES = [  # T, K, N, G: many rows: every tile, groups that end after one, two and more half steps, K that ends in
    # the middle of a step, 1 to 13 steps, ragged last tiles
    (3000, 512, 520, 128), (3001, 416, 776, 32), (2500, 832, 392, 64), (4000, 96, 1032, 96), (9000, 64, 640, 64),
    (5000, 160, 776, 32), (4990, 256, 904, 128), (5003, 192, 776, 192), (6000, 640, 520, 640),
    (9000, 96, 1032, 96), (9000, 128, 1032, 64), (8200, 384, 1288, 128), (7000, 448, 1544, 64),
    (16400, 128, 1160, 128), (16390, 32, 1288, 32), (16500, 64, 1160, 64), (13000, 320, 1544, 64),
    (12900, 384, 1672, 128), (12850, 224, 1800, 32)]
TILES += [  # rows between few and many, by tiles of 64 x 64: up to 256, up to 512, up to 1024 of them; groups of one,
    # two, three and more steps of 64, K of one step (shares of K without any), odd numbers of steps, ragged tiles
    (33, 64, 10376, 64), (64, 192, 10248, 64), (65, 128, 5256, 128), (70, 1088, 5320, 64), (130, 576, 3496, 192),
    (500, 2048, 1288, 128), (961, 640, 648, 320), (2000, 512, 392, 512), (4033, 384, 184, 128), (10300, 320, 8, 64),
    (129, 64, 5640, 64), (40, 448, 16648, 64), (100, 1024, 10504, 256), (300, 896, 3592, 128), (1000, 1088, 2008, 64),
    (2049, 2048, 648, 2048), (190, 960, 6600, 192), (16500, 128, 72, 128),
    (255, 64, 8264, 64), (257, 704, 8200, 64), (600, 1280, 4104, 640), (1025, 1536, 2056, 128), (4000, 384, 776, 128),
    (511, 128, 16392, 128), (65, 192, 33288, 64), (40000, 64, 72, 64)]


@pytest.mark.parametrize("T,K,N,G", TILES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_exact_sums_of_many_rows(T, K, N, G, dtype):
    """Scales are powers of two again, some of them zero: their groups count nothing."""
    q, z, qw, qz, g = make(K, N, G)
    x = torch.randint(-2, 3, (T, K), generator=g).to(dtype)
    s = torch.tensor([0.25, 0.5, 1.0, 0.0, -0.5])[torch.randint(0, 5, (K // G, N), generator=g)].half()
    s[-1, ::3] = 0.0
    bias = torch.randint(-8, 9, (N,), generator=g).to(dtype) if T % 2 else None
    want = exact(x.cuda(), q.cuda(), z.cuda(), s.cuda(), G, None if bias is None else bias.cuda()).float().to(dtype)
    got = ops.int4_linear(x.cuda(), qw.cuda(), qz.cuda(), s.cuda(), group_size=G,
                          bias=None if bias is None else bias.cuda())
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("T,K,N,G", [(1, 2048, 512, 128), (13, 1056, 200, 32), (40, 512, 264, 64),
                                     (150, 2048, 328, 128), (700, 1024, 520, 64), (1200, 384, 1032, 384), (1500, 2048, 1032, 128), (2600, 1056, 520, 32),
                                     (4400, 512, 4104, 64), (4096, 1024, 2056, 128),
                                     (100, 2048, 5448, 128), (200, 1088, 8200, 64), (700, 1024, 4104, 128)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_random_values(T, K, N, G, dtype):
    q, z, qw, qz, g = make(K, N, G, 1)
    x = torch.randn(T, K, generator=g)
    x = (x * torch.where(torch.rand(K, generator=g) < 0.02, 20.0, 1.0)).to(dtype)
    s = (0.01 * (0.5 + torch.rand(K // G, N, generator=g))).half()
    bias = torch.randn(N, generator=g).to(dtype)
    on = lambda t: t.cuda()  # noqa: E731
    want = exact(on(x), on(q), on(z), on(s), G, on(bias)).cpu()
    size = x.double().abs().view(T, -1, G).sum(2) @ s.double()
    got = ops.int4_linear(x.cuda(), qw.cuda(), qz.cuda(), s.cuda(), group_size=G, bias=bias.cuda())
    half = torch.finfo(dtype).eps / 2
    tol = (1 + half) * ((G + K // G + 12) * U * 286 * size + U * want.abs()) + half * want.abs() + 2.0 ** -25
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def test_the_layer_is_the_dequantised_product():
    """dequantize gives the same weights (to their rounding, 2^-8 or 2^-11 of each)."""
    q, z, qw, qz, g = make(512, 256, 64, 2)
    s = (0.02 * (0.5 + torch.rand(8, 256, generator=g))).half()
    x = torch.randn(20, 512, generator=g).to(BF).cuda()
    w = ops.dequantize(qw.cuda(), qz.cuda(), s.cuda(), group_size=64, dtype=torch.float32)
    want = x.float().cpu().double() @ w.cpu().double().T
    got = ops.int4_linear(x, qw.cuda(), qz.cuda(), s.cuda(), group_size=64).cpu().double()
    size = x.float().cpu().double().abs() @ w.cpu().double().T.abs()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -11 * size).all())


def test_awq_projection():
    """A dense AWQ projection, repacked as one expert."""
    K, N, G = 256, 128, 128
    g = torch.Generator().manual_seed(4)
    b = torch.randint(0, 256, (1, N, K // 2), generator=g).to(torch.uint8)
    zp = torch.randint(0, 256, (1, N // 2, K // G), generator=g).to(torch.uint8)
    s = torch.full((1, N, K // G), 0.5).half()
    st = awq.awq_to_gptq(b.cuda(), zp.cuda(), s.cuda(), layout="wna16", in_features=K, group_size=G)
    x = torch.randint(-2, 3, (9, K), generator=g).to(BF)
    q = torch.stack((b[0] & 15, b[0] >> 4), 2).view(N, K).T.contiguous()
    z = torch.stack((zp[0] & 15, zp[0] >> 4), 1).view(N, K // G).T.contiguous()
    want = exact(x, q, z, s[0].T, G).float().to(BF)
    got = ops.int4_linear(x.cuda(), st.qweight[0], st.qzeros[0], st.scales[0], group_size=G)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("T", [1, 20, 100, 600, 3500])
def test_rows_do_not_touch_each_other(T):
    """An infinity or NaN in one token leaves the others' results; zeros of scale and padding of the
    output are left as they are."""
    K, N, G = 512, 264, 128
    q, z, qw, qz, g = make(K, N, G, 3)
    s = (0.01 * torch.rand(K // G, N, generator=g)).half()
    s[1] = 0.0
    x = torch.randn(T, K, generator=g).to(BF)
    args = qw.cuda(), qz.cuda(), s.cuda()
    clean = ops.int4_linear(x.cuda(), *args)
    bad = x.clone()
    bad[T // 2, 5], bad[0, 130] = float("nan"), float("inf")
    got = ops.int4_linear(bad.cuda(), *args)
    keep = [t for t in range(T) if t not in (0, T // 2)]
    assert bool(clean.isfinite().all()) and torch.equal(got[keep], clean[keep])
    assert not bool(got[T // 2].isfinite().any())


@pytest.mark.parametrize("T", [1, 16, 50, 260, 700, 7000])
def test_unaligned_tensors(T):
    """x, bias and scales 2 bytes off a boundary, int32 tensors 4 bytes off."""
    K, N, G = 256, 136, 64
    q, z, qw, qz, g = make(K, N, G, 5)

    def off(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        return flat[1:].view(t.shape).copy_(t)

    x = torch.randint(-2, 3, (T, K), generator=g).to(FP)
    s = torch.tensor([0.25, 0.5, 1.0])[torch.randint(0, 3, (K // G, N), generator=g)].half()
    bias = torch.randint(-8, 9, (N,), generator=g).to(FP)
    want = exact(x, q, z, s, G, bias).float().to(FP)
    got = ops.int4_linear(off(x), off(qw), off(qz), off(s), group_size=G, bias=off(bias))
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("T", [4, 150, 500, 1400])
def test_a_bias_off_a_boundary(T):
    """Only the bias starts 2 bytes off: the kernels for aligned tensors take it."""
    K, N, G = 256, 5448, 128
    q, z, qw, qz, g = make(K, N, G, 6)
    x = torch.randint(-2, 3, (T, K), generator=g).to(BF)
    s = torch.tensor([0.25, 0.5, 1.0])[torch.randint(0, 3, (K // G, N), generator=g)].half()
    bias = torch.randint(-8, 9, (N,), generator=g).to(BF)
    off = torch.zeros(N + 1, dtype=BF, device="cuda")[1:].copy_(bias)
    got = ops.int4_linear(x.cuda(), qw.cuda(), qz.cuda(), s.cuda(), group_size=G, bias=off)
    assert torch.equal(got.cpu(), exact(x, q, z, s, G, bias).float().to(BF))


def test_no_tokens():
    _, _, qw, qz, _ = make(128, 64, 128)
    s = torch.ones(1, 64).half().cuda()
    assert ops.int4_linear(torch.empty(0, 128, dtype=BF, device="cuda"), qw.cuda(), qz.cuda(), s).shape == (0, 64)


@pytest.mark.parametrize("sizes", [((1, 2048, 512, 128), (1, 4096, 264, 128)), ((90, 1024, 520, 64),) * 2,
                                   ((3200, 512, 520, 128), (9, 512, 264, 128)),
                                   ((3000, 640, 520, 64),) * 2])
def test_captured_calls_on_streams_of_their_own(sizes):
    """Two captured layers replayed on two streams at once, on changing inputs."""
    made = []
    for i, (T, K, N, G) in enumerate(sizes):
        q, z, qw, qz, g = make(K, N, G, i)
        s = torch.tensor([0.25, 0.5, 1.0])[torch.randint(0, 3, (K // G, N), generator=g)].half()
        x = torch.zeros(T, K, dtype=BF, device="cuda")
        args = qw.cuda(), qz.cuda(), s.cuda()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.int4_linear(x, *args, group_size=G)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = ops.int4_linear(x, *args, group_size=G)
        made.append((x, args, out, graph, stream, (q, z, s, G), g))
    for _ in range(3):
        news = []
        for x, _, _, _, _, _, g in made:
            new = torch.randint(-2, 3, tuple(x.shape), generator=g).to(BF)
            x.copy_(new)
            news.append(new)
        torch.cuda.synchronize()
        for *_, graph, stream, _, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for new, (_, _, out, _, _, (q, z, s, G), _) in zip(news, made):
            assert torch.equal(out.cpu(), exact(new, q, z, s, G).float().to(BF))


def test_decode_step_of_a_block():
    """layer_norm -> int4 projection -> router -> int8-free routing of a serving step: the norm's rounded
    rows through the projection, and the projection's through the router."""
    T, H, N, E = 6, 512, 256, 32
    q, z, qw, qz, g = make(H, N, 128, 8)
    s = (0.01 * (0.5 + torch.rand(H // 128, N, generator=g))).half()
    x = torch.randn(T, H, generator=g).to(BF).cuda()
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(BF).cuda()
    xn = ops.layer_norm(x, w)
    y = ops.int4_linear(xn, qw.cuda(), qz.cuda(), s.cuda())
    want = exact(xn.cpu(), q, z, s, 128)
    size = xn.cpu().double().abs().view(T, -1, 128).sum(2) @ s.double()
    tol = 2.0 ** -8 * want.abs() + 160 * U * 286 * size
    assert bool(((y.cpu().double() - want).abs() <= tol).all())
    router = torch.randn(E, N, generator=g).to(BF).cuda()
    ids, weights, _, logits = ops.router_topk(y, router, 4)
    route = ops.route_tokens(logits.contiguous(), 4)
    assert torch.equal(ids, route.topk_ids)
    assert bool(((weights - route.topk_weights).abs() <= 100 * U * weights).all())
    assert int(route.counts.sum()) == 4 * T
