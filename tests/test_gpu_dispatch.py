"""Token rows sorted by expert and back (dispatch_tokens, combine_tokens) and their gradients,
against plain 64-bit computations on the host.

Tables and rows are copies and integers: equal. Sums: u = 2^-24 is fp32's half step, h the row
type's. A sum of k products in a chain of fused multiply-adds is off by at most (k + 1) u times the
sum of the terms' magnitudes, the store by h times the result; a dot product adds per thread over its
columns (8 for every 512 columns at the least), then over 6 butterfly steps and up to 4 waves.
"""

from __future__ import annotations

import math

import pytest
import torch

from mtp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# smallest half step of a type: where results are subnormal
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def half(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def make_ids(T, k, E, seed, dropped=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T, k), generator=g, dtype=torch.int32)
    drop = torch.rand(T, k, generator=g) < dropped
    bad = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31])[torch.randint(0, 4, (T, k), generator=g)]
    return torch.where(drop, bad.to(torch.int32), ids)


def plain_tables(ids, E):
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    row_slot = torch.argsort(key, stable=True)
    row = torch.empty_like(row_slot)
    row[row_slot] = torch.arange(flat.numel())
    offsets = torch.zeros(E + 1, dtype=torch.long)
    offsets[1:] = torch.bincount(key, minlength=E + 1)[:E].cumsum(0)
    return offsets, row_slot, torch.where(key < E, row, ~row).view(ids.shape)


CASES = [  # T, k, E, H, dtype
    (1, 1, 1, 1, torch.float32), (1, 8, 256, 2048, torch.bfloat16), (3, 64, 7, 72, torch.float16),
    (8, 8, 256, 2048, torch.bfloat16), (33, 5, 60, 1000, torch.float32),
    (17, 3, 512, 333, torch.bfloat16), (256, 8, 256, 512, torch.float16),
    (257, 8, 511, 520, torch.bfloat16), (700, 9, 512, 77, torch.float16),
    (2050, 2, 3, 1032, torch.float32), (999, 11, 64, 4104, torch.bfloat16)]


@pytest.mark.parametrize("T,k,E,H,dtype", CASES)
def test_dispatch_tables_and_rows(T, k, E, H, dtype):
    ids = make_ids(T, k, E, T + k)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dtype)
    x.view(-1)[0] = float("nan")  # a row is copied bit for bit; a dropped slot's is zeros
    d = ops.dispatch_tokens(x.cuda(), ids.cuda(), E)
    offsets, row_slot, slot_row = plain_tables(ids, E)
    assert torch.equal(d.offsets.cpu().long(), offsets)
    assert torch.equal(d.row_slot.cpu().long(), row_slot)
    assert torch.equal(d.slot_row.cpu().long(), slot_row)
    rows = x[row_slot // k]
    rows[offsets[-1]:] = 0
    as_int = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(d.rows.cpu().view(as_int), rows.view(as_int))


@pytest.mark.parametrize("T,k,E,H,dtype", CASES)
def test_combine_and_gradients(T, k, E, H, dtype):
    g = torch.Generator().manual_seed(T * 7 + k)
    ids = make_ids(T, k, E, T + k)
    _, row_slot, slot_row = plain_tables(ids, E)
    y = torch.randn(T * k, H, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g)
    kept = slot_row >= 0
    row = torch.where(kept, slot_row, ~slot_row)
    y[row[~kept]] = float("nan")     # what dropped slots hold does not matter
    w[~kept] = float("inf")
    dout = torch.randn(T, H, generator=g).to(dtype)
    yg, wg = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = ops.combine_tokens(yg, slot_row.to(torch.int32).cuda(), wg)
    dy, dw = torch.autograd.grad(out, (yg, wg), dout.cuda())
    h = half(dtype)
    y0 = torch.where(kept[..., None], y[row].double(), 0.0)   # [T, k, H]
    w0 = torch.where(kept, w.double(), 0.0)
    want = (w0[..., None] * y0).sum(1)
    size = (w0[..., None] * y0).abs().sum(1)
    err = (out.detach().cpu().double() - want).abs()
    assert bool((err <= h * (want.abs() + (k + 1) * U * size) + (k + 1) * U * size
                 + TINY[dtype]).all())
    # d rows: one product in fp32, rounded to the type
    want = torch.zeros(T * k, H, dtype=torch.float64)
    want[row] = w0[..., None] * dout.double()[:, None, :]
    err = (dy.cpu().double() - want).abs()
    assert bool((err <= (h + 2 * U) * want.abs() + TINY[dtype]).all())
    terms = dout.double()[:, None, :] * y0
    depth = 8 * math.ceil(H / 512) + 12
    err = (dw.cpu().double() - terms.sum(2)).abs()
    assert bool((err <= depth * U * terms.abs().sum(2) + 2.0 ** -150).all())


@pytest.mark.parametrize("T,k,E,H,dtype", [(5, 8, 16, 64, torch.bfloat16),
                                           (300, 9, 64, 1000, torch.float32),
                                           (64, 3, 7, 33, torch.float16)])
def test_dispatch_gradient(T, k, E, H, dtype):
    ids = make_ids(T, k, E, T * 3)
    _, _, slot_row = plain_tables(ids, E)
    x = torch.randn(T, H).to(dtype).cuda().requires_grad_()
    d = ops.dispatch_tokens(x, ids.cuda(), E)
    drows = torch.randn(T * k, H, generator=torch.Generator().manual_seed(3)).to(dtype)
    (dx,) = torch.autograd.grad(d.rows, x, drows.cuda())
    kept = slot_row >= 0
    terms = torch.where(kept[..., None], drows[slot_row.clamp_min(0)].double(), 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    err = (dx.cpu().double() - want).abs()
    h = half(dtype)
    assert bool((err <= h * want.abs() + (1 + h) * k * U * size + TINY[dtype]).all())


def test_gradients_against_differences():
    """A scalar of dispatch -> a product per row -> combine moves with its inputs as the gradients
    say: central differences, whose rounding error (values of about 10 in fp32 over a step of 2^-6)
    stays under 2^-15 and whose truncation is zero (the scalar is linear in each input)."""
    T, k, E, H = 6, 3, 4, 16
    g = torch.Generator().manual_seed(0)
    ids = make_ids(T, k, E, 1, 0.1).cuda()
    x = torch.randn(T, H, generator=g).cuda().requires_grad_()
    w = torch.rand(T, k, generator=g).cuda().requires_grad_()
    m = (torch.randn(T * k, 1, generator=g)).cuda()
    v = torch.randn(T, H, generator=g).cuda()

    def value(x, w):
        d = ops.dispatch_tokens(x, ids, E)
        return (ops.combine_tokens(d.rows * m, d.slot_row, w) * v).double().sum()

    gx, gw = torch.autograd.grad(value(x, w), (x, w))
    step = 2.0 ** -6
    with torch.no_grad():
        for t, grad in ((x, gx), (w, gw)):
            for i in range(0, t.numel(), 5):
                e = torch.zeros_like(t).view(-1)
                e[i] = step
                e = e.view_as(t)
                hi, lo = ((value(x + s * e, w) if t is x else value(x, w + s * e)) for s in (1, -1))
                assert abs(float((hi - lo) / (2 * step)) - float(grad.reshape(-1)[i])) < 2.0 ** -12


def test_broadcast_gradients_and_partial_needs():
    """Expanded gradients (a sum's), gradients of one input only, and rows that are not used."""
    ids = make_ids(9, 4, 8, 2).cuda()
    x = torch.randn(9, 40).cuda().requires_grad_()
    d = ops.dispatch_tokens(x, ids, 8)
    d.rows.sum().backward()
    kept = (d.slot_row >= 0).sum(1, keepdim=True).float()
    assert torch.equal(x.grad, kept.expand_as(x))
    y = torch.randn(36, 40).cuda()
    w = torch.rand(9, 4).cuda()
    yg, wg = y.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(ops.combine_tokens(yg, d.slot_row, wg).sum(), (yg, wg))
    only_y = torch.autograd.grad(ops.combine_tokens(yg, d.slot_row, w).sum(), yg)[0]
    only_w = torch.autograd.grad(ops.combine_tokens(y, d.slot_row, wg).sum(), wg)[0]
    assert torch.equal(both[0], only_y) and torch.equal(both[1], only_w)
    out = ops.dispatch_tokens(x, ids, 8)
    assert not out.offsets.requires_grad and not out.slot_row.requires_grad
    with torch.no_grad():
        assert not ops.dispatch_tokens(x, ids, 8).rows.requires_grad


def test_no_tokens_and_all_dropped():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids = torch.empty(0, 4, device="cuda", dtype=torch.int32)
    d = ops.dispatch_tokens(x, ids, 5)
    assert torch.equal(d.offsets.cpu(), torch.zeros(6, dtype=torch.int32))
    out = ops.combine_tokens(d.rows, d.slot_row, torch.empty(0, 4, device="cuda"))
    assert out.shape == (0, 64)
    out.sum().backward()
    assert x.grad.shape == (0, 64)
    x = torch.randn(3, 64).cuda()
    d = ops.dispatch_tokens(x, torch.full((3, 4), -1, dtype=torch.int32).cuda(), 5)
    assert int(d.offsets.abs().sum()) == 0 and float(d.rows.abs().sum()) == 0.0
    assert torch.equal(d.slot_row.cpu().reshape(-1), ~torch.arange(12, dtype=torch.int32))
    out = ops.combine_tokens(torch.full((12, 64), float("nan")).cuda(), d.slot_row,
                             torch.ones(3, 4).cuda())
    assert float(out.abs().sum()) == 0.0


@pytest.mark.parametrize("off", [1, 2, 4])
def test_unaligned_bases(off):
    """Contiguous tensors that start off a 16-byte boundary take the narrow accesses."""
    T, k, E, H = 40, 8, 16, 64
    ids = make_ids(T, k, E, 5).cuda()
    x = torch.randn(T, H).to(torch.bfloat16).cuda()
    buf = torch.empty(T * H + off, dtype=torch.bfloat16, device="cuda")
    xo = buf[off:].view(T, H)
    xo.copy_(x)
    a, b = ops.dispatch_tokens(x, ids, E), ops.dispatch_tokens(xo, ids, E)
    assert torch.equal(a.rows, b.rows)
    w = torch.rand(T, k).cuda()
    buf2 = torch.empty(T * k * H + off, dtype=torch.bfloat16, device="cuda")
    ro = buf2[off:].view(T * k, H)
    ro.copy_(a.rows)
    assert torch.equal(ops.combine_tokens(a.rows, a.slot_row, w),
                       ops.combine_tokens(ro, a.slot_row, w))


def test_two_streams_and_graph_replays():
    """Calls on two streams at once, and a captured pass with gradients replayed between eager ones,
    give the eager results."""
    T, k, E, H = 900, 8, 64, 256
    ids = [make_ids(T, k, E, s).cuda() for s in (1, 2)]
    x = [torch.randn(T, H).to(torch.bfloat16).cuda() for _ in range(2)]
    w = torch.rand(T, k).cuda()
    eager = []
    for i in range(2):
        d = ops.dispatch_tokens(x[i], ids[i], E)
        eager.append((d, ops.combine_tokens(d.rows, d.slot_row, w)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            d = ops.dispatch_tokens(x[i], ids[i], E)
            got.append((d, ops.combine_tokens(d.rows, d.slot_row, w)))
    torch.cuda.synchronize()
    for (d0, o0), (d1, o1) in zip(eager, got):
        assert all(torch.equal(a, b) for a, b in zip(d0, d1)) and torch.equal(o0, o1)

    xs, wl = x[0].clone().requires_grad_(), w.clone().requires_grad_()
    ids_s, v = ids[0].clone(), torch.randn(T, H).to(torch.bfloat16).cuda()

    def step():
        d = ops.dispatch_tokens(xs, ids_s, E)
        out = ops.combine_tokens(d.rows, d.slot_row, wl)
        return (out.detach(), d.slot_row, *torch.autograd.grad(out, (xs, wl), v))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in (1, 0, 1):
        with torch.no_grad():
            xs.copy_(x[i])
            ids_s.copy_(ids[i])
        graph.replay()
        torch.cuda.synchronize()
        held = [t.detach().clone() for t in static]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.detach()) for a, b in zip(held, want))


def test_rows_beyond_4_gib():
    """The copies and sums of a routing whose rows take more than 2^32 bytes (4.4 GB of bf16), against
    the same values gathered and summed for some of the tokens."""
    T, k, E, H = 1 << 17, 8, 64, 2096
    gen = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-1, E, (T, k), generator=gen, dtype=torch.int32, device="cuda")
    x = torch.randn(T, H, generator=gen, dtype=torch.bfloat16, device="cuda")
    w = torch.rand(T, k, generator=gen, device="cuda")
    d = ops.dispatch_tokens(x, ids, E)
    assert d.rows.numel() * 2 > 1 << 32
    want = plain_tables(ids.cpu(), E)
    for a, b in zip((d.offsets, d.row_slot, d.slot_row), want):
        assert torch.equal(a.cpu().long(), b)
    kept = int(d.offsets[-1])
    for a in range(0, T * k, 1 << 17):
        slots = d.row_slot[a:a + (1 << 17)].long()
        rows = x[slots // k]
        rows[max(kept - a, 0):] = 0
        assert torch.equal(d.rows[a:a + (1 << 17)], rows)
    out = ops.combine_tokens(d.rows, d.slot_row, w)
    some = torch.cat([torch.arange(512), torch.arange(T - 512, T)]).cuda()
    part = ops.dispatch_tokens(x[some], ids[some], E)
    assert torch.equal(out[some], ops.combine_tokens(part.rows, part.slot_row, w[some]))
    rows, wl = d.rows.requires_grad_(), w.clone().requires_grad_()
    drows, dw = torch.autograd.grad(ops.combine_tokens(rows, d.slot_row, wl), (rows, wl), x)
    prows, pw = part.rows.requires_grad_(), w[some].requires_grad_()
    pdrows, pdw = torch.autograd.grad(ops.combine_tokens(prows, part.slot_row, pw), (prows, pw),
                                      x[some])
    assert torch.equal(dw[some], pdw)
    at, pat = d.slot_row[some].long().view(-1), part.slot_row.long().view(-1)
    assert torch.equal(drows[torch.where(at < 0, ~at, at)], pdrows[torch.where(pat < 0, ~pat, pat)])
