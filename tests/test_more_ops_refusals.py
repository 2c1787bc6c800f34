"""Refusals of the int4 linear layer, the routing with its losses and the layer norm, and the derivatives
that they do not have: nothing is launched (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mtp_amd import _lib, ops

F, I, HALF = torch.bfloat16, torch.int32, torch.float16


def z(*shape, dtype=F):
    return torch.zeros(*shape, dtype=dtype)


def int4(x=None, K=128, N=16, G=128, **kw):
    at = {"qweight": z(K // 8, N, dtype=I), "qzeros": z(K // G, N // 8, dtype=I),
          "scales": z(K // G, N, dtype=HALF), "group_size": G, **kw}
    return ops.int4_linear(z(4, K) if x is None else x, at["qweight"], at["qzeros"], at["scales"],
                           group_size=at["group_size"], bias=at.get("bias"))


@pytest.mark.parametrize("call,error", [
    (lambda: int4(), ValueError),  # host tensors
    (lambda: int4(z(4, 128, dtype=torch.float32)), TypeError),
    (lambda: int4(z(4, 128, dtype=torch.float64)), TypeError),
    (lambda: int4(z(128)), ValueError),
    (lambda: int4(z(4, 120)), ValueError),
    (lambda: int4(qweight=z(16, 16)), TypeError),
    (lambda: int4(scales=z(1, 16)), TypeError),
    (lambda: int4(scales=z(2, 16, dtype=HALF)), ValueError),
    (lambda: int4(qzeros=z(1, 3, dtype=I)), ValueError),
    (lambda: int4(qweight=z(1, 16, 16, dtype=I)), ValueError),
    (lambda: int4(group_size=96), ValueError),
    (lambda: int4(group_size=0), ValueError),
    (lambda: int4(bias=torch.zeros(16)), ValueError),
    (lambda: int4(bias=z(8)), ValueError),
    (lambda: ops.route_tokens(z(4, 8), 2), ValueError),  # host tensors
    (lambda: ops.route_tokens(z(4, 8, dtype=torch.float64), 2), TypeError),
    (lambda: ops.route_tokens(z(4, 8, 1), 2), ValueError),
    (lambda: ops.route_tokens(z(4, 8), 9), ValueError),
    (lambda: ops.route_tokens(z(4, 8), 0), ValueError),
    (lambda: ops.route_tokens(z(4, 100), 65), ValueError),
    (lambda: ops.route_tokens(z(4, 513), 2), ValueError),
    (lambda: ops.route_tokens(z(4, 0), 1), ValueError),
    (lambda: ops.route_tokens(z(4, 8), 2, mask=z(4)), ValueError),
    (lambda: ops.route_tokens(z(4, 8), 2, mask=z(5, dtype=torch.bool)), ValueError),
    (lambda: ops.layer_norm(z(4, 8)), ValueError),  # host tensors
    (lambda: ops.layer_norm(z(4, 8, dtype=torch.float64)), TypeError),
    (lambda: ops.layer_norm(z(8)), ValueError),
    (lambda: ops.layer_norm(z(4, 8), z(7)), ValueError),
    (lambda: ops.layer_norm(z(4, 8), torch.zeros(8)), ValueError),
    (lambda: ops.layer_norm(z(4, 8), z(8), z(1, 8)), ValueError),
])
def test_wrappers_refuse(call, error):
    with pytest.raises(error):
        call()


NULL, SHAPE, UNSUP, WS = (_lib.MOE_ERR_NULL, _lib.MOE_ERR_SHAPE, _lib.MOE_ERR_UNSUPPORTED,
                          _lib.MOE_ERR_WORKSPACE)
A, B, C, D, G, W, X, Y = (0x10000000 * i for i in range(1, 9))  # never dereferenced
BIG = 1 << 40


def proj(q=B, zeros=C, scales=D):
    return _lib.GptqProj(q, zeros, scales)


def lin(x=A, T=4, K=256, dt=0, p=None, N=64, gs=128, bias=None, ws=None, nb=0, out=G):
    return "moe_int4_linear_v1", (x, T, K, dt, proj() if p is None else p, N, gs, bias, ws, nb, out)


def route(logits=A, T=4, E=64, dt=0, k=2, mask=None, ws=None, nb=0, ids=B, w=C, counts=D, bal=G, zl=W, lse=X):
    return "moe_route_v1", (logits, T, E, dt, k, mask, 1, ws, nb, ids, w, counts, bal, zl, lse)


def route_b(logits=A, T=4, E=64, dt=0, k=2, ids=B, w=C, counts=D, lse=G, dw=W, db=X, dz=X + 64, dl=Y):
    return "moe_route_backward_v1", (logits, T, E, dt, k, 1, ids, w, counts, lse, dw, db, dz, dl)


def norm(x=A, T=4, H=64, dt=0, w=B, b=C, eps=1e-5, y=D, st=G):
    return "moe_layer_norm_v1", (x, T, H, dt, w, b, eps, y, st)


def norm_b(x=A, T=4, H=64, dt=0, w=B, st=C, dy=D, ws=W, nb=1 << 24, dx=G, dw=X, db=Y):
    return "moe_layer_norm_backward_v1", (x, T, H, dt, w, st, dy, ws, nb, dx, dw, db)


@pytest.mark.parametrize("code,call", [
    (UNSUP, lin(dt=2)), (UNSUP, lin(dt=-1)), (SHAPE, lin(T=-1)), (SHAPE, lin(N=60)), (SHAPE, lin(N=0)),
    (SHAPE, lin(gs=16)), (SHAPE, lin(gs=48)), (SHAPE, lin(gs=96)), (SHAPE, lin(K=192)), (SHAPE, lin(gs=512)),
    (SHAPE, lin(K=131072)), (SHAPE, lin(T=1 << 23, out=BIG)), (SHAPE, lin(K=65536, N=65536, out=BIG)),
    (SHAPE, lin(T=1 << 20, K=32, gs=32, N=8192, out=BIG)), (NULL, lin(x=None)), (NULL, lin(out=None)),
    (NULL, lin(p=proj(q=None))), (NULL, lin(p=proj(zeros=None))), (NULL, lin(p=proj(scales=None))),
    (SHAPE, lin(p=proj(q=B + 2))), (SHAPE, lin(p=proj(zeros=C + 2))), (SHAPE, lin(out=A + 64)),
    (SHAPE, lin(out=B + 64)), (SHAPE, lin(out=C)), (SHAPE, lin(out=D + 2)), (SHAPE, lin(bias=G + 8)),
    (UNSUP, route(dt=3)), (SHAPE, route(E=0)), (SHAPE, route(E=513)), (SHAPE, route(k=0)), (SHAPE, route(k=65)),
    (SHAPE, route(E=4, k=5)), (SHAPE, route(T=-1)), (SHAPE, route(T=1 << 22)), (NULL, route(logits=None)),
    (NULL, route(ids=None)), (NULL, route(w=None)), (NULL, route(counts=None)), (NULL, route(bal=None)),
    (NULL, route(zl=None)), (WS, route(T=100)), (WS, route(T=100, ws=Y + 16, nb=1 << 24)),
    (WS, route(T=100, ws=Y, nb=64)), (SHAPE, route(ids=A + 4)), (SHAPE, route(w=B + 8)),
    (SHAPE, route(counts=B)), (SHAPE, route(lse=C)), (SHAPE, route(bal=W)), (SHAPE, route(mask=B)),
    (SHAPE, route(T=100, ws=A, nb=1 << 24)),
    (NULL, route_b(logits=None)), (NULL, route_b(ids=None)), (NULL, route_b(w=None)), (NULL, route_b(counts=None)),
    (NULL, route_b(lse=None)), (NULL, route_b(dl=None)), (SHAPE, route_b(dl=A)), (SHAPE, route_b(dl=W + 8)),
    (SHAPE, route_b(dl=G)), (UNSUP, route_b(dt=4)), (SHAPE, route_b(k=99)),
    (UNSUP, norm(dt=3)), (SHAPE, norm(H=0)), (SHAPE, norm(H=8193)), (SHAPE, norm(T=-1)), (SHAPE, norm(eps=-1.0)),
    (SHAPE, norm(eps=float("nan"))), (NULL, norm(x=None)), (NULL, norm(y=None)), (SHAPE, norm(y=A)),
    (SHAPE, norm(y=B + 16)), (SHAPE, norm(st=D + 16)), (SHAPE, norm(st=A + 16)), (SHAPE, norm(st=G + 4)),
    (NULL, norm_b(x=None)), (NULL, norm_b(st=None)), (NULL, norm_b(dy=None)), (WS, norm_b(ws=None)),
    (WS, norm_b(nb=64)), (WS, norm_b(ws=W + 8)), (SHAPE, norm_b(dx=A)), (SHAPE, norm_b(dx=D + 16)),
    (SHAPE, norm_b(dw=B)), (SHAPE, norm_b(db=X + 32)), (SHAPE, norm_b(dw=W + 64)), (SHAPE, norm_b(st=C + 4)),
    (SHAPE, norm_b(H=8193)), (UNSUP, norm_b(dt=-2))])
def test_entry_points_refuse(code, call):
    entry, args = call
    assert getattr(_lib.load(), entry)(*args, None) == code, _lib.load().moe_w4a16_last_error()


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    for entry, args in (lin(T=0, x=None, out=None), norm(T=0, x=None, y=None),
                        norm_b(T=0, x=None, st=None, dy=None, dw=None, db=None),
                        norm_b(dx=None, dw=None, db=None, ws=None, nb=0),
                        route_b(T=0, logits=None, ids=None, w=None, counts=None, lse=None, dl=None)):
        assert getattr(lib, entry)(*args, None) == 0, lib.moe_w4a16_last_error()


def test_workspace_queries():
    lib = _lib.load()
    assert lib.moe_int4_linear_workspace_bytes_v1(-1, 256, 64, 128) == -1
    assert lib.moe_int4_linear_workspace_bytes_v1(4, 200, 64, 128) == -1
    assert lib.moe_int4_linear_workspace_bytes_v1(4, 256, 64, 128) >= 0
    assert lib.moe_route_workspace_bytes_v1(4, 0) == lib.moe_route_workspace_bytes_v1(-1, 8) == -1
    assert lib.moe_route_workspace_bytes_v1(4, 513) == -1 and lib.moe_route_workspace_bytes_v1(4, 8) == 0
    most = lib.moe_route_workspace_bytes_v1(2 ** 31 - 1, 512)
    assert most == lib.moe_route_workspace_bytes_v1(1 << 20, 512) > 0
    query = lib.moe_layer_norm_workspace_bytes_v1
    assert query(-1, 64) == query(4, 0) == query(4, 8193) == -1
    for hidden in (8, 512, 513, 8192):
        assert query(2 ** 31 - 1, hidden) == query(1 << 20, hidden) > query(1, hidden) > 0


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    monkeypatch.setattr(ops, "_call", lambda entry, device, *args: None)


def linear(t, name):
    at = {"x": (4, 128), "scales": (1, 16), "bias": (16,)}
    at = {n: t(*s).half() if n == name else torch.ones(s, dtype=HALF) for n, s in at.items()}
    return ops.int4_linear(at["x"], z(16, 16, dtype=I), z(1, 2, dtype=I), at["scales"], bias=at["bias"])


def layer_norm(t, name):
    at = {"x": (4, 32), "weight": (32,), "bias": (32,)}
    return ops.layer_norm(**{n: t(*s) if n == name else torch.ones(s) for n, s in at.items()})


DIFFERENTIABLE = {**{f"layer_norm {n}": (lambda t, n=n: layer_norm(t, n)) for n in ("x", "weight", "bias")},
                  "route logits": lambda t: ops.route_tokens(t(4, 32), 2).topk_weights}
NOT = {f"int4_linear {n}": (lambda t, n=n: linear(t, n)) for n in ("x", "scales", "bias")}


def leaf(*shape):
    return torch.ones(*shape, requires_grad=True)


@pytest.mark.parametrize("name", [*DIFFERENTIABLE, *NOT])
def test_forward_mode_is_refused(name, no_launch):
    call = {**DIFFERENTIABLE, **NOT}[name]
    with fwd.dual_level():
        dual = lambda *shape: fwd.make_dual(torch.ones(*shape), torch.ones(*shape))  # noqa: E731
        for grads in (torch.enable_grad(), torch.no_grad()):
            with grads, pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                call(dual)
        call(torch.ones)


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_gradients_are_recorded_where_wanted(name, no_launch):
    call = DIFFERENTIABLE[name]
    assert call(leaf).requires_grad and not call(torch.ones).requires_grad
    with torch.no_grad():
        assert not call(leaf).requires_grad


@pytest.mark.parametrize("name", ["layer_norm x", "route logits"])
def test_forward_mode_of_a_backward_pass_is_refused(name, no_launch):
    leaves = []
    out = DIFFERENTIABLE[name](lambda *s: leaves.append(leaf(*s)) or leaves[-1])
    one = torch.ones_like(out)
    with fwd.dual_level():
        torch.autograd.grad(out, leaves, one, retain_graph=True)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(out, leaves, fwd.make_dual(one, one))


@pytest.mark.parametrize("name", NOT)
def test_a_gradient_that_does_not_exist_is_an_error(name, no_launch):
    out = NOT[name](leaf)
    assert out.requires_grad
    with pytest.raises(NotImplementedError, match="int4_linear"):
        out.float().sum().backward()
    assert not NOT[name](torch.ones).requires_grad


def test_routing_ids_and_counts_carry_no_gradient(no_launch):
    r = ops.route_tokens(leaf(4, 32), 2)
    assert r.topk_weights.requires_grad and r.balance_loss.requires_grad and r.z_loss.requires_grad
    assert not r.topk_ids.requires_grad and not r.counts.requires_grad


def test_ctypes_structs_are_taken_by_reference():
    entry, args = lin(T=0)
    assert getattr(_lib.load(), entry)(*args[:4], ctypes.byref(args[4]), *args[5:], None) == 0
