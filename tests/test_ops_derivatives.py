"""No operator beside the int4 path drops a derivative in silence. What it asks of autograd does not
depend on the kernels, so these run on host tensors with the entry points left out."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mtp_amd import ops
from mtp_amd.weights import Int8Experts


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    monkeypatch.setattr(ops, "_call", lambda entry, device, *args: None)
    monkeypatch.setattr(ops, "_workspace", lambda workspace, need, device: torch.empty(1))


T, H, E, K = 4, 32, 8, 2
IDS = torch.zeros(T, K, dtype=torch.int32)


def block_norm(t, name):
    at = {"y": (T, H), "res": (T, H), "post_w": (H,), "gate": (H,), "pre_w": (H,)}
    at = {n: torch.ones(s) for n, s in at.items()}
    return ops.block_norm(**{**at, name: t(*at[name].shape)})


DIFFERENTIABLE = {
    "dispatch x": lambda t: ops.dispatch_tokens(t(T, H), IDS, E),
    "combine rows": lambda t: ops.combine_tokens(t(T * K, H), IDS, torch.ones(T, K)),
    "combine weights": lambda t: ops.combine_tokens(torch.ones(T * K, H), IDS, t(T, K)),
    **{f"norm {n}": (lambda t, n=n: block_norm(t, n)) for n in ("y", "res", "post_w", "gate", "pre_w")}}


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_forward_mode_is_refused(name):
    """The operators have a backward pass and no forward-mode derivative: a dual tensor is refused,
    whether gradients are on or off, and not handed on without its tangent."""
    call = DIFFERENTIABLE[name]
    with fwd.dual_level():
        dual = lambda *shape: fwd.make_dual(torch.ones(*shape), torch.ones(*shape))  # noqa: E731
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(dual)
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(dual)
        call(torch.ones)  # other tensors are taken there as everywhere


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_function_transforms_are_refused(name):
    """torch.func's transforms, which the autograd functions do not take part in."""
    call = DIFFERENTIABLE[name]
    shape = []
    call(lambda *s: (shape.extend(s), torch.ones(*s))[1])
    x = torch.ones(*shape)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: call(lambda *s: v), (x,), (x,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: call(lambda *s: v)[0].sum())(x)


@pytest.mark.parametrize("name", ["dispatch x", "combine rows", "norm y"])
def test_forward_mode_of_a_backward_pass_is_refused(name):
    leaves = []
    out = DIFFERENTIABLE[name](lambda *s: leaves.append(torch.ones(*s, requires_grad=True)) or leaves[-1])
    out = out[0] if isinstance(out, tuple) else out
    one = torch.ones_like(out)
    with fwd.dual_level():
        torch.autograd.grad(out, leaves, one, retain_graph=True)
        with pytest.raises(NotImplementedError, match="jvp"):
            torch.autograd.grad(out, leaves, fwd.make_dual(one, one))


@pytest.mark.parametrize("name", DIFFERENTIABLE)
def test_only_wanted_gradients_are_recorded(name):
    call = DIFFERENTIABLE[name]
    leaf = lambda *shape: torch.ones(*shape, requires_grad=True)  # noqa: E731

    def first(out):
        return out[0] if isinstance(out, tuple) else out

    assert first(call(leaf)).requires_grad or (name == "norm pre_w" and call(leaf)[1].requires_grad)
    assert not first(call(torch.ones)).requires_grad
    with torch.no_grad():
        assert not first(call(leaf)).requires_grad


def int8(*shape):
    return torch.ones(*shape, dtype=torch.int8)


def experts(t, name):
    at = {"x": (T, H), "topk_weights": (T, K), "gate_scale": (E, 16), "up_scale": (E, 16),
          "down_scale": (E, H)}
    at = {n: t(*s) if n == name else torch.ones(s) for n, s in at.items()}
    ex = Int8Experts(int8(E, 16, H), at["gate_scale"], int8(E, 16, H), at["up_scale"], int8(E, H, 16),
                     at["down_scale"])
    return ops.int8_experts(at["x"], IDS, at["topk_weights"], ex, workspace=None)


NOT_DIFFERENTIABLE = {
    "quantize x": lambda t: ops.quantize_tokens(t(T, H))[1],
    "matmul q_scale": lambda t: ops.int8_matmul(int8(T, H), t(T), int8(16, H), torch.ones(16)),
    "matmul weight_scale": lambda t: ops.int8_matmul(int8(T, H), torch.ones(T), int8(16, H), t(16)),
    "matmul bias": lambda t: ops.int8_matmul(int8(T, H), torch.ones(T), int8(16, H), torch.ones(16),
                                             bias=t(16), dtype=torch.float32),
    "linear x": lambda t: ops.int8_linear(t(T, H), int8(16, H), torch.ones(16)),
    "linear weight_scale": lambda t: ops.int8_linear(torch.ones(T, H), int8(16, H), t(16)),
    "linear bias": lambda t: ops.int8_linear(torch.ones(T, H), int8(16, H), torch.ones(16), bias=t(16)),
    **{f"experts {n}": (lambda t, n=n: experts(t, n))
       for n in ("x", "topk_weights", "gate_scale", "up_scale", "down_scale")}}


@pytest.mark.parametrize("name", NOT_DIFFERENTIABLE)
def test_a_gradient_that_does_not_exist_is_an_error(name):
    """The int8 products have no gradient. The call itself runs, as inference without no_grad does; a
    backward pass that reaches it raises instead of going on without what lies ahead of it."""
    call = NOT_DIFFERENTIABLE[name]
    leaf = lambda *shape: torch.ones(*shape, requires_grad=True)  # noqa: E731
    out = call(leaf)
    assert out.requires_grad and not out._is_view()
    with pytest.raises(NotImplementedError, match=name.split()[0]):
        out.float().sum().backward()
    assert not call(torch.ones).requires_grad
    with torch.no_grad():
        assert not call(leaf).requires_grad
    assert not call(lambda *shape: leaf(*shape).detach()).requires_grad


@pytest.mark.parametrize("name", NOT_DIFFERENTIABLE)
def test_forward_mode_of_the_int8_products_is_refused(name):
    call = NOT_DIFFERENTIABLE[name]
    with fwd.dual_level():
        dual = lambda *shape: fwd.make_dual(torch.ones(*shape), torch.ones(*shape))  # noqa: E731
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(dual)
        assert not call(torch.ones).requires_grad


def test_quantising_stacks_records_no_gradient():
    """Weights are often parameters; quantising them is no part of a graph."""
    w = torch.ones(E, 16, H, requires_grad=True)
    ex = Int8Experts.from_dense(w, w, torch.ones(E, H, 16, requires_grad=True))
    assert not ex.gate_scale.requires_grad and not ex.down_scale.requires_grad
