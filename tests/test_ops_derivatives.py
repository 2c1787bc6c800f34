"""No operator beside the int4 path drops a derivative in silence. What it asks of autograd does not
depend on the kernels, so these run on host tensors with the entry points left out."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mtp_amd import ops


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu", lambda *tensors: None)
    monkeypatch.setattr(ops, "_call", lambda entry, device, *args: None)


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
