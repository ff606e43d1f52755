"""Forward-mode derivatives of ``dr.group_norm`` and ``dr.dropout``: neither has them, and a call
whose input carries a tangent says so instead of returning a result without one. Checked on the
CPU, with stand-ins for the kernels."""

import contextlib

import pytest
import torch
from torch.autograd import forward_ad

import diffrast_b200 as dr
from diffrast_b200 import _kernels as K
from diffrast_b200 import ops

X, Y = torch.randn(2, 3, 3, 4), torch.randn(2, 3, 3, 4)
W, B = torch.rand(4) + 0.5, torch.randn(4)

# Calls by the input that may carry a tangent.
CALLS = {
    "norm x": (X, lambda t: dr.group_norm(t, 2, W, B, activation="silu")),
    "norm x alone": (X, lambda t: dr.group_norm(t, 2)),
    "norm weight": (W, lambda t: dr.group_norm(X, 2, t, B)),
    "norm bias": (B, lambda t: dr.group_norm(X, 2, None, t, dropout=0.5, seed=1)),
    "dropout x": (X, lambda t: dr.dropout(t, 0.5, 1)),
    "dropout x beside residual": (X, lambda t: dr.dropout(t, 0.5, 1, residual=Y)),
    "dropout residual": (Y, lambda t: dr.dropout(X, 0.5, 1, residual=t)),
}


@pytest.fixture
def stand_ins(monkeypatch):
    monkeypatch.setattr(ops, "require_cuda", lambda device: None)
    monkeypatch.setattr(ops, "_on_device", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(K, "group_norm_fwd", lambda x, *rest: (x.detach().clone(), torch.empty(1)))
    monkeypatch.setattr(K, "dropout", lambda x, *rest: x.detach().clone())


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [False, True], ids=["no_grad", "grad"])
def test_tangents_are_refused(stand_ins, name, grad):
    primal, call = CALLS[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(primal, torch.ones_like(primal)))


@pytest.mark.parametrize("name", CALLS)
def test_calls_without_tangents_pass_beside_them(stand_ins, name):
    primal, call = CALLS[name]
    with forward_ad.dual_level():
        forward_ad.make_dual(torch.ones(3), torch.ones(3))
        assert forward_ad.unpack_dual(call(primal)).tangent is None
        leaf = primal.clone().requires_grad_(True)
        assert call(leaf).requires_grad
    assert call(primal).shape == X.shape


def gradient(monkeypatch, name):
    """The gradient, for an upstream gradient that carries a tangent."""
    monkeypatch.setattr(K, "group_norm_bwd", lambda x, g, *rest: (g.detach().clone(), None, None))
    primal, call = CALLS[name]
    leaf = primal.clone().requires_grad_(True)
    y = call(leaf)
    return torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))[0]


@pytest.mark.parametrize("name", ["norm x", "norm x alone", "dropout x", "dropout x beside residual"])
def test_tangents_of_the_upstream_gradient_are_refused(stand_ins, monkeypatch, name):
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        gradient(monkeypatch, name)


def test_the_residuals_gradient_keeps_its_tangent(stand_ins, monkeypatch):
    """It is the upstream gradient itself."""
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(gradient(monkeypatch, "dropout residual")).tangent
    assert torch.equal(tangent, torch.ones_like(X))
