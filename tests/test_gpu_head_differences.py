"""The draft-head gradients against differences of the losses, tightly enough that a gradient that
is off by a tenth fails, at temperatures other than 1 too.

Inputs lie on grids on which X + d u and W + d U are exact in bf16 (at most 256 steps of the grid
from 0). The direction u is the sign of the gradient itself, so that what is compared is the
gradient's 1-norm. A central difference over 2 d is off by
  * d^2 / 6 times the third derivative along u: the third cumulant of the logits' own movement
    under p, at most sqrt(3) / 18 R^3 for a movement whose values span R;
  * the losses' own bounds, twice, over 2 d.
The gradient is off by its bound in every element (test_gpu_head.formula, which takes only sizes
and magnitudes for it). Together they are 1 to 3% of the norm."""
import math
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
sys.path.insert(0, os.path.dirname(HERE))
from k3lib import load  # noqa: E402
from test_gpu_head import formula, targets_distill, targets_xent  # noqa: E402

pytestmark = pytest.mark.gpu

T, N, VOCAB, K = 24, 64, 500, 5
STEP_X, STEP_W = 2.0 ** -6, 2.0 ** -10


@pytest.fixture(scope="module")
def k3():
    return load()


def case(k3, temp):
    """X, W, g; the loss and lse of (X, W); the gradients; the 64-bit values with their bounds."""
    gen = torch.Generator(device="cuda").manual_seed(31)
    X = (torch.randint(-120, 121, (T, N), generator=gen, device="cuda") * STEP_X).bfloat16()
    W = (torch.randint(-130, 131, (VOCAB, N), generator=gen, device="cuda") * STEP_W).bfloat16()
    g = torch.rand(T, generator=gen, device="cuda") + 0.5
    if temp is None:
        label = torch.randint(0, VOCAB, (T,), generator=gen, device="cuda").int()
        return (X, W, g, lambda x, w: k3.lm_head_xent(x, w, label),
                lambda x, w, lse: k3.lm_head_xent_grad(x, w, label, lse, g=g),
                lambda x, w: formula(x, w, targets_xent(label, VOCAB), 1.0, g))
    ids = torch.randint(0, VOCAB, (T, K), generator=gen, device="cuda").int()
    top = torch.randn((T, K), generator=gen, device="cuda")
    return (X, W, g, lambda x, w: k3.lm_head_distill(x, w, ids, top, temp=temp),
            lambda x, w, lse: k3.lm_head_distill_grad(x, w, ids, top, lse, temp=temp, g=g),
            lambda x, w: formula(x, w, targets_distill(ids, top, temp, VOCAB), temp, g))


def third(span):
    return math.sqrt(3) / 18 * span ** 3


@pytest.mark.parametrize("temp", [None, 1.0, 0.5, 2.5])     # None: cross entropy
def test_dx(k3, temp):
    X, W, g, loss, grad, exact = case(k3, temp)
    dX = grad(X, W, loss(X, W)[1])[0].double()
    u = dX.sign()
    up, down = (X.double() + STEP_X * u).bfloat16(), (X.double() - STEP_X * u).bfloat16()
    assert torch.equal(up.double() - X.double(), STEP_X * u) and torch.equal(X.double() - down.double(), STEP_X * u)
    got = (loss(up, W)[0].double() - loss(down, W)[0].double()) * g.double() / (2 * STEP_X)
    want = (dX * u).sum(1)
    move = u @ W.double().T / (temp or 1.0)
    bounds = torch.maximum(exact(up, W)["loss"][1], exact(down, W)["loss"][1])
    tol = g.double() * (STEP_X ** 2 / 6 * third(move.amax(1) - move.amin(1)) + bounds / STEP_X)
    tol += exact(X, W)["dX"][1].sum(1)
    assert bool(((got - want).abs() <= tol).all())
    for k in (0.0, 0.9, 1.1):                                   # what is to fail does
        assert bool(((got - k * want).abs() > tol).all())


@pytest.mark.parametrize("temp", [None, 1.0, 0.5, 2.5])
def test_dw(k3, temp):
    X, W, g, loss, grad, exact = case(k3, temp)
    dW = grad(X, W, loss(X, W)[1])[1].double()
    U = dW.sign()
    up, down = (W.double() + STEP_W * U).bfloat16(), (W.double() - STEP_W * U).bfloat16()
    assert torch.equal(up.double() - W.double(), STEP_W * U) and torch.equal(W.double() - down.double(), STEP_W * U)
    got = float(((loss(X, up)[0].double() - loss(X, down)[0].double()) * g.double()).sum() / (2 * STEP_W))
    want = float((dW * U).sum())
    move = X.double() @ U.T / (temp or 1.0)
    bounds = torch.maximum(exact(X, up)["loss"][1], exact(X, down)["loss"][1])
    tol = float((g.double() * (STEP_W ** 2 / 6 * third(move.amax(1) - move.amin(1)) + bounds / STEP_W)).sum())
    tol += float(exact(X, W)["dW"][1].sum())
    assert abs(got - want) <= tol
    for k in (0.0, 0.9, 1.1):
        assert abs(got - k * want) > tol
