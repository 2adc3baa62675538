"""The draft-head gradients of up to 32 rows: dz enters the products in two bf16 parts, so that the
outputs' own rounding is all that bf16 costs them.

Tolerances as in test_gpu_head's docstring, with the two parts in dz's place: the first is off by at
most 2^-8 of the value, and the second, the rest, by 2^-8 of that: 2^-16 |dz|. On inputs like these
one rounding alone is off by more where a sum cancels."""
import math
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
sys.path.insert(0, os.path.dirname(HERE))
from k3lib import load  # noqa: E402
from test_gpu_head import distill_all, holds, inputs, targets_distill, targets_xent, xent_all  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k3():
    return load()


def gradients(X, W, tgt, temp, g, off):
    """dX and dW in 64 bits with their bounds; `off` bounds dz's own rounding, relative."""
    ids, q, ent, live = tgt
    Xd, Wd = torch.where(live[:, None], X.double(), 0.0), W.double()
    n, vocab, T = X.shape[1], W.shape[0], X.shape[0]
    z = (Xd @ Wd.T) / temp
    ez = ((n / 16 + 16) * 2.0 ** -23 * (Xd.abs() @ Wd.abs().T) / temp).amax(1)
    lse = torch.logsumexp(z, 1)
    mag = lse.abs() + z.abs().amax(1) + torch.as_tensor(ent, device=z.device).abs() + 1
    p = (z - lse[:, None]).exp()
    gt = (g.double() / temp * live.double())[:, None]
    dz = gt * p.clone().scatter_add_(1, ids, -q)
    b_p = (2 * ez + 2.0 ** -20)[:, None] + 2.0 ** -19 * (z.abs() + mag[:, None])
    b = dz.abs() * off + gt.abs() * p * b_p
    b += gt.abs() * torch.zeros_like(p).scatter_add_(1, ids, q) * 2.0 ** -22
    dX, dW = dz @ Wd, dz.T @ Xd
    b_dX = b @ Wd.abs() + (vocab + 16) * 2.0 ** -23 * (dz.abs() @ Wd.abs()) + dX.abs() * 2.0 ** -8
    b_dW = b.T @ Xd.abs() + (T + 16) * 2.0 ** -23 * (dz.abs().T @ Xd.abs()) + dW.abs() * 2.0 ** -8
    return {"dX": (dX, b_dX), "dW": (dW, b_dW)}, (dz, Xd)


# one split and no vocabulary to split, many splits, two pieces of it; X read in place (10 rows)
@pytest.mark.parametrize("T,n,vocab", [(1, 8, 1), (1, 264, 3001), (4, 2968, 9000), (31, 72, 255), (32, 136, 257),
                                       (17, 520, 1000), (32, 1024, 3001), (10, 7168, 2000), (9, 64, 270000),
                                       (30, 64, 270000)])
@pytest.mark.parametrize("K,temp", [(0, 1.0), (2, 2.0), (7, 0.5)])
def test_two_parts(k3, T, n, vocab, K, temp):
    X, W, g, gen = inputs(T, n, vocab, T * 5 + n + vocab + K)
    if K:
        ids = torch.randint(0, vocab, (T, K), generator=gen, device="cuda").int()
        top = torch.randn((T, K), generator=gen, device="cuda")
        if T > 3 and T != 10:
            ids[T // 2] = -1
        got, tgt = distill_all(k3, X, W, ids, top, temp, g), targets_distill(ids, top, temp, vocab)
    else:
        label = torch.randint(0, vocab, (T,), generator=gen, device="cuda").int()
        if T > 3 and T != 10:
            label[::3] = -1
        got, tgt = xent_all(k3, X, W, label, g), targets_xent(label, vocab)
    want, (dz, Xd) = gradients(X, W, tgt, temp, g, 2.0 ** -16)
    for name in want:
        holds(name, got[name], want[name])
    if vocab > 1000:
        # a dz rounded once is outside these bounds, so the test would see one
        once = (dz.float().bfloat16().double().T @ Xd).bfloat16().double()
        assert bool(((once - want["dW"][0]).abs() > want["dW"][1]).any())
    assert k3.device_status(0) == 0


def test_the_error_is_the_outputs_rounding(k3):
    """4 rows of 2 entries over 163,840 ids, where one rounding of dz shows whole (0.0025 of the
    norm): in the norm an error of a rounding to bf16 (at most 2^-8, 0.0017 for mantissas as they come)
    with a tenth to spare."""
    X, W, g, gen = inputs(4, 2968, 163840, 9)
    ids = torch.randint(0, 163840, (4, 2), generator=gen, device="cuda").int()
    top = torch.tensor([[0.0, math.log(2.0)]] * 4, device="cuda")         # masses of 1/3 and 2/3
    got = distill_all(k3, X, W, ids, top, 1.0, torch.ones_like(g))
    want, _ = gradients(X, W, targets_distill(ids, top, 1.0, 163840), 1.0, torch.ones_like(g), 2.0 ** -16)
    for name in want:
        value = want[name][0]
        rounded = float((value.bfloat16().double() - value).norm())
        assert float((got[name].double() - value).norm()) < 1.1 * rounded, name


def test_unbounded_weights_stay_in_their_row(k3):
    """An infinite weight, and one at the end of fp32: the other rows' dX are what they are without."""
    X, W, _, gen = inputs(20, 64, 300, 10)
    label = torch.randint(0, 300, (20,), generator=gen, device="cuda").int()
    g = torch.rand(20, generator=gen, device="cuda") + 0.5
    g[3] = math.inf
    got = xent_all(k3, X, W, label, g)["dX"]
    g2 = g.clone()
    g2[3] = 1.0
    tgt = targets_xent(label, 300)
    want, _ = gradients(X, W, tgt, 1.0, g2, 2.0 ** -16)
    other = torch.arange(20, device="cuda") != 3
    holds("dX", got[other], (want["dX"][0][other], want["dX"][1][other]))
    assert not bool(torch.isfinite(got[3]).any())
