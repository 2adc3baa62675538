"""The draft-head losses (k3gpu_lm_head_xent, k3gpu_lm_head_distill and their gradients)
against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic the header states. Products of bf16
pairs are exact. A product's fp32 sum of n terms takes at most n additions, each off by at
most 2^-23 of the partial sum, which sum |x w| =: S bounds; the tensor core adds 16 products
a step, so ez = (n / 16 + 16) 2^-23 S bounds a logit's error. Then, with one temperature:
  lse, loss   off by at most max ez (a softmax moves by no more than its logits do), twice for
              the loss, plus 2^-21 of the magnitudes for the scaling by log2 e and the exp2
  p           relative: 2 max ez + 2^-19 |z| (argument rounding of the exp2) + 2^-20
  dz          |dz| 2^-8 (one bf16 rounding) + that times p
  dX, dW      the sum of their terms' errors, the sums' own (n + 16) 2^-23 sum |.|, and the bf16
              rounding of the output, 2^-8 of it
"""
import math
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
sys.path.insert(0, os.path.dirname(HERE))
from k3lib import load  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k3():
    return load()


def inputs(T, n, vocab, seed, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    X = torch.randn((T, n), generator=gen, device="cuda").bfloat16()
    W = (torch.randn((vocab, n), generator=gen, device="cuda") * (spread / math.sqrt(n))).bfloat16()
    g = torch.rand(T, generator=gen, device="cuda") * 2 - 0.5
    return X, W, g, gen


def targets_xent(label, vocab):
    """(ids, mass, entropy, live) of labels: one entry of mass 1."""
    live = (label >= 0) & (label < vocab)
    return label.long().clamp(0, vocab - 1)[:, None], live.double()[:, None], 0.0, live


def targets_distill(ids, top, temp, vocab):
    ok = (ids >= 0) & (ids < vocab) & (top != -math.inf)
    live = ok.any(1)
    t = torch.where(ok, top.double(), -math.inf)
    t = (t - torch.where(live, t.amax(1), 0.0)[:, None]) / temp
    e = torch.where(ok, t.exp(), 0.0)
    s = e.sum(1, keepdim=True)
    q = torch.where(live[:, None], e / s, 0.0)
    ent = torch.where(q > 0, q * (t - s.log()), 0.0).sum(1)
    return ids.long().clamp(0, vocab - 1), q, torch.where(live, ent, 0.0), live


def formula(X, W, tgt, temp, g):
    """Everything in 64 bits, and the bounds of the module's docstring."""
    ids, q, ent, live = tgt
    lv = live.double()
    Xd = torch.where(live[:, None], X.double(), 0.0)
    Wd = W.double()
    n, vocab, T = X.shape[1], W.shape[0], X.shape[0]
    z = (Xd @ Wd.T) / temp
    S = (Xd.abs() @ Wd.abs().T) / temp
    ez = (n / 16 + 16) * 2.0 ** -23 * S
    ez1 = ez.amax(1)
    lse = torch.logsumexp(z, 1)
    zt = (q * z.gather(1, ids)).sum(1)
    loss = (ent + lse - zt) * lv
    mag = lse.abs() + z.abs().amax(1) + torch.as_tensor(ent, device=z.device).abs() + 1
    b_lse = ez1 + 2.0 ** -21 * mag
    b_loss = 2 * ez1 + 2.0 ** -21 * mag
    p = (z - lse[:, None]).exp()
    dz = p.clone().scatter_add_(1, ids, -q)
    gt = (g.double() / temp * lv)[:, None]
    dz *= gt
    b_p = (2 * ez1 + 2.0 ** -20)[:, None] + 2.0 ** -19 * (z.abs() + mag[:, None])
    b_dz = dz.abs() * 2.0 ** -8 + gt.abs() * p * b_p
    b_dz += gt.abs() * torch.zeros_like(p).scatter_add_(1, ids, q) * 2.0 ** -22
    dX, dW = dz @ Wd, dz.T @ Xd
    b_dX = b_dz @ Wd.abs() + (vocab + 16) * 2.0 ** -23 * (dz.abs() @ Wd.abs()) + dX.abs() * 2.0 ** -8
    b_dW = b_dz.T @ Xd.abs() + (T + 16) * 2.0 ** -23 * (dz.abs().T @ Xd.abs()) + dW.abs() * 2.0 ** -8
    return {"loss": (loss, b_loss), "lse": (lse * lv, b_lse), "dX": (dX, b_dX), "dW": (dW, b_dW)}


def holds(name, got, want):
    value, bound = want
    assert got.shape == value.shape
    off = (got.double() - value).abs()
    assert bool(torch.isfinite(got).all()), name
    worst = float((off - bound).max())
    assert worst <= 1e-40, (name, worst, float(off.max()))          # (half a step of bf16's smallest values)


def xent_all(k3, X, W, label, g, **kw):
    loss, lse = k3.lm_head_xent(X, W, label)
    dX, dW = k3.lm_head_xent_grad(X, W, label, lse, g=g, **kw)
    return {"loss": loss, "lse": lse, "dX": dX, "dW": dW}


def distill_all(k3, X, W, ids, top, temp, g, **kw):
    loss, lse = k3.lm_head_distill(X, W, ids, top, temp=temp)
    dX, dW = k3.lm_head_distill_grad(X, W, ids, top, lse, temp=temp, g=g, **kw)
    return {"loss": loss, "lse": lse, "dX": dX, "dW": dW}


# one token, one id, one 16-byte row; edges of the tiles (128, 256, 64) on each side; several
# pieces of the vocabulary (the last three), worked on by single CTAs and by pairs
SIZES = [(1, 8, 1), (1, 64, 1000), (3, 72, 255), (129, 136, 257), (128, 64, 256), (257, 512, 1024), (300, 1000, 3001),
         (40, 7168, 2000), (520, 64, 100003), (16389, 64, 5000), (8200, 200, 10007)]


@pytest.mark.parametrize("T,n,vocab", SIZES)
@pytest.mark.parametrize("masked", [0.0, 0.4])
def test_xent(k3, T, n, vocab, masked):
    X, W, g, gen = inputs(T, n, vocab, T * 7 + n + vocab)
    label = torch.randint(0, vocab, (T,), generator=gen, device="cuda")
    label = torch.where(torch.rand(T, generator=gen, device="cuda") < masked, -100, label).int()
    got = xent_all(k3, X, W, label, g)
    want = formula(X, W, targets_xent(label, vocab), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    assert k3.device_status(0) == 0


@pytest.mark.parametrize("T,n,vocab,K,temp", [(1, 8, 1, 1, 1.0), (1, 64, 1000, 128, 2.0), (130, 136, 257, 7, 0.5),
                                              (300, 1000, 3001, 64, 1.0), (257, 72, 5, 33, 1.5),
                                              (8200, 200, 10007, 16, 3.0)])
def test_distill(k3, T, n, vocab, K, temp):
    """Entries in any order, doubled ids (vocab 5 has nothing else), empty entries, rows without any."""
    X, W, g, gen = inputs(T, n, vocab, T + n + vocab + K)
    ids = torch.randint(0, vocab, (T, K), generator=gen, device="cuda")
    top = torch.randn((T, K), generator=gen, device="cuda") * 3 + 5
    ids = torch.where(torch.rand((T, K), generator=gen, device="cuda") < 0.1, -1, ids)
    if T > 2:
        ids[T // 2] = -1
        top[T // 3] = -math.inf
    top[0, 0] = -math.inf if K > 1 else 0.25
    ids = ids.int()
    got = distill_all(k3, X, W, ids, top, temp, g)
    want = formula(X, W, targets_distill(ids, top, temp, vocab), temp, g)
    for name in want:
        holds(name, got[name], want[name])
    assert k3.device_status(0) == 0


def test_distill_of_one_entry_is_xent(k3):
    """K = 1 has mass 1 whatever its logit: the same numbers as the cross entropy."""
    X, W, g, gen = inputs(70, 256, 900, 3)
    label = torch.randint(-1, 900, (70,), generator=gen, device="cuda").int()
    a = xent_all(k3, X, W, label, g)
    top = torch.randn((70, 1), generator=gen, device="cuda") * 50
    b = distill_all(k3, X, W, label[:, None].contiguous(), top, 1.0, g)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_teacher_of_lowest_values(k3):
    """Teacher logits of the type's lowest value: alone they share the mass; beside a larger one
    they get none of it, though their distance from it overflows at a low temperature."""
    X, W, g, gen = inputs(2, 64, 100, 4)
    low = torch.finfo(torch.float32).min
    ids = torch.tensor([[3, 7, 11, 13], [3, 7, 11, 13]], dtype=torch.int32, device="cuda")
    top = torch.tensor([[low] * 4, [low, 1.0, low, 2.0]], device="cuda")
    got = distill_all(k3, X, W, ids, top, 0.25, g)
    want = formula(X, W, targets_distill(ids, top, 0.25, 100), 0.25, g)
    for name in want:
        holds(name, got[name], want[name])


@pytest.mark.parametrize("n", [0, 1])
def test_rows_without_target(k3, n):
    """None (or one) of the rows has a target: zeros, whatever NaN the others hold."""
    X, W, g, gen = inputs(150, 128, 700, 5)
    label = torch.full((150,), -1, dtype=torch.int32, device="cuda")
    keep = torch.zeros(150, dtype=torch.bool, device="cuda")
    if n:
        label[77], keep[77] = 699, True
    Xn = torch.where(keep[:, None], X, torch.full_like(X, float("nan")))
    got = xent_all(k3, Xn, W, label, torch.where(keep, g, torch.full_like(g, float("nan"))))
    want = formula(X, W, targets_xent(label, 700), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    for name in ("loss", "lse", "dX"):
        assert (got[name][~keep] == 0).all()


def test_out_of_range_targets_are_flagged_and_left_out(k3):
    X, W, g, gen = inputs(20, 64, 300, 6)
    label = torch.arange(20, dtype=torch.int32, device="cuda")
    label[4], label[9] = 300, 2 ** 31 - 1
    k3.device_status(0)
    got = xent_all(k3, X, W, label, g)
    assert k3.device_status(0) == 1
    want = formula(X, W, targets_xent(label, 300), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    ids = torch.stack([label, torch.full_like(label, 7)], 1)
    top = torch.ones((20, 2), device="cuda")
    got = distill_all(k3, X, W, ids, top, 1.0, g)
    assert k3.device_status(0) == 1
    want = formula(X, W, targets_distill(ids, top, 1.0, 300), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])


def test_nan_stays_in_its_row(k3):
    """A NaN hidden state or teacher logit of a row that counts: its loss and dX are NaN, the
    other rows' are what they are without it."""
    X, W, g, gen = inputs(33, 64, 600, 7)
    label = torch.randint(0, 600, (33,), generator=gen, device="cuda").int()
    clean = xent_all(k3, X, W, label, g)
    X2 = X.clone()
    X2[5, 3] = float("nan")
    got = xent_all(k3, X2, W, label, g, need_dw=False)
    other = torch.arange(33, device="cuda") != 5
    for name in ("loss", "lse", "dX"):
        assert torch.isnan(got[name][5]).all()
        assert torch.equal(got[name][other], clean[name][other])
    top = torch.randn((33, 4), generator=gen, device="cuda")
    ids = torch.randint(0, 600, (33, 4), generator=gen, device="cuda").int()
    clean = distill_all(k3, X, W, ids, top, 1.0, g)
    for bad in (float("nan"), math.inf):
        top2 = top.clone()
        top2[8, 2] = bad
        got = distill_all(k3, X, W, ids, top2, 1.0, g, need_dw=False)
        assert torch.isnan(got["loss"][8])
        other = torch.arange(33, device="cuda") != 8
        for name in ("loss", "lse", "dX"):
            assert torch.equal(got[name][other], clean[name][other])


@pytest.mark.parametrize("masked", [False, True])
def test_strided_and_unaligned_hidden_states(k3, masked):
    """X a slice of wider rows: at an aligned stride it is read in place, at an odd one it is
    packed first; the numbers do not change. Nothing beside the slice is read."""
    X, W, g, gen = inputs(140, 200, 400, 8)
    label = torch.randint(0, 400, (140,), generator=gen, device="cuda").int()
    if masked:
        label[::3] = -1
    base = xent_all(k3, X, W, label, g)
    for width, off in ((208, 8), (211, 5), (203, 0)):
        wide = torch.full((140, width), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, off:off + 200] = X
        got = xent_all(k3, wide[:, off:off + 200], W, label, g)
        for name in base:
            assert torch.equal(got[name], base[name]), (name, width, off)


def test_strided_dx_leaves_its_neighbours(k3):
    """dX into a slice of a wider buffer, aligned and not: only the slice is written."""
    X, W, g, gen = inputs(140, 72, 300, 9)
    label = torch.randint(-1, 300, (140,), generator=gen, device="cuda").int()
    _, lse = k3.lm_head_xent(X, W, label)
    want, _ = k3.lm_head_xent_grad(X, W, label, lse, g=g, need_dw=False)
    lib = k3.lib
    ws = k3.workspace(lib.k3gpu_lm_head_xent_workspace(140, 72, 300))
    for width, off in ((80, 8), (77, 3)):
        wide = torch.full((140, width), 7.0, dtype=torch.bfloat16, device="cuda")
        part = wide[:, off:off + 72]
        k3.check(lib.k3gpu_lm_head_xent_grad(part.data_ptr(), width, None, k3.ptr(g), k3.ptr(lse), k3.ptr(X), 72,
                                             k3.ptr(W), k3.ptr(label), 72, 300, 140, k3.ptr(ws), ws.numel(),
                                             k3.stream_ptr()))
        assert torch.equal(part, want)
        assert (wide[:, :off] == 7).all() and (wide[:, off + 72:] == 7).all()


def test_gradient_against_differences(k3):
    """Central differences of the loss itself: a step of d along a direction of X moves g . loss by
    2 d <dX, direction>. X + d u is exact in bf16 (steps of 2^-3 on a grid), the third
    derivative of a log-sum-exp of logits moved by |W u| is at most |W u|^3 / 6 a row, and the
    losses carry their own bounds."""
    T, n, vocab, d = 24, 64, 500, 2.0 ** -3
    _, W, g, gen = inputs(T, n, vocab, 10, spread=0.5)
    X = (torch.randint(-8, 9, (T, n), generator=gen, device="cuda") / 8).bfloat16()
    u = torch.where(torch.rand((T, n), generator=gen, device="cuda") < 0.5, -1.0, 1.0).bfloat16()
    label = torch.randint(0, vocab, (T,), generator=gen, device="cuda").int()
    ids = torch.randint(0, vocab, (T, 5), generator=gen, device="cuda").int()
    top = torch.randn((T, 5), generator=gen, device="cuda")
    for fwd, bwd in ((lambda x: k3.lm_head_xent(x, W, label),
                      lambda x, l: k3.lm_head_xent_grad(x, W, label, l, g=g)[0]),
                     (lambda x: k3.lm_head_distill(x, W, ids, top),
                      lambda x, l: k3.lm_head_distill_grad(x, W, ids, top, l, g=g)[0])):
        _, lse = fwd(X)
        dX = bwd(X, lse).double()
        up, down = fwd(X + d * u)[0].double(), fwd(X - d * u)[0].double()
        got = (up - down) * g.double() / (2 * d)
        want = (dX * u.double()).sum(1)
        move = (u.double() @ W.double().T).abs().amax(1) * 2            # of z_i - E z, at most
        S = (X.double().abs() + d) @ W.double().abs().T
        ez = (n / 16 + 16) * 2.0 ** -23 * S.amax(1)
        loss_err = (2 * ez + 2.0 ** -21 * (up.abs() * 2 + 20)) / d
        grad_err = 2.0 ** -7 * (W.double().abs().amax(1).max() * n * 2 + dX.abs().sum(1) / g.double().abs())
        assert ((got - want).abs() <= g.double().abs() * (move ** 3 * d * d / 6 + loss_err + grad_err)).all()


@pytest.mark.parametrize("T,n,vocab", [(70, 1024, 2000), (200, 3200, 900), (300, 7168, 5000)])
def test_sure_rows(k3, T, n, vocab):
    """Rows that are nearly right (p of the label 0.99 to 0.9999): the loss and p - 1 are small
    differences. The same z stands on both sides of them, so what is left is
      loss  2 (1 - p) ez, and the fp32 sum of 2^(z - max): 32 additions beside a 1, 2^-19
      p     the fp32 lse and its product with log2 e, 2^-22 |lse|, and the exp2, 2^-22 =: d
      dX    a row's norm: d (|W_label| + sum p |W|), and the roundings of dz and dX."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    W = (torch.randn((vocab, n), generator=gen, device="cuda") * (1.7 / math.sqrt(n))).bfloat16()
    label = torch.randint(0, vocab, (T,), generator=gen, device="cuda").int()
    X = torch.randn((T, n), generator=gen, device="cuda")
    Wl = W[label.long()].float()
    lean = torch.empty(T, device="cuda").uniform_(5, 9, generator=gen) + math.log(vocab)
    X = (X + Wl * ((lean - (X * Wl).sum(1)) / (Wl * Wl).sum(1))[:, None]).bfloat16()
    Xd, Wd, at = X.double(), W.double(), label.long()[:, None]
    z = Xd @ Wd.T
    lse, zl = torch.logsumexp(z, 1), z.gather(1, at)[:, 0]
    rest = torch.logsumexp(z.scatter(1, at, -math.inf), 1) - zl
    loss = torch.log1p(rest.exp())
    miss = -torch.expm1(-loss)                                        # 1 - p
    assert 1e-5 < float(miss.min()) and float(miss.median()) < 0.02
    dz = (z - lse[:, None]).exp().scatter(1, at, -miss[:, None])
    dX = dz @ Wd
    got, got_lse = k3.lm_head_xent(X, W, label)
    grad, _ = k3.lm_head_xent_grad(X, W, label, got_lse, need_dw=False)
    ez = ((n / 16 + 16) * 2.0 ** -23 * (Xd.abs() @ Wd.abs().T)).amax(1)
    assert bool(((got.double() - loss).abs() <= 2 * miss * ez + 2.0 ** -19).all())
    d, norms = 2.0 ** -22 * (lse.abs() + 1), Wd.norm(dim=1)
    bound = d * (norms[at[:, 0]] + (z - lse[:, None]).exp() @ norms) + 2.0 ** -8 * (dz.abs() @ norms + dX.norm(dim=1))
    assert bool(((grad.double() - dX).norm(dim=1) <= bound + 2 * miss * ez * norms.max()).all())


@pytest.mark.parametrize("kind", ["mean", "spread", "tiny", "huge", "zeros", "signs"])
def test_weights(k3, kind):
    """Incoming gradients as they come: a mean's 1/n, 40 orders of magnitude apart, all tiny or
    huge, all zero, of either sign; an infinite one does not touch the other rows' dX."""
    X, W, _, gen = inputs(90, 136, 700, 22)
    label = torch.randint(-1, 700, (90,), generator=gen, device="cuda").int()
    r = torch.rand(90, generator=gen, device="cuda") + 0.5
    far = 10.0 ** torch.linspace(-20, 20, 90, device="cuda")
    g = {"mean": torch.full((90,), 1 / 77, device="cuda"), "spread": r * far, "tiny": r * 1e-33, "huge": r * 1e33,
         "zeros": torch.zeros(90, device="cuda"), "signs": r * 2 - 2}[kind]
    got = xent_all(k3, X, W, label, g)
    want = formula(X, W, targets_xent(label, 700), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    # (rows as they are scaled without the infinite one: by 1)
    one = xent_all(k3, X, W, label, r)["dX"]
    r2 = r.clone()
    r2[11] = math.inf
    label[11] = 5
    far = xent_all(k3, X, W, label, r2)["dX"]
    other = torch.arange(90, device="cuda") != 11
    assert bool(torch.isfinite(far[other]).all())
    assert float((far[other].double() - one[other].double()).norm() / one[other].double().norm()) < 2.0 ** -6


def test_frozen_head_and_head_alone(k3):
    X, W, g, gen = inputs(100, 264, 777, 11)
    label = torch.randint(-1, 777, (100,), generator=gen, device="cuda").int()
    _, lse = k3.lm_head_xent(X, W, label)
    dX, dW = k3.lm_head_xent_grad(X, W, label, lse, g=g)
    a, none = k3.lm_head_xent_grad(X, W, label, lse, g=g, need_dw=False)
    assert none is None and torch.equal(a, dX)
    none, b = k3.lm_head_xent_grad(X, W, label, lse, g=g, need_dx=False)
    assert none is None and torch.equal(b, dW)
    one = k3.lm_head_xent_grad(X, W, label, lse)
    two = k3.lm_head_xent_grad(X, W, label, lse, g=torch.ones_like(g))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_no_rows(k3):
    X, W, g, _ = inputs(4, 64, 50, 12)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse = k3.lm_head_xent(X[:0], W, none)
    dX, dW = k3.lm_head_xent_grad(X[:0], W, none, lse)
    assert loss.shape == lse.shape == (0,) and dX.shape == (0, 64) and (dW == 0).all()


def test_repeatable_on_another_stream_and_in_a_graph(k3):
    """Twice the same bits; on a side stream; captured once and replayed on new inputs."""
    X, W, g, gen = inputs(270, 520, 2050, 13)
    label = torch.randint(-1, 2050, (270,), generator=gen, device="cuda").int()
    base = xent_all(k3, X, W, label, g)
    again = xent_all(k3, X, W, label, g)
    for name in base:
        assert torch.equal(base[name], again[name])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = xent_all(k3, X, W, label, g)
    torch.cuda.current_stream().wait_stream(side)
    for name in base:
        assert torch.equal(base[name], other[name])
    Xs, ls = X.clone(), label.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = xent_all(k3, Xs, W, ls, g)
    X2, _, _, gen = inputs(270, 520, 2050, 14)
    l2 = torch.randint(0, 2050, (270,), generator=gen, device="cuda").int()     # now every row counts
    for x, lab in ((X2, l2), (X, label)):
        Xs.copy_(x)
        ls.copy_(lab)
        graph.replay()
        want = xent_all(k3, x, W, lab, g)
        for name in want:
            assert torch.equal(got[name], want[name]), name
    assert k3.device_status(0) == 0


def test_a_sweep_teaches_a_head(k3):
    """The operators as they are used together: a target's logits, their top entries, the
    distillation of a draft head from them and both gradients, against the formulas."""
    Xt, Wt, _, gen = inputs(90, 256, 1500, 15, spread=4.0)
    logits = k3.matmul_bf16(Xt.float(), Wt)
    ids, top = k3.topk_logits(logits, 24)
    order = logits.double().cpu().sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids.cpu().long(), order.indices[:, :24])
    X, W, g, _ = inputs(90, 128, 1500, 16)
    got = distill_all(k3, X, W, ids, top, 2.0, g)
    want = formula(X, W, targets_distill(ids, top, 2.0, 1500), 2.0, g)
    for name in want:
        holds(name, got[name], want[name])
    # the hard-label loss on the teacher's first choice
    got = xent_all(k3, X, W, ids[:, 0].contiguous(), g)
    want = formula(X, W, targets_xent(ids[:, 0], 1500), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])


def test_stream_argument(k3):
    """stream=: the call and what it allocates belong to that stream; a stream of the caller's that
    is still busy does not disturb it."""
    X, W, g, gen = inputs(200, 256, 3000, 17)
    label = torch.randint(-1, 3000, (200,), generator=gen, device="cuda").int()
    want = xent_all(k3, X, W, label, g)
    wi, wv = k3.topk_logits(X.float(), 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        torch.randn(1 << 22, device="cuda").sort()                  # the current stream stays busy
        loss, lse = k3.lm_head_xent(X, W, label, stream=side)
        dX, dW = k3.lm_head_xent_grad(X, W, label, lse, g=g, stream=side)
        got.append((loss, lse, dX, dW, *k3.topk_logits(X.float(), 9, stream=None)))
    side.synchronize()
    for loss, lse, dX, dW, ti, tv in got:
        assert torch.equal(loss, want["loss"]) and torch.equal(lse, want["lse"])
        assert torch.equal(dX, want["dX"]) and torch.equal(dW, want["dW"])
        assert torch.equal(ti, wi) and torch.equal(tv, wv)


def test_two_streams_at_once(k3):
    """Two steps in flight together, each with its own workspace."""
    a, b = inputs(300, 320, 4000, 18), inputs(310, 312, 4100, 19)
    la = torch.randint(-1, 4000, (300,), generator=a[3], device="cuda").int()
    lb = torch.randint(-1, 4100, (310,), generator=b[3], device="cuda").int()
    wa, wb = xent_all(k3, a[0], a[1], la, a[2]), xent_all(k3, b[0], b[1], lb, b[2])
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    out = []
    for _ in range(6):
        with torch.cuda.stream(sa):
            out.append((xent_all(k3, a[0], a[1], la, a[2]), wa))
        with torch.cuda.stream(sb):
            out.append((xent_all(k3, b[0], b[1], lb, b[2]), wb))
    torch.cuda.synchronize()
    for got, want in out:
        for name in want:
            assert torch.equal(got[name], want[name]), name
    assert k3.device_status(0) == 0


def test_first_call_inside_a_capture():
    """A process whose first call of each entry point is captured."""
    code = (
        "import sys; sys.path[:0] = [%r, %r]\n"
        "import torch\n"
        "from k3lib import load\n"
        "k3 = load()\n"
        "X = torch.randn((300, 128), device='cuda').bfloat16()\n"
        "W = torch.randn((2000, 128), device='cuda').bfloat16()\n"
        "ids = torch.randint(0, 2000, (300, 6), device='cuda').int()\n"
        "top = torch.randn((300, 6), device='cuda')\n"
        "lg = torch.randn((30, 20000), device='cuda')\n"
        "torch.cuda.synchronize()\n"
        "def run():\n"
        "    t = k3.topk_logits(lg, 5)\n"
        "    l = k3.lm_head_distill(X, W, ids, top)\n"
        "    return (*t, *l, *k3.lm_head_distill_grad(X, W, ids, top, l[1]))\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    got = run()\n"
        "g.replay()\n"
        "for a, b in zip(got, run()):\n"
        "    assert torch.equal(a, b)\n"
        "print('same')\n" % (HERE, os.path.dirname(HERE)))
    import subprocess
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_far_offsets(k3):
    """A head of 4.6e9 elements: offsets past 2^32 in W and dW. The logits of two rows in 64 bits,
    a slice of the head at a time; dW at the first id, the targets and the last."""
    n, vocab, T = 65536, 70001, 2
    gen = torch.Generator(device="cuda").manual_seed(20)
    X = torch.randn((T, n), generator=gen, device="cuda").bfloat16()
    W = torch.empty((vocab, n), dtype=torch.bfloat16, device="cuda").normal_(0, 1 / math.sqrt(n), generator=gen)
    label = torch.tensor([vocab - 1, 65537], dtype=torch.int32, device="cuda")
    g = torch.tensor([0.75, -0.4], device="cuda")
    got = xent_all(k3, X, W, label, g)
    z, S = [], []
    for v in range(0, vocab, 4096):
        w = W[v:v + 4096].double()
        z.append(X.double() @ w.T)
        S.append(X.double().abs() @ w.abs().T)
    z, S = torch.cat(z, 1), torch.cat(S, 1)
    ez = ((n / 16 + 16) * 2.0 ** -23 * S).amax(1)
    lse = torch.logsumexp(z, 1)
    loss = lse - z.gather(1, label.long()[:, None])[:, 0]
    mag = lse.abs() + z.abs().amax(1) + 1
    holds("lse", got["lse"], (lse, ez + 2.0 ** -21 * mag))
    holds("loss", got["loss"], (loss, 2 * ez + 2.0 ** -21 * mag))
    p = (z - lse[:, None]).exp()
    for v in (0, 32768, 65537, vocab - 1):
        hit = (label == v).double()
        dz = (p[:, v] - hit) * g.double()
        b = dz.abs() * 2.0 ** -8 + g.double().abs() * (p[:, v] * (2 * ez + 2.0 ** -18 * mag) + hit * 2.0 ** -22)
        want = dz @ X.double()
        sums = 2.0 ** -18 * (dz.abs() @ X.double().abs())
        holds("dW", got["dW"][v], (want, b @ X.double().abs() + want.abs() * 2.0 ** -8 + sums))


def test_wrappers_refuse(k3):
    X, W, g, gen = inputs(8, 64, 100, 21)
    label = torch.zeros(8, dtype=torch.int32, device="cuda")
    lse = torch.zeros(8, device="cuda")
    ids, top = torch.zeros((8, 3), dtype=torch.int32, device="cuda"), torch.zeros((8, 3), device="cuda")
    bad = [lambda: k3.lm_head_xent(X.float(), W, label), lambda: k3.lm_head_xent(X, W.half(), label),
           lambda: k3.lm_head_xent(X[:, :56], W, label), lambda: k3.lm_head_xent(X, W, label.long()),
           lambda: k3.lm_head_xent(X, W, label[:7]), lambda: k3.lm_head_xent(X, W, label.cpu()),
           lambda: k3.lm_head_xent(X.cpu(), W, label), lambda: k3.lm_head_xent(X, W.cpu(), label),
           lambda: k3.lm_head_xent(X, W.t().contiguous().t(), label), lambda: k3.lm_head_xent(X.t(), W, label),
           lambda: k3.lm_head_xent(X[:1].expand(8, 64), W, label),
           lambda: k3.lm_head_xent(X[:, :60], W[:, :60].contiguous(), label),           # not a multiple of 8
           lambda: k3.lm_head_xent(X, W, label, ws=torch.empty(16, dtype=torch.uint8, device="cuda")),
           lambda: k3.lm_head_xent(X, W, label, ws=torch.empty(1 << 20, device="cuda")),
           lambda: k3.lm_head_xent_grad(X, W, label, lse.double()), lambda: k3.lm_head_xent_grad(X, W, label, lse[:4]),
           lambda: k3.lm_head_xent_grad(X, W, label, lse, g=g.half()),
           lambda: k3.lm_head_distill(X, W, ids, top[:, :2]), lambda: k3.lm_head_distill(X, W, ids.long(), top),
           lambda: k3.lm_head_distill(X, W, ids, top, temp=0.0),
           lambda: k3.lm_head_distill(X, W, ids, top, temp=math.nan),
           lambda: k3.lm_head_distill(X, W, ids.repeat(1, 43), top.repeat(1, 43)),      # 129 entries
           lambda: k3.lm_head_distill_grad(X, W, ids, top, lse, temp=-1.0),
           lambda: k3.topk_logits(X, 4), lambda: k3.topk_logits(top.t(), 2), lambda: k3.topk_logits(top, 129),
           lambda: k3.topk_logits(top, 0), lambda: k3.topk_logits(top.cpu(), 2)]
    for i, call in enumerate(bad):
        with pytest.raises(k3.K3Error):
            call()
            pytest.fail(f"call {i} was taken")
    k3.lm_head_xent_grad(X, W, label, lse, need_dx=False, need_dw=False)
    assert k3.device_status(0) == 0


def test_a_model_sweep_teaches_a_head(k3, tmp_path):
    """From the whole model's verify sweep: the top entries of its logits buffer (the first of them
    the sweep's own argmax), and a draft head's step on them."""
    model = k3.Model.from_checkpoint(k3._sibling("synth").write_checkpoint(str(tmp_path), seed=0), B=1, max_T=8,
                                     kv_cap=64)
    prompt = torch.randint(0, model.vocab, (1, 6), device="cuda").int()
    model.prefill(prompt)
    arg, logits = model.verify(torch.randint(0, model.vocab, (1, 8), device="cuda").int())
    flat = logits.view(8, model.vocab)
    ids, top = k3.topk_logits(flat, 16)
    assert torch.equal(ids[:, 0], arg[0])
    want = flat.double().cpu().sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids.cpu().long(), want.indices[:, :16])
    assert torch.equal(top.cpu().double(), want.values[:, :16])
    X, W, g, _ = inputs(8, 128, model.vocab, 23)
    got = distill_all(k3, X, W, ids, top, 1.0, g)
    bounds = formula(X, W, targets_distill(ids, top, 1.0, model.vocab), 1.0, g)
    model.close()
    for name in bounds:
        holds(name, got[name], bounds[name])
