"""Forms of the draft-head calls: one gradient without the other, hidden states as bits, pairs of CTAs
over wide rows, side streams inside a capture, several graphs."""
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
sys.path.insert(0, os.path.dirname(HERE))
from k3lib import load  # noqa: E402
from test_gpu_head import (distill_all, formula, holds, inputs, targets_distill, targets_xent,  # noqa: E402
                           xent_all)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k3():
    return load()


def entries(T, vocab, K, gen):
    ids = torch.randint(-1, vocab, (T, K), generator=gen, device="cuda").int()
    return ids, torch.randn((T, K), generator=gen, device="cuda") * 2


@pytest.mark.parametrize("T,n,vocab", [(9, 264, 777), (250, 520, 3001)])
def test_one_gradient_of_the_distillation(k3, T, n, vocab):
    X, W, g, gen = inputs(T, n, vocab, 41)
    ids, top = entries(T, vocab, 6, gen)
    _, lse = k3.lm_head_distill(X, W, ids, top, temp=1.5)
    dX, dW = k3.lm_head_distill_grad(X, W, ids, top, lse, temp=1.5, g=g)
    a, none = k3.lm_head_distill_grad(X, W, ids, top, lse, temp=1.5, g=g, need_dw=False)
    assert none is None and torch.equal(a, dX)
    none, b = k3.lm_head_distill_grad(X, W, ids, top, lse, temp=1.5, g=g, need_dx=False)
    assert none is None and torch.equal(b, dW)
    want = formula(X, W, targets_distill(ids, top, 1.5, vocab), 1.5, g)
    holds("dW", b, want["dW"])
    assert k3.lm_head_distill_grad(X, W, ids, top, lse, need_dx=False, need_dw=False) == (None, None)


@pytest.mark.parametrize("T,n,vocab", [(130, 3208, 700), (250, 1032, 5003), (1000, 7168, 1500), (9, 7168, 3001)])
def test_wide_rows(k3, T, n, vocab):
    """dW of many column tiles, in pairs (all but the last), beside the rest."""
    X, W, g, gen = inputs(T, n, vocab, 42)
    label = torch.randint(-1, vocab, (T,), generator=gen, device="cuda").int()
    got = xent_all(k3, X, W, label, g)
    want = formula(X, W, targets_xent(label, vocab), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    again = xent_all(k3, X, W, label, g)
    for name in got:
        assert torch.equal(got[name], again[name]), name


@pytest.mark.parametrize("dtype", [torch.int16, torch.uint16])
def test_bits_are_bf16(k3, dtype):
    X, W, g, gen = inputs(20, 64, 300, 43)
    label = torch.randint(-1, 300, (20,), generator=gen, device="cuda").int()
    want, got = xent_all(k3, X, W, label, g), xent_all(k3, X.view(dtype), W.view(dtype), label, g)
    for name in want:
        assert torch.equal(got[name], want[name]) and got[name].dtype == want[name].dtype


def test_a_side_stream_inside_a_capture(k3):
    """stream= with a stream that the capture has forked: the call is part of the graph."""
    X, W, g, gen = inputs(70, 136, 900, 44)
    label = torch.randint(-1, 900, (70,), generator=gen, device="cuda").int()
    side, graph, held = torch.cuda.Stream(), torch.cuda.CUDAGraph(), X.clone()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        loss, lse = k3.lm_head_xent(held, W, label, stream=side)
        dX, dW = k3.lm_head_xent_grad(held, W, label, lse, g=g, stream=side)
        torch.cuda.current_stream().wait_stream(side)
    X2 = inputs(70, 136, 900, 45)[0]
    for x in (X, X2):
        held.copy_(x)
        graph.replay()
        want = xent_all(k3, x, W, label, g)
        for name, t in (("loss", loss), ("lse", lse), ("dX", dX), ("dW", dW)):
            assert torch.equal(t, want[name]), name


def test_two_graphs_of_one_workspace(k3):
    """Two captured steps of different sizes that share the caller's workspace, replayed in turn on one
    stream, with eager steps between them."""
    a, b = inputs(300, 320, 4000, 46), inputs(9, 1032, 2100, 47)
    la = torch.randint(-1, 4000, (300,), generator=a[3], device="cuda").int()
    ib, tb = entries(9, 2100, 7, b[3])
    lib = k3.lib
    ws = k3.workspace(max(lib.k3gpu_lm_head_xent_workspace(300, 320, 4000),
                          lib.k3gpu_lm_head_distill_workspace(9, 1032, 2100, 7)))

    def step_a(ws=None):
        loss, lse = k3.lm_head_xent(a[0], a[1], la, ws=ws)
        return (loss, lse, *k3.lm_head_xent_grad(a[0], a[1], la, lse, g=a[2], ws=ws))

    def step_b(ws=None):
        loss, lse = k3.lm_head_distill(b[0], b[1], ib, tb, ws=ws)
        return (loss, lse, *k3.lm_head_distill_grad(b[0], b[1], ib, tb, lse, g=b[2], ws=ws))

    wa, wb = step_a(), step_b()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        oa = step_a(ws)
    with torch.cuda.graph(gb):
        ob = step_b(ws)
    for _ in range(3):
        for t in (*oa, *ob):
            t.fill_(-1)
        ga.replay()
        gb.replay()
        for got, want in zip((*oa, *ob, *step_a(ws), *step_b(ws)), (*wa, *wb, *wa, *wb)):
            assert torch.equal(got, want)
    assert k3.device_status(0) == 0


def test_same_rows_and_ids_many_times(k3):
    """One id the target of every row, and every entry of a row the same id."""
    X, W, g, gen = inputs(140, 72, 500, 48)
    label = torch.full((140,), 123, dtype=torch.int32, device="cuda")
    got, want = xent_all(k3, X, W, label, g), formula(X, W, targets_xent(label, 500), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
    ids, top = torch.full((140, 128), 499, dtype=torch.int32, device="cuda"), torch.zeros((140, 128), device="cuda")
    got, want = distill_all(k3, X, W, ids, top, 1.0, g), formula(X, W, targets_distill(ids, top, 1.0, 500), 1.0, g)
    for name in want:
        holds(name, got[name], want[name])
