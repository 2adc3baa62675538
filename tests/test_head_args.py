"""What the draft-head losses and the top-K refuse, without a device: every check comes before
the first CUDA call."""
import ctypes as C
import math

import pytest

from tests import k3lib

P = C.c_void_p(1 << 20)         # never dereferenced


@pytest.fixture(scope="module")
def m():
    return k3lib.load()


def xent(m, **kw):
    a = dict(loss=P, lse=P, X=P, ldx=64, W=P, label=P, n=64, vocab=100, T=8, ws=P, bytes=1 << 30)
    a.update(kw)
    return m.lib.k3gpu_lm_head_xent(a["loss"], a["lse"], a["X"], a["ldx"], a["W"], a["label"], a["n"], a["vocab"],
                                    a["T"], a["ws"], a["bytes"], None)


def xent_grad(m, **kw):
    a = dict(dX=P, lddx=64, dW=P, g=None, lse=P, X=P, ldx=64, W=P, label=P, n=64, vocab=100, T=8, ws=P, bytes=1 << 30)
    a.update(kw)
    return m.lib.k3gpu_lm_head_xent_grad(a["dX"], a["lddx"], a["dW"], a["g"], a["lse"], a["X"], a["ldx"], a["W"],
                                         a["label"], a["n"], a["vocab"], a["T"], a["ws"], a["bytes"], None)


def distill(m, **kw):
    a = dict(loss=P, lse=P, X=P, ldx=64, W=P, ids=P, top=P, K=4, temp=1.0, n=64, vocab=100, T=8, ws=P, bytes=1 << 30)
    a.update(kw)
    return m.lib.k3gpu_lm_head_distill(a["loss"], a["lse"], a["X"], a["ldx"], a["W"], a["ids"], a["top"], a["K"],
                                       a["temp"], a["n"], a["vocab"], a["T"], a["ws"], a["bytes"], None)


def distill_grad(m, **kw):
    a = dict(dX=P, lddx=64, dW=P, g=None, lse=P, X=P, ldx=64, W=P, ids=P, top=P, K=4, temp=1.0, n=64, vocab=100, T=8,
             ws=P, bytes=1 << 30)
    a.update(kw)
    return m.lib.k3gpu_lm_head_distill_grad(a["dX"], a["lddx"], a["dW"], a["g"], a["lse"], a["X"], a["ldx"], a["W"],
                                            a["ids"], a["top"], a["K"], a["temp"], a["n"], a["vocab"], a["T"],
                                            a["ws"], a["bytes"], None)


HEAD = [dict(X=None), dict(W=None), dict(ws=None), dict(lse=None), dict(n=0), dict(n=60), dict(n=1 << 17, ldx=1 << 17),
        dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(T=0), dict(T=-1), dict(T=(1 << 20) + 1), dict(ldx=63),
        dict(W=C.c_void_p((1 << 20) + 8)), dict(X=C.c_void_p((1 << 20) + 1)), dict(ws=C.c_void_p((1 << 20) + 16))]
TEACHER = [dict(ids=None), dict(top=None), dict(K=0), dict(K=129), dict(temp=0.0), dict(temp=-1.0), dict(temp=math.inf),
           dict(temp=math.nan), dict(temp=1e-42)]
GRADS = [dict(dX=None, dW=None), dict(lddx=63), dict(dX=C.c_void_p((1 << 20) + 1)), dict(dW=C.c_void_p((1 << 20) + 8))]


@pytest.mark.parametrize("kw", HEAD + [dict(label=None), dict(loss=None)])
def test_xent_refuses(m, kw):
    assert xent(m, **kw) == m.K3GPU_EINVAL


@pytest.mark.parametrize("kw", HEAD + GRADS + [dict(label=None)])
def test_xent_grad_refuses(m, kw):
    assert xent_grad(m, **kw) == m.K3GPU_EINVAL


@pytest.mark.parametrize("kw", HEAD + TEACHER + [dict(loss=None)])
def test_distill_refuses(m, kw):
    assert distill(m, **kw) == m.K3GPU_EINVAL


@pytest.mark.parametrize("kw", HEAD + TEACHER + GRADS)
def test_distill_grad_refuses(m, kw):
    assert distill_grad(m, **kw) == m.K3GPU_EINVAL


def test_workspace_short(m):
    need = m.lib.k3gpu_lm_head_xent_workspace(8, 64, 100)
    assert need > 0
    assert xent(m, bytes=need - 1) == xent_grad(m, bytes=need - 1) == m.K3GPU_ECAPACITY
    need = m.lib.k3gpu_lm_head_distill_workspace(8, 64, 100, 4)
    assert distill(m, bytes=need - 1) == distill_grad(m, bytes=need - 1) == m.K3GPU_ECAPACITY


def test_workspace_sizes(m):
    """0 for refused sizes; far below the logits' own size; growing with no T * vocab."""
    lib = m.lib
    assert lib.k3gpu_lm_head_xent_workspace(0, 64, 100) == 0
    assert lib.k3gpu_lm_head_xent_workspace(8, 60, 100) == 0
    assert lib.k3gpu_lm_head_distill_workspace(8, 64, 100, 0) == 0
    assert lib.k3gpu_lm_head_distill_workspace(8, 64, 100, 129) == 0
    T, n, V = 8192, 2048, 163840
    assert lib.k3gpu_lm_head_xent_workspace(T, n, V) < T * V * 4 // 8
    assert lib.k3gpu_topk_logits_workspace(0, 10, 1) == lib.k3gpu_topk_logits_workspace(1, 10, 129) == 0


@pytest.mark.parametrize("kw", [dict(idx=None), dict(val=None), dict(logits=None), dict(ws=None), dict(rows=0),
                                dict(rows=65536), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(K=0), dict(K=129),
                                dict(ws=C.c_void_p((1 << 20) + 4)), dict(logits=C.c_void_p((1 << 20) + 2))])
def test_topk_refuses(m, kw):
    a = dict(idx=P, val=P, logits=P, rows=2, vocab=10, K=3, ws=P, bytes=1 << 20)
    a.update(kw)
    assert m.lib.k3gpu_topk_logits(a["idx"], a["val"], a["logits"], a["rows"], a["vocab"], a["K"], a["ws"],
                                   a["bytes"], None) == m.K3GPU_EINVAL


def test_topk_workspace_short(m):
    need = m.lib.k3gpu_topk_logits_workspace(9, 163840, 64)
    assert m.lib.k3gpu_topk_logits(P, P, P, 9, 163840, 64, P, need - 1, None) == m.K3GPU_ECAPACITY


ODD = C.c_void_p((1 << 20) + 2)         # not on a 4-byte boundary


@pytest.mark.parametrize("call,names", [(xent, ("loss", "lse", "label")), (xent_grad, ("lse", "label", "g")),
                                        (distill, ("loss", "lse", "ids", "top")),
                                        (distill_grad, ("lse", "ids", "top", "g"))])
def test_misaligned_values_refused(m, call, names):
    """32-bit inputs and outputs off their boundary: an error, not a fault of the kernels'."""
    for name in names:
        assert call(m, **{name: ODD}) == m.K3GPU_EINVAL, name


def test_topk_misaligned_outputs_refused(m):
    for idx, val in ((ODD, P), (P, ODD)):
        assert m.lib.k3gpu_topk_logits(idx, val, P, 2, 10, 3, P, 1 << 20, None) == m.K3GPU_EINVAL
