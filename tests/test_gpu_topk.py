"""k3gpu_topk_logits: the K largest logits of each row, exactly: a stable descending sort's
first K over the values that are not NaN, then -1 / -inf."""
import math
import os
import sys

import numpy as np
import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
from k3lib import load  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def k3():
    return load()


def want_of(a, K):
    idx = np.full((a.shape[0], K), -1, np.int32)
    val = np.full((a.shape[0], K), -np.inf, np.float32)
    for r, row in enumerate(a):
        ids = np.flatnonzero(~np.isnan(row))
        ids = ids[np.argsort(-row[ids].astype(np.float64), kind="stable")][:K]
        idx[r, :len(ids)], val[r, :len(ids)] = ids, row[ids]
    return idx, val


def check(k3, a, K):
    a = np.ascontiguousarray(a, np.float32)
    idx, val = k3.topk_logits(torch.from_numpy(a).cuda(), K)
    wi, wv = want_of(a, K)
    np.testing.assert_array_equal(idx.cpu().numpy(), wi)
    np.testing.assert_array_equal(val.cpu().numpy(), wv)


@pytest.mark.parametrize("rows,vocab,K", [(1, 1, 1), (1, 5, 128), (3, 127, 128), (2, 4096, 64), (5, 4097, 1),
                                          (9, 8191, 33), (1, 163840, 128), (9, 163840, 64), (70, 50257, 10),
                                          (600, 20011, 7), (2, 400003, 100)])
def test_random(k3, rows, vocab, K):
    rng = np.random.default_rng(rows + vocab + K)
    check(k3, rng.standard_normal((rows, vocab)), K)


@pytest.mark.parametrize("K", [1, 64, 128])
def test_orders_and_ties(k3, K):
    """Ascending and descending rows, one value everywhere, few values, the K best all in one
    thread's stride, ties across the K-th place."""
    n = 40001
    rng = np.random.default_rng(K)
    up = np.arange(n, dtype=np.float32)
    stride = rng.standard_normal(n).astype(np.float32)
    stride[17::512] += 100
    ties = np.zeros(n, np.float32)
    ties[rng.permutation(n)[:K // 2]] = 1
    check(k3, np.stack([up, -up, np.full(n, -3.5, np.float32), rng.integers(0, 3, n).astype(np.float32), stride, ties]), K)


def test_special_values(k3):
    """NaN never, -inf last, +inf first, the lowest finite value, both zeros equal, subnormals in
    order; rows of NaN alone and of few values."""
    n, K = 9001, 32
    rng = np.random.default_rng(1)
    a = rng.standard_normal((8, n)).astype(np.float32)
    a[0, rng.random(n) < 0.5] = np.nan
    a[1] = np.nan
    a[2] = np.nan
    a[2, [5, 4097, 8999]] = [-np.inf, 3, np.inf]
    a[3] = -np.inf
    a[3, 7000] = np.finfo(np.float32).min
    a[4] = np.where(rng.random(n) < 0.5, 0.0, -0.0)
    a[5] = rng.integers(-40, 40, n) * 1e-45
    a[6, ::2] = np.inf
    a[7, :n - 10] = np.nan
    check(k3, a, K)


def test_rows_start_at_any_address(k3):
    """An odd vocabulary puts rows off every alignment, and the first off 16 bytes too."""
    rng = np.random.default_rng(2)
    a = rng.standard_normal((7, 12347)).astype(np.float32)
    flat = torch.from_numpy(np.concatenate([np.zeros(1, np.float32), a.ravel()])).cuda()
    idx, val = k3.topk_logits(flat[1:].view(7, 12347), 20)
    wi, wv = want_of(a, 20)
    np.testing.assert_array_equal(idx.cpu().numpy(), wi)
    np.testing.assert_array_equal(val.cpu().numpy(), wv)


def test_stream_and_graph(k3):
    a = torch.randn((12, 30000), device="cuda")
    graph = torch.cuda.CUDAGraph()
    k3.topk_logits(a, 16)
    with torch.cuda.graph(graph):
        idx, val = k3.topk_logits(a, 16)
    for seed in (1, 2):
        a.copy_(torch.randn((12, 30000), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        wi, wv = want_of(a.cpu().numpy(), 16)
        np.testing.assert_array_equal(idx.cpu().numpy(), wi)
        np.testing.assert_array_equal(val.cpu().numpy(), wv)
    assert k3.topk_logits(a[:0], 16)[0].shape == (0, 16)


def test_agrees_with_argmax(k3):
    a = torch.randn((40, 163840), device="cuda")
    assert torch.equal(k3.topk_logits(a, 1)[0][:, 0], k3.argmax(a))


def test_far_offsets(k3):
    """Rows past 2^31 elements from the first."""
    rows, vocab, K = 14000, 163840, 16
    a = torch.randn((rows, vocab), device="cuda")
    idx, val = k3.topk_logits(a, K)
    for r in (0, 13107, 13108, rows - 1):
        wi, wv = want_of(a[r:r + 1].cpu().numpy(), K)
        np.testing.assert_array_equal(idx[r:r + 1].cpu().numpy(), wi)
        np.testing.assert_array_equal(val[r:r + 1].cpu().numpy(), wv)


@pytest.mark.parametrize("K", [1, 100])
def test_mostly_banned_rows(k3, K):
    """Rows of which all but a few, or exactly K, or fewer than K ids are -inf, and rows of one value."""
    n = 50000
    rng = np.random.default_rng(K)
    a = np.full((5, n), -np.inf, np.float32)
    for r, m in enumerate((0, 1, K, K + 3)):
        a[r, rng.permutation(n)[:m]] = rng.standard_normal(m)
    a[4] = 1.5
    check(k3, a, K)
