"""What the draft-head losses ask for as workspace, without a device: each direction no more than
what it keeps, at one row as at a million."""
import ctypes as C

import pytest

from tests import k3lib
from tests.test_head_args import P, distill, distill_grad, xent, xent_grad

GRAIN = 1 << 18                 # sizes come in whole 256 KB
MB = 1 << 20

SIZES = [(T, n, V) for T in (1, 9, 64, 129, 301, 576, 2048, 8192, 1 << 20)
         for n, V in ((1024, 32000), (1000, 50257), (7168, 163840), (8, 1))] + [(257, 65536, 163840), (1, 65536, 1 << 24)]


@pytest.fixture(scope="module")
def m():
    return k3lib.load()


def up(x, to):
    return -(-x // to) * to


def small(T, K):
    """Counts, the rows' records and teacher entries, each array on 256 bytes."""
    return 12 * 256 + T * (16 + 8 + 8 * K)


def loss_bytes(T, n, V, K):
    """A copy of the rows that count, padded to 256; two (maximum, sum) pairs a row and 256 ids; the
    targets' logits."""
    rows = up(T, 256)
    return rows * n * 2 + up(V, 256) // 256 * 2 * rows * 8 + T * max(K, 1) * 4 + small(T, K) + GRAIN


def grad_bytes(T, n, V, K):
    """That copy; dz, bf16, of one piece of the vocabulary that holds all of it, else of two of 128 MB
    (of eight tiles of 256 ids, if that is more), its rows padded to 64; dX in fp32, its rows padded
    to 32, split 32 times at most and while the splits fit 256 MB together, unless one alone is
    larger; up to 32 rows two sets of them."""
    rows = up(T, 64)
    piece = max(8, 128 * MB // (up(T, 256) * 512)) * 256
    dz = rows * up(V, 256) * 2 if V <= piece else 2 * rows * piece * 2
    one = (64 if T <= 32 else up(T, 32)) * up(n, 256) * 4
    return up(T, 256) * n * 2 + dz + max(one, min(32 * one, 256 * MB)) + small(T, K) + GRAIN


@pytest.mark.parametrize("T,n,V", SIZES)
@pytest.mark.parametrize("K", [0, 1, 128])
def test_no_more_than_what_is_kept(m, T, n, V, K):
    lib = m.lib
    if K:
        loss, both = lib.k3gpu_lm_head_distill_loss_workspace(T, n, V, K), lib.k3gpu_lm_head_distill_workspace(T, n, V, K)
    else:
        loss, both = lib.k3gpu_lm_head_xent_loss_workspace(T, n, V), lib.k3gpu_lm_head_xent_workspace(T, n, V)
    assert 0 < loss <= both
    assert loss <= loss_bytes(T, n, V, K)
    assert both <= max(loss_bytes(T, n, V, K), grad_bytes(T, n, V, K))


def test_one_sweep_under_the_full_head(m):
    """9 rows over 163,840 ids, whose fp32 logits are 5.9 MB."""
    lib = m.lib
    assert lib.k3gpu_lm_head_xent_loss_workspace(9, 7168, 163840) < 7 * MB
    assert lib.k3gpu_lm_head_xent_workspace(9, 7168, 163840) < 70 * MB


def test_a_loss_takes_its_own_size(m):
    """The loss alone runs in its own workspace, which the gradient refuses."""
    T, n, V, K = 9, 7168, 163840, 64
    size = dict(T=T, n=n, vocab=V, ldx=n)
    lib = m.lib
    need, both = lib.k3gpu_lm_head_xent_loss_workspace(T, n, V), lib.k3gpu_lm_head_xent_workspace(T, n, V)
    assert xent(m, bytes=need - 1, **size) == m.K3GPU_ECAPACITY
    assert xent_grad(m, bytes=need, lddx=n, **size) == xent_grad(m, bytes=both - 1, lddx=n, **size) == m.K3GPU_ECAPACITY
    need, both = lib.k3gpu_lm_head_distill_loss_workspace(T, n, V, K), lib.k3gpu_lm_head_distill_workspace(T, n, V, K)
    assert distill(m, bytes=need - 1, K=K, **size) == m.K3GPU_ECAPACITY
    assert distill_grad(m, bytes=both - 1, K=K, lddx=n, **size) == m.K3GPU_ECAPACITY


def test_refused_sizes_have_none(m):
    lib = m.lib
    for T, n, V in ((0, 64, 100), (8, 60, 100), (8, 64, 0), (1 << 21, 64, 100), (8, 1 << 17, 100)):
        assert lib.k3gpu_lm_head_xent_loss_workspace(T, n, V) == 0
        assert lib.k3gpu_lm_head_distill_loss_workspace(T, n, V, 4) == 0
    assert lib.k3gpu_lm_head_distill_loss_workspace(8, 64, 100, 0) == 0
    assert lib.k3gpu_lm_head_distill_loss_workspace(8, 64, 100, 129) == 0


# single rows, few rows over a wide head (split sums), pairs, two pieces and more, no target at all
RUNS = [(1, 8, 1), (9, 7168, 20000), (65, 264, 3001), (250, 1032, 5003), (300, 520, 9000), (520, 64, 100003),
        (8200, 200, 10007)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,V", RUNS)
@pytest.mark.parametrize("K", [0, 5])
def test_nothing_past_the_workspace(m, T, n, V, K):
    """Each direction in a workspace of its own size, between bytes of the test's: they stay, and the
    outputs are those of the wrappers' own workspaces."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(T + n + V + K)
    X = torch.randn((T, n), generator=gen, device="cuda").bfloat16()
    W = (torch.randn((V, n), generator=gen, device="cuda") / n ** 0.5).bfloat16()
    label = torch.randint(-1, V, (T,), generator=gen, device="cuda").int()
    ids = torch.randint(-1, V, (T, 5), generator=gen, device="cuda").int()
    top = torch.randn((T, 5), generator=gen, device="cuda")
    lib, args = m.lib, (X, W, ids, top) if K else (X, W, label)
    fwd, bwd = (m.lm_head_distill, m.lm_head_distill_grad) if K else (m.lm_head_xent, m.lm_head_xent_grad)
    loss, both = ((lib.k3gpu_lm_head_distill_loss_workspace(T, n, V, K), lib.k3gpu_lm_head_distill_workspace(T, n, V, K))
                  if K else (lib.k3gpu_lm_head_xent_loss_workspace(T, n, V), lib.k3gpu_lm_head_xent_workspace(T, n, V)))
    wants = list(fwd(*args))
    wants += bwd(*args, wants[1])
    for need, call, want in ((loss, lambda ws: fwd(*args, ws=ws), wants[:2]),
                             (both, lambda ws: fwd(*args, ws=ws), wants[:2]),
                             (both, lambda ws: bwd(*args, wants[1], ws=ws), wants[2:])):
        room = torch.full((need + 2 * MB,), 0xA5, dtype=torch.uint8, device="cuda")
        ws = room[MB:MB + need]
        ws.fill_(0xFF)                                  # NaN wherever it is read before it is written
        got = call(ws)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert bool((room[:MB] == 0xA5).all()) and bool((room[MB + need:] == 0xA5).all())
    assert m.device_status(0) == 0
