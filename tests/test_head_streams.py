"""The draft-head wrappers on a stream or device that is not the current one: the device that they
make current, the names of their arguments, how long what a call reads stays alive, and how a model
in torch goes on from their gradients."""
import contextlib
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from k3lib import load  # noqa: E402


@pytest.fixture(scope="module")
def k3():
    return load()


# ---------------------------------------------------------------- without a device --
class Fake:
    """A tensor's device and record_stream, as far as the wrappers look at them."""
    is_cuda = True

    def __init__(self, index=0):
        self.device = torch.device("cuda", index)
        self.seen = []

    def record_stream(self, stream):
        self.seen.append(stream)


class FakeStream:
    def __init__(self, index=0):
        self.device = torch.device("cuda", index)


@pytest.fixture
def current(monkeypatch):
    """torch.cuda's current device and stream as plain names; `stack` lists what was entered."""
    stack = []

    @contextlib.contextmanager
    def enter(x):
        stack.append(x)
        yield
        stack.append(None)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", enter)
    monkeypatch.setattr(torch.cuda, "stream", enter)
    return stack


def test_another_device_is_made_current(k3, current):
    x = Fake(1)
    call = k3._on_device_of(lambda X, y: (list(current), X, y))
    entered, got, y = call(x, 5)
    assert entered == [x.device] and current == [x.device, None] and got is x and y == 5


def test_the_current_device_is_left_alone(k3, current):
    assert k3._on_device_of(lambda X: list(current))(Fake(0)) == [] and current == []


def test_a_stream_of_another_device_is_refused(k3, current):
    with pytest.raises(k3.K3Error):
        k3._on_device_of(lambda X: None)(Fake(0), stream=FakeStream(1))
    assert current == []


def test_inputs_are_recorded_on_the_stream(k3, current, monkeypatch):
    """With stream=, every tensor of the call is recorded there (its memory is not given to another
    before the kernels have read it), by place or by name; without, none is."""
    monkeypatch.setattr(k3, "_is_cuda_tensor", lambda t: isinstance(t, Fake))
    call = k3._on_device_of(lambda X, label, g=None, ws=None: list(current))
    x, lab, g, ws, s = Fake(), Fake(), Fake(), Fake(), FakeStream()
    assert call(x, lab, g=g, ws=ws, stream=s) == [s]
    assert x.seen == lab.seen == g.seen == ws.seen == [s]
    call(x, lab, g=None)
    assert x.seen == [s]


def test_first_argument_by_name(k3, current):
    """The first argument goes by its own name too, as help() shows it."""
    call = k3._on_device_of(lambda X, y=0: (X, y))
    x = Fake(1)
    assert call(X=x, y=3) == (x, 3) and current == [x.device, None]
    with pytest.raises(TypeError):
        call(x=Fake())
    with pytest.raises(TypeError):
        call()
    with pytest.raises(TypeError):
        call(x, X=x)


@pytest.mark.parametrize("name,first", [("topk_logits", "logits"), ("lm_head_xent", "X"), ("lm_head_xent_grad", "X"),
                                        ("lm_head_distill", "X"), ("lm_head_distill_grad", "X")])
def test_wrappers_take_their_first_argument_by_name(k3, name, first):
    """Far enough to be told that a host tensor will not do."""
    with pytest.raises(k3.K3Error, match="CUDA"):
        getattr(k3, name)(**{first: torch.zeros(1)})


class FakeTensor(Fake):
    """As far as a wrapper's checks look before anything is allocated."""

    def __init__(self, dtype, *shape):
        super().__init__()
        self.dtype, self.shape = dtype, torch.Size(shape)

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return 1 << 20


@pytest.mark.parametrize("rows", [0, 5])
@pytest.mark.parametrize("K", [-1, 0, 129])
def test_topk_refuses_k_before_it_allocates(k3, current, K, rows):
    with pytest.raises(k3.K3Error, match="K"):
        k3.topk_logits(FakeTensor(torch.float32, rows, 100), K)


@pytest.mark.parametrize("shape", [(), (8,), (8, 2, 2), (8, 0), (8, 129)])
def test_distill_refuses_entries_of_another_shape(k3, current, shape):
    X, W = FakeTensor(torch.bfloat16, 8, 64), FakeTensor(torch.bfloat16, 100, 64)
    ids, top, lse = FakeTensor(torch.int32, *shape), FakeTensor(torch.float32, *shape), FakeTensor(torch.float32, 8)
    with pytest.raises(k3.K3Error, match="ids"):
        k3.lm_head_distill(X, W, ids, top)
    with pytest.raises(k3.K3Error, match="ids"):
        k3.lm_head_distill_grad(X, W, ids, top, lse)


@pytest.mark.parametrize("name", ["lm_head_xent", "lm_head_xent_grad", "lm_head_distill", "lm_head_distill_grad"])
def test_documented_as_outside_autograd(k3, name):
    assert "utside autograd" in " ".join(getattr(k3, name).__doc__.split())


# ------------------------------------------------------------------- on a device ------
def inputs():
    gen = torch.Generator(device="cuda").manual_seed(1)
    X = torch.randn((300, 2048), generator=gen, device="cuda").bfloat16()
    W = (torch.randn((5000, 2048), generator=gen, device="cuda") / 45).bfloat16()
    label = torch.randint(-1, 5000, (300,), generator=gen, device="cuda").int()
    logits = torch.randn((300, 5000), generator=gen, device="cuda")
    return X, W, label, logits


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_a_temporary_outlives_its_call(k3, which):
    """A temporary given to a call on a side stream that is still busy: its memory is not handed
    out again until the kernels have read it. Without the call it is, at once."""
    X, W, label, logits = inputs()
    ids, top = k3.topk_logits(logits, 8)
    lse_x, lse_d = k3.lm_head_xent(X, W, label)[1], k3.lm_head_distill(X, W, ids, top)[1]
    call, first = [(lambda x, **kw: k3.topk_logits(x, 8, **kw), logits),
                   (lambda x, **kw: k3.lm_head_xent(x, W, label, **kw), X),
                   (lambda x, **kw: k3.lm_head_xent_grad(x, W, label, lse_x, **kw), X),
                   (lambda x, **kw: k3.lm_head_distill(x, W, ids, top, **kw), X),
                   (lambda x, **kw: k3.lm_head_distill_grad(x, W, ids, top, lse_d, **kw), X)][which]
    want = call(first)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

    def handed_out_again(use):
        temporary = first.clone()
        at = temporary.data_ptr()
        torch.cuda.synchronize()
        use(temporary)
        del temporary
        again = [torch.empty_like(first) for _ in range(8)]
        return at in [t.data_ptr() for t in again]

    got = []

    def on_the_side(x):
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)                 # a tenth of a second, ahead of the call
        got.append(call(x, stream=side))

    assert handed_out_again(lambda x: None)
    assert not handed_out_again(on_the_side)
    side.synchronize()
    for a, b in zip(got[0], want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_model_in_torch_goes_on_from_the_gradients(k3):
    """Parameters that require grad: the loss carries no graph, X.backward(dX) takes the gradient into
    the model that made X, dW is the head's."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((40, 64), generator=gen, device="cuda")
    trunk = torch.nn.Parameter(torch.randn((128, 64), generator=gen, device="cuda") / 8)
    head = torch.nn.Parameter((torch.randn((500, 128), generator=gen, device="cuda") / 11).bfloat16())
    label = torch.randint(-1, 500, (40,), generator=gen, device="cuda").int()
    X = (x @ trunk.T).bfloat16()
    loss, lse = k3.lm_head_xent(X, head, label)
    dX, head.grad = k3.lm_head_xent_grad(X, head, label, lse)
    assert not loss.requires_grad and not dX.requires_grad
    X.backward(dX)
    assert torch.equal(trunk.grad, torch.autograd.grad((x @ trunk.T).bfloat16(), trunk, dX)[0])
    assert float(trunk.grad.norm()) > 0 and head.grad.shape == head.shape
    # the same as from tensors that require none
    d, w = k3.lm_head_xent_grad(X.detach(), head.detach(), label, lse)
    assert torch.equal(d, dX) and torch.equal(w, head.grad)
