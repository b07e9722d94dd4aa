"""What the binding of the operators past the cube does around a call on torch tensors (no GPU: the library is replaced by a recorder, tensors
in host memory say that they lie on the GPU)."""
import numpy as np
import pytest

from friedrich_amd.device import Context
from test_operator_arguments import Recorder

torch = pytest.importorskip("torch")
KERNEL = ("squared_exp", 1.0, 1.0)


class OnGpu(torch.Tensor):
    is_cuda = True


def there(*shape, dtype=torch.float64):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu)


def columns(rows, cols, dtype=torch.float64):
    return there(cols, rows, dtype=dtype).t()


@pytest.fixture
def ctx(monkeypatch):
    c = Context.__new__(Context)
    c.lib, c.h, c._children = Recorder(), 1, set()

    class Stream:
        def synchronize(self):
            c.lib.calls.append(("torch waits", ()))

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    yield c
    c.h = None


def calls(c):
    """one call of every operator on tensors"""
    x, g, off = there(5, 4), there(5, 1), there(3, dtype=torch.int64)
    X, Xq, e, w = columns(10, 3), columns(4, 3), columns(4, 2, torch.int32), columns(4, 2)
    v = [there(n) for n in (10, 4)]
    return {
        "fr_recurrence": lambda: c.recurrence(g, x, offsets=off),
        "fr_recurrence_backward": lambda: c.recurrence_backward(g, None, x, x, offsets=off),
        "fr_markov_product": lambda: c.markov_product(("exponential", 1.0, 1.0), v[0], columns(10, 2)),
        "fr_route": lambda: c.route(there(6, 8), 2),
        "fr_route_backward": lambda: c.route_backward(columns(4, 8), e, w),
        "fr_experts_predict": lambda: c.experts_predict(KERNEL, X, v[0], off, Xq, e, w),
        "fr_experts_backward": lambda: c.experts_backward(KERNEL, X, off, Xq, e, w, w, v[1]),
    }


def test_turns_on_the_contexts_own_stream(ctx):
    for name, call in calls(ctx).items():
        ctx.lib.calls.clear()
        call()
        assert [n for n, _ in ctx.lib.calls] == ["torch waits", name, "fr_ctx_synchronize"], name


def test_no_waits_on_a_stream_that_was_given(ctx):
    ctx.set_stream(0)
    for name, call in calls(ctx).items():
        ctx.lib.calls.clear()
        call()
        assert [n for n, _ in ctx.lib.calls] == [name], name


def test_no_waits_for_host_arrays(ctx):
    ctx.recurrence(np.zeros((5, 1)), np.zeros((5, 4)))
    ctx.route(np.zeros((6, 8)), 2)
    assert [n for n, _ in ctx.lib.calls] == ["fr_recurrence", "fr_route"]


def test_the_contexts_own_stream_cannot_be_captured(ctx, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for name, call in calls(ctx).items():
        with pytest.raises(ValueError, match="set_stream"):
            call()
    assert not ctx.lib.calls
    ctx.set_stream(0)
    for call in calls(ctx).values():
        call()


def test_gradients_are_not_lost_silently(ctx):
    """a call on tensors that autograd follows would return results without a graph: refused, allowed where autograd is off"""
    x, g = torch.zeros(5, 4, dtype=torch.float64, requires_grad=True), torch.zeros(5, 1, dtype=torch.float64)
    z = torch.zeros(6, 8, requires_grad=True)
    w = columns(4, 2).requires_grad_()
    refused = [lambda: ctx.recurrence(g, x), lambda: ctx.recurrence(g, x.detach(), h0=torch.zeros(1, 4, dtype=torch.float64, requires_grad=True)),
               lambda: ctx.recurrence_backward(g, None, x.detach(), x), lambda: ctx.route(z, 2),
               lambda: ctx.markov_product(("exponential", 1.0, 1.0), there(10), columns(10, 2).requires_grad_()),
               lambda: ctx.route_backward(columns(4, 8), columns(4, 2, torch.int32), w),
               lambda: ctx.experts_predict(KERNEL, columns(10, 3), there(10), there(3, dtype=torch.int64), columns(4, 3), columns(4, 2, torch.int32), w),
               lambda: ctx.experts_backward(KERNEL, columns(10, 3), there(3, dtype=torch.int64), columns(4, 3), columns(4, 2, torch.int32), w, columns(4, 2), there(4))]
    for call in refused:
        with pytest.raises(ValueError, match="autograd"):
            call()
    assert not ctx.lib.calls
    with torch.no_grad():
        for call in refused:
            call()

    class Paths(torch.autograd.Function):
        @staticmethod
        def forward(f, gate, x):
            h, _ = ctx.recurrence(gate, x)
            f.save_for_backward(gate, x, h)
            return h

        @staticmethod
        def backward(f, dh):
            gate, x, h = f.saved_tensors
            return ctx.recurrence_backward(gate, x, h, dh.contiguous())[:2]

    ctx.lib.calls.clear()
    Paths.apply(g.detach().requires_grad_(), x).sum().backward()
    assert [n for n, _ in ctx.lib.calls] == ["fr_recurrence", "fr_recurrence_backward"] and x.grad.shape == x.shape


def test_kernels_given_as_lists(ctx):
    """a spec is a sequence, as for the other calls that take one: lists, lists within tuples, a program made before"""
    from friedrich_amd import _capi as C

    X, Xq = np.zeros((10, 3), order="F"), np.zeros((4, 3), order="F")
    off, e, w = np.array([0, 4, 10]), np.zeros((4, 2), np.int32, order="F"), np.zeros((4, 2), order="F")
    for spec in (["squared_exp", 0.5, 2.0], ("sum", ["squared_exp", 0.5, 2.0], ("linear", 0.1)), C.kprog(("squared_exp", 0.5, 2.0))):
        ctx.experts_predict(spec, X, np.zeros(10), off, Xq, e, w)
        ctx.experts_backward(spec, X, off, Xq, e, w, w, np.zeros(4))
    assert [n for n, _ in ctx.lib.calls] == ["fr_experts_predict", "fr_experts_backward"] * 3


def test_inputs_of_a_markov_product(ctx):
    """inputs of another type or with gaps would be read beyond their end"""
    V = columns(10, 2)
    for t in (there(10, dtype=torch.float32), there(20)[::2], there(10, dtype=torch.float16)):
        with pytest.raises(ValueError, match="t: "):
            ctx.markov_product(("exponential", 1.0, 1.0), t, V)
    assert not ctx.lib.calls
    for t in (there(10), there(10, 1), np.arange(10), np.arange(20.0)[::2]):
        ctx.markov_product(("exponential", 1.0, 1.0), t, V)
