"""What the binding of the recurrence, the router and the experts' product refuses before it calls the library (no GPU: the library is
replaced by a recorder), and what the entry points do without a context."""
import ctypes

import numpy as np
import pytest

from friedrich_amd import _capi as C
from friedrich_amd.device import Context, FriedrichError, _layout

NAMES = ("fr_recurrence", "fr_recurrence_backward", "fr_markov_product", "fr_route", "fr_route_backward", "fr_experts_predict", "fr_experts_backward")


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if not name.startswith("fr_"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, args))
            assert len(args) == len(C.SIGNATURES[name][1]), name
            return C.FR_OK

        return call


@pytest.fixture
def ctx():
    c = Context.__new__(Context)
    c.lib, c.h, c._children = Recorder(), 1, set()
    yield c
    c.h = None


def test_no_context():
    lib = C.load()
    for name in NAMES:
        args = []
        for t in C.SIGNATURES[name][1]:
            args.append(0.0 if t is ctypes.c_double else None if t in (ctypes.c_void_p, ctypes.POINTER(C.KProg)) else 0)
        assert getattr(lib, name)(*args) == C.FR_INVALID_ARGUMENT, name


def test_layouts():
    a = np.zeros((4, 3))
    assert _layout(a) == C.FR_LAYOUT_ROWMAJOR and _layout(np.asfortranarray(a)) == C.FR_LAYOUT_COLMAJOR
    assert _layout(a[:1]) == C.FR_LAYOUT_COLMAJOR and _layout(a[:1], None, a) == C.FR_LAYOUT_ROWMAJOR  # one row fits both: the next decides
    assert _layout(a[:, :1]) == C.FR_LAYOUT_ROWMAJOR  # a column of a row-major matrix is strided
    with pytest.raises(ValueError):
        _layout(np.zeros((4, 6))[:, ::2])
    with pytest.raises(ValueError):
        _layout(np.zeros(4))


def test_recurrence_arguments(ctx):
    g, x = np.zeros((5, 1)), np.zeros((5, 4))
    h, last = ctx.recurrence(g, x)
    name, args = ctx.lib.calls[-1]
    assert name == "fr_recurrence" and args[1:6] == (C.FR_F64, C.FR_LAYOUT_ROWMAJOR, 1, 5, 4) and h.shape == (5, 4) and last.shape == (1, 4)
    h, last = ctx.recurrence(g.astype(np.float16), x.astype(np.float16), offsets=np.array([0, 2, 5]))
    assert h.dtype == np.float16 and last.dtype == np.float32 and last.shape == (2, 4)
    ctx.recurrence_backward(g, None, x, x)
    assert ctx.lib.calls[-1][0] == "fr_recurrence_backward"
    for kw, error in [(dict(h0=np.zeros((2, 4))), FriedrichError), (dict(h0=np.zeros((1, 4), np.float32)), ValueError), (dict(out=np.zeros((5, 4), order="F")), ValueError),
                      (dict(out=np.zeros((5, 3))), FriedrichError), (dict(offsets=np.array([0, 5], np.int32)), ValueError), (dict(form="cubic"), KeyError),
                      (dict(last=np.zeros((3, 4))), FriedrichError)]:
        with pytest.raises(error):
            ctx.recurrence(g, x, **kw)
    with pytest.raises(ValueError):
        ctx.recurrence(g.astype(np.float32), x)
    with pytest.raises(ValueError):
        ctx.recurrence(g.astype(np.int32), x.astype(np.int32))
    with pytest.raises(FriedrichError):
        ctx.recurrence(np.zeros((4, 1)), x)
    with pytest.raises(FriedrichError):
        ctx.recurrence_backward(g, x, np.zeros((4, 4)), x)


def test_route_arguments(ctx):
    z = np.zeros((6, 8), np.float32)
    e, w = ctx.route(z, 2)
    assert e.dtype == np.int32 and w.dtype == np.float32 and e.shape == w.shape == (6, 2)
    assert ctx.lib.calls[-1][1][9:13] == (1, 1, 2, 1)  # groups, kept groups, slots, renormalise
    assert ctx.route_backward(z, e, w).shape == z.shape
    with pytest.raises(ValueError):
        ctx.route_backward(z, e.astype(np.int64), w)
    with pytest.raises(ValueError):
        ctx.route_backward(z, e, w.astype(np.float64))
    with pytest.raises(FriedrichError):
        ctx.route(z, 2, bias=np.zeros(7))
    with pytest.raises(FriedrichError):
        ctx.route(z, 2, counts=np.zeros(7, np.int64))
    with pytest.raises(KeyError):
        ctx.route(z, 2, score="tanh")


def test_experts_arguments(ctx):
    kernel = ("squared_exp", 1.0, 1.0)
    X, Xq = np.zeros((10, 3), order="F"), np.zeros((4, 3), order="F")
    off, e, w, alpha = np.array([0, 4, 10]), np.zeros((4, 2), np.int32, order="F"), np.zeros((4, 2), order="F"), np.zeros(10)
    mean, slots = ctx.experts_predict(kernel, X, alpha, off, Xq, e, w)
    assert mean.shape == (4,) and slots.shape == (4, 2) and slots.flags.f_contiguous
    dw, da = ctx.experts_backward(kernel, X, off, Xq, e, w, slots, mean)
    assert dw.shape == (4, 2) and da.shape == (10,)
    with pytest.raises(ValueError):
        ctx.experts_predict(kernel, np.ascontiguousarray(X), alpha, off, Xq, e, w)
    with pytest.raises(ValueError):
        ctx.experts_predict(kernel, X.astype(np.float32), alpha, off, Xq, e, w)
    with pytest.raises(FriedrichError):
        ctx.experts_predict(kernel, X, alpha[:9], off, Xq, e, w)
    with pytest.raises(FriedrichError):
        ctx.experts_predict(kernel, X, alpha, off, Xq[:, :2], e, w)
    with pytest.raises(ValueError):
        ctx.experts_predict(kernel, X, alpha, off.astype(np.int32), Xq, e, w)
    with pytest.raises(FriedrichError):
        ctx.markov_product(("exponential", 1.0, 1.0), np.zeros(5), np.zeros((4, 1), order="F"))
