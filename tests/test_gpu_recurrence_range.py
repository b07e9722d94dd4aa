"""fr_recurrence where gates grow, and gates shared by numbers of channels that no workgroup's lanes divide.  Bounds as in
test_gpu_recurrence.py: (6 L + 8) u of the terms' size for L rows, 16 u more backward, and what is said at a test."""
import numpy as np
import pytest

import plain_operators as P
from test_gpu_recurrence import HALF_STEP, TINY, UNIT, check, host, put, tctx, torch_types  # noqa: F401

pytestmark = pytest.mark.gpu

# layout, channels, gate columns: a gate a channel, shared gates, one channel, several channels a lane
SHAPES = [("row", 70, 70), ("row", 70, 1), ("row", 256, 2), ("row", 3, 1), ("row", 1, 1), ("col", 1, 1), ("col", 3, 3), ("col", 6, 1)]


@pytest.mark.parametrize("layout,d,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["value", "log"])
def test_nothing_grows_to_nothing(tctx, form, dtype, layout, d, cols):  # noqa: F811
    """gates beyond 1 over a state of 0, for more rows than their product has a number for: row by row the state stays 0"""
    rng = np.random.default_rng(51)
    t = torch_types()[dtype]
    for n in (300, 5000, 40000):
        gate = put(np.full((n, cols), 2.0 if form == "value" else 0.75), layout, t)
        x = np.zeros((n, d))
        x[n - 20:] = rng.standard_normal((20, d))
        x = put(x, layout, t)
        h, last = tctx.recurrence(gate, x, form=form)
        tail = slice(n - 20, n)
        want, want_last, z, zl = P.recurrence(form, host(gate)[tail], host(x)[tail], None, None)
        assert (h[: n - 20] == 0).all(), (n, "rows of nothing")
        check(h[tail], want, z, 128 * UNIT[dtype], HALF_STEP[dtype], ("h", n))
        check(last, want_last, zl, 128 * UNIT[dtype], 0.0, ("last", n))
        # the gradient runs the other way: only the first rows have one
        dh = np.zeros((n, d))
        dh[:20] = rng.standard_normal((20, d))
        dh = put(dh, layout, t)
        hb = put(rng.standard_normal((n, d)), layout, t)
        dg, dx, dh0 = tctx.recurrence_backward(gate, None, hb, dh, form=form)
        ref = P.recurrence_backward(form, host(gate)[:20], None, host(hb)[:20], host(dh)[:20], None, None, None)
        assert (dg[20:] == 0).all() and (dx[20:] == 0).all(), n
        check(dg[:20], *ref["dgate"], (6 * 20 + 24 + d // cols) * UNIT[dtype], HALF_STEP[dtype], ("dgate", n))
        check(dx[:20], *ref["dx"], 144 * UNIT[dtype], HALF_STEP[dtype], ("dx", n))
        check(dh0, *ref["dh0"], 144 * UNIT[dtype], 0.0, ("dh0", n))


@pytest.mark.parametrize("layout,d,cols", SHAPES)
def test_a_forgotten_state_does_not_grow(tctx, layout, d, cols):  # noqa: F811
    """a state, a gate of 0, and gates beyond 1 over nothing behind it"""
    rng = np.random.default_rng(52)
    t = torch_types()["f32"]
    for n, at in ((5000, 1000), (5000, 4096), (40000, 20000), (40000, 131)):
        g, x = np.full((n, cols), 0.5), np.ones((n, d))
        g[at], x[at:n - 20] = 0.0, 0.0
        g[at + 1:] = 2.0
        x[n - 20:] = rng.standard_normal((20, d))
        gate, x = put(g, layout, t), put(x, layout, t)
        h, last = tctx.recurrence(gate, x, form="value")
        want, want_last, z, zl = P.recurrence("value", host(gate), host(x), None, None)
        assert (h[at:n - 20] == 0).all(), (n, at)
        check(h, want, z, 8 * 64 * UNIT["f32"], 0.0, ("h", n, at), TINY["f32"])
        check(last, want_last, zl, 128 * UNIT["f32"], 0.0, ("last", n, at))


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("layout,n,d,cols", [("row", 3, 3000, 1), ("row", 5, 2000, 2), ("row", 1400, 3000, 1), ("row", 9, 4097, 1), ("col", 40, 4097, 1), ("col", 700, 1002, 1)])
def test_gates_of_thousands_of_channels(tctx, dtype, layout, n, d, cols):  # noqa: F811
    """the gradient of a gate that many channels share, terms all alike (a running sum of them rounds the same way every time: thousands of
    half steps).  A term is off by the gate's 4 u twice and five roundings, those it carries from rows behind it weigh a / (1 - a)^2 = 0.06 of 6 u a
    row; the sum may add the roundings of a tree: 6 of a wave and 8 of the parts.  Together less than 32 u."""
    t = torch_types()
    wide = t["f64"] if dtype == "f64" else t["f32"]
    gate = put(np.full((n, cols), -3.0), layout, t[dtype])
    h, dh, h0 = put(np.full((n, d), 1.1), layout, t[dtype]), put(np.full((n, d), 0.7), layout, t[dtype]), put(np.full((1, d), 1.3), layout, wide)
    dg, _, _ = tctx.recurrence_backward(gate, None, h, dh, form="log", h0=h0)
    g, want = 0.0, np.empty((n, cols))
    a, y = np.exp(-3.0), float(dh[0, 0])
    for r in range(n - 1, -1, -1):
        g = y + a * g
        want[r] = (d // cols) * (g * float(h[0, 0] if r else h0[0, 0]) * a)
    check(dg, want, want, 32 * UNIT[dtype], HALF_STEP[dtype], ("dgate", n, d))
