"""fr_recurrence, fr_recurrence_backward and fr_markov_product against the row-by-row statement in 64 bits.

Bounds.  Let u be the unit round-off of the wide type (2^-53 for f64 data, 2^-24 otherwise) and z_t = |a_t| z_{t-1} + |c_t x_t| the size of
the terms that make up h_t.  A gate is the exponential of a stored number: relative error at most 4 u with the library's exp, expm1 and sqrt, whatever the
number (the argument is exact).  Each row multiplies and adds once, and joining stretches of rows multiplies the same gates in another order, so a
term that is L rows old carries at most L (4 + 2) u + 8 u: |error| <= (6 L + 8) u z_t with L the rows of the sequence.  A 16-bit result is
rounded once more, half a step: eps / 2 |h|.  The backward pass adds a few products to that (16 u) and the sum over the channels of a gate (width u)."""
import ctypes

import numpy as np
import pytest

import plain_operators as P

pytestmark = pytest.mark.gpu

UNIT = {"f64": 2.0**-53, "f32": 2.0**-24, "bf16": 2.0**-24, "f16": 2.0**-24}
HALF_STEP = {"f64": 0.0, "f32": 0.0, "bf16": 2.0**-8, "f16": 2.0**-11}
TINY = {"f64": 1e-300, "f32": 1e-37, "bf16": 1e-37, "f16": 2.0**-25}  # half the smallest step of a subnormal 16-bit result


def torch_types():
    import torch

    return {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def put(values, layout, dtype, pad=0):
    """device matrix in a layout, its leading dimension `pad` beyond the least"""
    import torch

    r, c = values.shape
    v = torch.as_tensor(np.asarray(values), dtype=torch.float64)
    if layout == "row":
        m = torch.full((r, c + pad), float("nan"), dtype=dtype, device="cuda")[:, :c]
    else:
        m = torch.full((c, r + pad), float("nan"), dtype=dtype, device="cuda")[:, :r].t()
    m.copy_(v.to("cuda"))
    return m


def host(t):
    return t.detach().double().cpu().numpy()


@pytest.fixture(scope="module")
def tctx():
    import torch
    from friedrich_amd.device import Context

    c = Context()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


def problem(rng, n, d, cols, nseq, form, dtype, layout, pad=0):
    t = torch_types()
    wide = t["f64"] if dtype == "f64" else t["f32"]
    log_gate = -np.exp(rng.uniform(-7, 1, (1, cols))) * rng.uniform(0.02, 1.0, (n, cols))
    gate = put(np.exp(log_gate) if form == "value" else log_gate, layout, t[dtype], pad)
    x = put(rng.standard_normal((n, d)), layout, t[dtype], pad)
    h0 = put(rng.standard_normal((nseq, d)), layout, wide, pad)
    return gate, x, h0, wide


def check(got, want, size, rel, half, what, tiny=0.0):
    got, bound = host(got), rel * size + half * np.abs(want) + tiny
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} beyond the bound, worst {np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)):.3g} times"


SIZES = [  # n, d, gate columns
    (1, 1, 1), (1, 5, 5), (2, 3, 1), (15, 4, 2), (16, 1, 1), (17, 66, 33), (64, 64, 64), (130, 7, 1), (257, 12, 3), (1023, 3, 3), (2049, 1, 1), (5001, 2, 1), (300, 260, 4),
]


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("form", ["value", "log", "stationary"])
def test_one_sequence(tctx, form, dtype, layout):
    rng = np.random.default_rng(1)
    for n, d, cols in SIZES:
        gate, x, h0, wide = problem(rng, n, d, cols, 1, form, dtype, layout, pad=n % 3)
        h, last = tctx.recurrence(gate, x, form=form, h0=h0)
        want, want_last, z, zl = P.recurrence(form, host(gate), host(x), None, host(h0))
        rel = (6 * n + 8) * UNIT[dtype]
        check(h, want, z, rel, HALF_STEP[dtype], ("h", n, d, cols), TINY[dtype])
        check(last, want_last, zl, rel, 0.0, ("last", n, d, cols))


RAGGED = [
    list(range(0, 300)), [0] * 90 + [1] * 80 + list(range(2, 140)), list(range(0, 1500, 3)) + [4000],
    [0, 1], [0, 1, 2, 3, 4], [0, 0, 5, 5, 5, 9], [3, 3, 40, 41, 41, 100], [0, 700, 1400], [0, 64, 128, 128, 129, 193], [0, 2049, 2050, 4097], [5, 5], [0, 0, 0, 0],
    [0, 16, 32, 48, 64], [0, 511, 1536, 3000],
]


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", ["f64", "bf16"])
def test_packed_sequences_forward_and_backward(tctx, dtype, layout):
    """empty sequences, rows in front of the first and behind the last, starts on and off every boundary"""
    import torch

    t = torch_types()[dtype]
    rng = np.random.default_rng(2)
    for i, cuts in enumerate(RAGGED):
        for d, cols in ((1, 1), (6, 3), (70, 1)):
            form = ("value", "log", "stationary")[i % 3]
            n, nseq = cuts[-1] + (7 if i % 2 else 0), len(cuts) - 1
            gate, x, h0, wide = problem(rng, n, d, cols, nseq, form, dtype, layout)
            offsets = torch.tensor(cuts, dtype=torch.int64, device="cuda")
            h, last = put(np.full((n, d), 7.0), layout, t), put(np.full((nseq, d), 7.0), layout, wide)
            tctx.recurrence(gate, x, form=form, offsets=offsets, h0=h0, out=h, last=last)
            want, want_last, z, zl = P.recurrence(form, host(gate), host(x), cuts, host(h0))
            longest = max(b - a for a, b in zip(cuts[:-1], cuts[1:]))
            rel = (6 * longest + 8) * UNIT[dtype]
            inside = ~np.isnan(want[:, 0]) if n else np.zeros(0, bool)
            assert np.all(host(h)[~inside] == 7.0), ("rows of no sequence were written", cuts)
            check(h[torch.from_numpy(inside).cuda()], want[inside], z[inside], rel, HALF_STEP[dtype], ("h", cuts, d), TINY[dtype])
            check(last, want_last, zl, rel, 0.0, ("last", cuts, d))

            dh, dlast = put(rng.standard_normal((n, d)), layout, t), put(rng.standard_normal((nseq, d)), layout, wide)
            dgate, dx, dh0 = put(np.full((n, cols), 7.0), layout, t), put(np.full((n, d), 7.0), layout, t), put(np.full((nseq, d), 7.0), layout, wide)
            tctx.recurrence_backward(gate, x, h, dh, form=form, offsets=offsets, h0=h0, dlast=dlast, dgate=dgate, dx=dx, dh0=dh0)
            ref = P.recurrence_backward(form, host(gate), host(x), host(h), host(dh), cuts, host(h0), host(dlast))
            for name, got in (("dgate", dgate), ("dx", dx)):
                assert np.all(host(got)[~inside] == 7.0), (name, "rows of no sequence were written", cuts)
                check(got[torch.from_numpy(inside).cuda()], ref[name][0][inside], ref[name][1][inside], (6 * longest + 24 + d // cols) * UNIT[dtype], HALF_STEP[dtype],
                      (name, cuts, d), TINY[dtype])
            check(dh0, *ref["dh0"], rel, 0.0, ("dh0", cuts, d))


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("form", ["value", "log", "stationary"])
def test_gradients_of_one_sequence(tctx, form, dtype, layout):
    rng = np.random.default_rng(3)
    for n, d, cols in SIZES:
        gate, x, h0, wide = problem(rng, n, d, cols, 1, form, dtype, layout, pad=n % 2)
        h, _ = tctx.recurrence(gate, x, form=form, h0=h0)
        dh, dlast = put(rng.standard_normal((n, d)), layout, x.dtype), put(rng.standard_normal((1, d)), layout, wide)
        got = tctx.recurrence_backward(gate, x, h, dh, form=form, h0=h0, dlast=dlast)
        ref = P.recurrence_backward(form, host(gate), host(x), host(h), host(dh), None, host(h0), host(dlast))
        for name, g in zip(("dgate", "dx", "dh0"), got):
            check(g, *ref[name], (6 * n + 24 + d // cols) * UNIT[dtype], 0.0 if name == "dh0" else HALF_STEP[dtype], (name, n, d, cols), 0.0 if name == "dh0" else TINY[dtype])


@pytest.mark.parametrize("form", ["value", "log", "stationary"])
@pytest.mark.parametrize("dtype,n,d,cols", [("bf16", 8200, 1024, 1024), ("bf16", 8200, 516, 129), ("f16", 8200, 520, 65), ("f32", 8200, 520, 65), ("f32", 600, 512, 512), ("bf16", 600, 512, 512)])
def test_several_channels_a_lane(tctx, dtype, n, d, cols, form):
    """rows layout, calls large enough for (or, of few rows, with) more than one channel a lane; sequences that begin anywhere"""
    import torch

    t = torch_types()[dtype]
    rng = np.random.default_rng(15)
    cuts = [2, 2, 40, 257, 258, n // 2, n // 2 + 128, n - 3]
    nseq, longest = len(cuts) - 1, n // 2
    gate, x, h0, wide = problem(rng, n, d, cols, nseq, form, dtype, "row")
    offsets = torch.tensor(cuts, dtype=torch.int64, device="cuda")
    h, last = put(np.full((n, d), 7.0), "row", t), put(np.full((nseq, d), 7.0), "row", wide)
    tctx.recurrence(gate, x, form=form, offsets=offsets, h0=h0, out=h, last=last)
    want, want_last, z, zl = P.recurrence(form, host(gate), host(x), cuts, host(h0))
    rel, within = (6 * longest + 8) * UNIT[dtype], slice(cuts[0], cuts[-1])
    assert (h[: cuts[0]] == 7.0).all() and (h[cuts[-1] :] == 7.0).all()
    check(h[within], want[within], z[within], rel, HALF_STEP[dtype], "h", TINY[dtype])
    check(last, want_last, zl, rel, 0.0, "last")
    dh, dlast = put(rng.standard_normal((n, d)), "row", t), put(rng.standard_normal((nseq, d)), "row", wide)
    dgate, dx, dh0 = put(np.full((n, cols), 7.0), "row", t), put(np.full((n, d), 7.0), "row", t), put(np.full((nseq, d), 7.0), "row", wide)
    tctx.recurrence_backward(gate, x, h, dh, form=form, offsets=offsets, h0=h0, dlast=dlast, dgate=dgate, dx=dx, dh0=dh0)
    ref = P.recurrence_backward(form, host(gate), host(x), host(h), host(dh), cuts, host(h0), host(dlast))
    for name, got in (("dgate", dgate), ("dx", dx)):
        assert (got[: cuts[0]] == 7.0).all() and (got[cuts[-1] :] == 7.0).all(), name
        check(got[within], ref[name][0][within], ref[name][1][within], (6 * longest + 24 + d // cols) * UNIT[dtype], HALF_STEP[dtype], name, TINY[dtype])
    check(dh0, *ref["dh0"], rel, 0.0, "dh0")


def test_gradients_against_differences(tctx):
    """central differences of a scalar loss in f64: error h^2 times a third derivative of the order of the loss, and round-off over h"""
    import torch

    rng = np.random.default_rng(4)
    for form in ("value", "log", "stationary"):
        n, d, cols = 23, 4, 2
        gate, x, h0, _ = problem(rng, n, d, cols, 2, form, "f64", "col")
        offsets = torch.tensor([0, 9, n], dtype=torch.int64, device="cuda")
        w, wl = put(rng.standard_normal((n, d)), "col", x.dtype), put(rng.standard_normal((2, d)), "col", x.dtype)

        def loss():
            h, last = tctx.recurrence(gate, x, form=form, offsets=offsets, h0=h0)
            return float((h * w).sum() + (last * wl).sum()), h

        _, h = loss()
        grads = tctx.recurrence_backward(gate, x, h, w, form=form, offsets=offsets, h0=h0, dlast=wl)
        for t, g in ((gate, grads[0]), (x, grads[1]), (h0, grads[2])):
            for _ in range(12):
                i, j = int(rng.integers(t.shape[0])), int(rng.integers(t.shape[1]))
                if form == "stationary" and t is gate and float(t[i, j]) > -1e-3:
                    continue  # the slope of sqrt(1 - a^2) grows without bound towards a = 1
                step, was = 1e-6, float(t[i, j])
                t[i, j] = was + step
                up = loss()[0]
                t[i, j] = was - step
                down = loss()[0]
                t[i, j] = was
                assert abs((up - down) / (2 * step) - float(g[i, j])) <= 2e-6 * (1.0 + abs(float(g[i, j]))), (form, i, j)


def test_state_carried_between_calls_is_one_run(tctx):
    """rows given one after the other, the state handed on, and all at once: the same sequence"""
    import torch

    rng = np.random.default_rng(5)
    for dtype, layout in (("f64", "col"), ("bf16", "row")):
        n, d = 40, 33
        gate, x, h0, wide = problem(rng, n, d, d, 1, "log", dtype, layout)
        whole, last = tctx.recurrence(gate, x, h0=h0)
        state, rows = h0, []
        for r in range(n):
            y, state = tctx.recurrence(gate[r:r + 1], x[r:r + 1], h0=state)
            rows.append(y)
        want, want_last, z, zl = P.recurrence("log", host(gate), host(x), None, host(h0))
        rel = (6 * n + 8) * UNIT[dtype]
        check(torch.cat(rows), want, z, rel, HALF_STEP[dtype], "row by row", TINY[dtype])
        check(state, want_last, zl, rel, 0.0, "last state")
        check(whole, want, z, rel, HALF_STEP[dtype], "at once", TINY[dtype])


def test_no_states_no_rows_no_channels(tctx):
    import torch

    rng = np.random.default_rng(6)
    gate, x, h0, _ = problem(rng, 50, 3, 3, 1, "log", "f64", "col")
    h, last = tctx.recurrence(gate, x)
    want, want_last, z, zl = P.recurrence("log", host(gate), host(x), None, None)
    check(h, want, z, 308 * 2.0**-53, 0.0, "no h0")
    dg, dx, dh0 = tctx.recurrence_backward(gate, x, h, x)
    ref = P.recurrence_backward("log", host(gate), None, host(h), host(x), None, None, None)
    check(dg, *ref["dgate"], 325 * 2.0**-53, 0.0, "dgate, no states")
    none = torch.zeros(0, 3, dtype=torch.float64, device="cuda")
    y, state = tctx.recurrence(none, none, h0=h0)  # a sequence of no rows ends where it began
    assert y.shape == (0, 3) and torch.equal(state, h0)
    dg, dx, dh0 = tctx.recurrence_backward(none, none, none, none, dlast=h0)
    assert torch.equal(dh0, h0)
    thin = torch.zeros(5, 0, dtype=torch.float64, device="cuda")
    tctx.recurrence(torch.zeros(5, 1, dtype=torch.float64, device="cuda"), thin)


def test_in_place_and_odd_addresses(tctx):
    import torch

    rng = np.random.default_rng(7)
    for dtype in ("f64", "bf16", "f16"):
        for layout in ("row", "col"):
            n, d = 3001, 3
            gate, x, h0, wide = problem(rng, n, d, 1, 1, "log", dtype, layout)
            # the same data one element behind an aligned address
            room = torch.zeros(n * d + 1, dtype=x.dtype, device="cuda")
            y = room[1:].view(n, d) if layout == "row" else room[1:].view(d, n).t()
            y.copy_(x)
            h, last = tctx.recurrence(gate, x, h0=h0)
            out, last2 = tctx.recurrence(gate, y, h0=h0, out=y)
            assert torch.equal(out, h) and torch.equal(last, last2), (dtype, layout)
            dg, dx, dh0 = tctx.recurrence_backward(gate, None, h, x, h0=h0)
            y.copy_(x)
            dg2, dx2, dh02 = tctx.recurrence_backward(gate, None, h, y, h0=h0, dx=y)
            assert torch.equal(dg, dg2) and torch.equal(dx, y) and torch.equal(dh0, dh02), (dtype, layout)


def test_gates_of_zero_one_and_beyond(tctx):
    """a = 0 forgets, a = 1 sums, |a| > 1 and a < 0 are gates like any other; a log gate of -inf is a = 0; values of the stationary form at
    a = 1: nothing comes in, and the slope there is taken as 0"""
    import torch

    n = 200
    x = torch.ones(n, 1, dtype=torch.float64, device="cuda")
    one = torch.ones_like(x)
    h, _ = tctx.recurrence(one, x, form="value")
    assert torch.equal(h[:, 0], torch.arange(1, n + 1, dtype=torch.float64, device="cuda"))
    h, _ = tctx.recurrence(0 * one, x, form="value")
    assert torch.equal(h, x)
    h, _ = tctx.recurrence(-one, x, form="value")
    assert torch.equal(h[:, 0], torch.arange(1, n + 1, device="cuda").remainder(2).double())
    h, _ = tctx.recurrence(torch.full_like(x, -float("inf")), x, form="log")
    assert torch.equal(h, x)
    grow, _ = tctx.recurrence(torch.full_like(x, 1.5), x, form="value")
    want, _, z, _ = P.recurrence("value", np.full((n, 1), 1.5), host(x), None, None)
    check(grow, want, z, (6 * n + 8) * 2.0**-53, 0.0, "growing")
    h0 = torch.full((1, 1), 3.0, dtype=torch.float64, device="cuda")
    h, _ = tctx.recurrence(0 * one, x, form="stationary", h0=h0)
    assert torch.equal(h, torch.full_like(h, 3.0))
    dg, dx, dh0 = tctx.recurrence_backward(0 * one, x, h, one, form="stationary", h0=h0)
    assert torch.isfinite(dg).all() and torch.equal(dx, 0 * dx) and float(dh0) == n


@pytest.mark.parametrize("layout", ["row", "col"])
def test_what_is_not_finite_stays_in_its_sequence(tctx, layout):
    """a NaN or an infinity reaches the later rows of its own sequence (the earlier ones in the gradient) and no other"""
    import torch

    rng = np.random.default_rng(14)
    for dtype in ("f64", "f32", "bf16"):
        for d in (2, 300):
            cuts = [0, 5, 700, 701, 2500, 2600, 5000]
            n, nseq = cuts[-1], len(cuts) - 1
            gate, x, h0, wide = problem(rng, n, d, d, nseq, "log", dtype, layout)
            offsets = torch.tensor(cuts, dtype=torch.int64, device="cuda")
            clean, clean_last = tctx.recurrence(gate, x, offsets=offsets, h0=h0)
            dh = put(rng.standard_normal((n, d)), layout, x.dtype)
            clean_dx = tctx.recurrence_backward(gate, None, clean, dh, offsets=offsets, h0=h0)[1].clone()
            for value in (float("nan"), float("inf")):
                for row in (4, 300, 700, 2499, 4000):
                    s = max(i for i, c in enumerate(cuts) if c <= row)
                    x2, dh2 = x.clone(), dh.clone()
                    x2[row], dh2[row] = value, value
                    h, last = tctx.recurrence(gate, x2, offsets=offsets, h0=h0)
                    touched = torch.zeros(n, dtype=torch.bool, device="cuda")
                    touched[row:cuts[s + 1]] = True
                    assert torch.equal(h[~touched], clean[~touched]) and not torch.isfinite(h[row:cuts[s + 1]]).any(), (dtype, d, row)
                    other = [i for i in range(nseq) if i != s]
                    assert torch.equal(last[other], clean_last[other])
                    dx = tctx.recurrence_backward(gate, None, clean, dh2, offsets=offsets, h0=h0)[1]
                    touched[:] = False
                    touched[cuts[s]:row + 1] = True
                    assert torch.equal(dx[~touched], clean_dx[~touched]) and not torch.isfinite(dx[cuts[s]:row + 1]).any(), (dtype, d, row)


def test_host_arrays(tctx):
    rng = np.random.default_rng(8)
    for order in ("F", "C"):
        for dtype in (np.float64, np.float32, np.float16):
            n, d = 77, 6
            g = np.array(-rng.uniform(0.01, 2, (n, 2)), dtype=dtype, order=order)
            x = np.array(rng.standard_normal((n, d)), dtype=dtype, order=order)
            offsets = np.array([2, 30, 30, 70], dtype=np.int64)
            out = np.full((n, d), 5.0, dtype=dtype, order=order)
            h, last = tctx.recurrence(g, x, offsets=offsets, out=out)
            want, want_last, z, _ = P.recurrence("log", g, x, offsets, None)
            inside = ~np.isnan(want[:, 0])
            half = 2.0**-11 if dtype == np.float16 else 0.0
            u = 2.0**-53 if dtype == np.float64 else 2.0**-24
            assert np.all(np.abs(h[inside] - want[inside]) <= 250 * u * z[inside] + half * np.abs(want[inside]) + (2.0**-25 if half else 0.0))
            assert np.all(h[~inside] == 5.0)
            dg, dx, dh0 = tctx.recurrence_backward(g, x, h, x, offsets=offsets)
            ref = P.recurrence_backward("log", g, x, h, x, offsets, None, None)
            assert np.all(np.abs(dg[inside] - ref["dgate"][0][inside]) <= 280 * u * ref["dgate"][1][inside] + half * np.abs(ref["dgate"][0][inside]) + (2.0**-25 if half else 0.0))


def test_on_another_stream_and_in_a_captured_graph():
    """the context works on the stream it was given; two captured graphs and an eager call share nothing that a replay could disturb"""
    import torch
    from friedrich_amd.device import Context

    rng = np.random.default_rng(9)
    side = torch.cuda.Stream()
    c = Context()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        c.set_stream(side.cuda_stream)
        cases = []
        for dtype, layout, n, d in (("f64", "col", 9000, 2), ("bf16", "row", 700, 130)):
            gate, x, h0, wide = problem(rng, n, d, 1, 1, "stationary", dtype, layout)
            dh = put(rng.standard_normal((n, d)), layout, x.dtype)
            out = [t.clone() for t in (x, h0, gate, x, h0)]
            # (clone of a transposed matrix keeps its strides)
            def call(gate=gate, x=x, h0=h0, dh=dh, out=out):
                c.recurrence(gate, x, form="stationary", h0=h0, out=out[0], last=out[1])
                c.recurrence_backward(gate, x, out[0], dh, form="stationary", h0=h0, dgate=out[2], dx=out[3], dh0=out[4])

            cases.append((call, x, out))
        graphs = []
        for call, x, out in cases:
            call()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call()
            graphs.append(g)
        for trial in range(4):
            for (call, x, out), g in zip(cases, graphs):
                x.copy_(torch.randn(x.shape, device="cuda", dtype=torch.float32).to(x.dtype))
                call()
                side.synchronize()
                eager = [t.clone() for t in out]
                for t in out:
                    t.zero_()
                for other in graphs:  # (the other case's replay must not reach into this one's workspace)
                    other.replay()
                side.synchronize()
                for a, b in zip(eager, out):
                    assert torch.equal(a, b), trial
        # a captured call cannot take host memory
        g = torch.cuda.CUDAGraph()
        bad = None
        with torch.cuda.graph(g, stream=side):
            try:
                c.recurrence(np.zeros((4, 1)), np.ones((4, 1)))
            except RuntimeError as e:
                bad = str(e)
        assert bad and "captured" in bad
    torch.cuda.synchronize()
    del graphs, g
    c.close()


def test_two_contexts_at_once():
    """calls of two threads, each with a context and a stream of its own, in which tiles wait for one another"""
    import threading

    import torch
    from friedrich_amd.device import Context

    rng = np.random.default_rng(15)
    work, errors = [], []
    for dtype, layout, n, d in (("f64", "col", 600000, 2), ("bf16", "row", 20000, 300)):
        gate, x, h0, wide = problem(rng, n, d, d, 1, "log", dtype, layout)
        work.append((gate, x, h0, put(rng.standard_normal((n, d)), layout, x.dtype)))
    torch.cuda.synchronize()

    def run(gate, x, h0, dh, results):
        try:
            c, s = Context(), torch.cuda.Stream()
            c.set_stream(s.cuda_stream)
            with torch.cuda.stream(s):
                for _ in range(6):
                    h, last = c.recurrence(gate, x, h0=h0)
                    results.append((h, last) + tuple(c.recurrence_backward(gate, x, h, dh, h0=h0)))
                s.synchronize()
            c.close()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    alone, together = [[], []], [[], []]
    for w, r in zip(work, alone):
        run(*w, r)
    threads = [threading.Thread(target=run, args=(*w, r)) for w, r in zip(work, together)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(alone, together):
        assert len(b) == 6
        for r in b:
            assert all(torch.equal(p, q) for p, q in zip(a[0], r))


def test_the_same_call_gives_the_same_bits(tctx):
    import torch

    rng = np.random.default_rng(10)
    for dtype, layout, n, d, cols in (("f64", "col", 200001, 2, 1), ("bf16", "row", 4001, 256, 4), ("f32", "row", 100000, 3, 1)):
        gate, x, h0, wide = problem(rng, n, d, cols, 1, "log", dtype, layout)
        dh = put(rng.standard_normal((n, d)), layout, x.dtype)
        runs = []
        for _ in range(3):
            h, last = tctx.recurrence(gate, x, h0=h0)
            runs.append((h, last) + tuple(tctx.recurrence_backward(gate, x, h, dh, h0=h0)))
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_long_sequences(tctx):
    """a million rows of gates near 1 in f64, and lengths around the sizes that the work is cut at, against the same rows in halves"""
    import torch

    rng = np.random.default_rng(11)
    for n in (1 << 20, (1 << 20) + 1, 999983):
        gate, x, h0, _ = problem(rng, n, 1, 1, 1, "log", "f64", "col")
        gate.mul_(0.01)
        h, last = tctx.recurrence(gate, x, h0=h0)
        a, c = P.gates("log", host(gate), 1)
        v, want = float(h0[0, 0]), np.empty(n)
        for i, (ai, xi) in enumerate(zip(a[:, 0].tolist(), host(x)[:, 0].tolist())):
            v = ai * v + xi
            want[i] = v
        z, zs = abs(float(h0[0, 0])), np.empty(n)
        for i, (ai, xi) in enumerate(zip(a[:, 0].tolist(), np.abs(host(x)[:, 0]).tolist())):
            z = ai * z + xi
            zs[i] = z
        # a term decays: its age at 1/e is 1 / (1 - a) rows, and no older than the sequence
        age = min(n, int(60 / (1 - a.max())) + 1)
        assert np.all(np.abs(host(h)[:, 0] - want) <= 2 * (6 * age + 8) * 2.0**-53 * zs)


@pytest.mark.parametrize("n,m", [(1, 1), (2, 3), (63, 1), (500, 4), (1500, 7)])
def test_markov_product_is_gram_times_v(tctx, n, m):
    """(K + noise^2 I) V by the recurrence against fr_gram and fr_gemm, ties among the inputs included.  Each covariance differs by the
    rounding of its exponent (sums of gaps against a difference: n u times the exponent, at most n u for factors above e^-1, less below) and each
    entry sums n terms: 8 n u of the terms' size."""
    rng = np.random.default_rng(12)
    t = np.sort(np.round(rng.uniform(0, 30, n), 2 if n > 100 else 6))
    V = np.asfortranarray(rng.standard_normal((n, m)))
    kernel, noise = ("exponential", 1.1, 0.7), 0.3
    got = tctx.markov_product(kernel, t, V, noise=noise)
    K = tctx.gram(kernel, t.reshape(-1, 1), t.reshape(-1, 1))
    want = tctx.gemm(K, V) + noise**2 * V
    size = np.abs(K) @ np.abs(V) + noise**2 * np.abs(V)
    assert np.all(np.abs(got - want) <= (8 * n + 32) * 2.0**-53 * size)


def test_prior_path_has_the_kernels_covariance(tctx):
    """the stationary form on unit vectors gives the columns of a factor of the covariance matrix: paths x paths^T = gram"""
    rng = np.random.default_rng(13)
    n, ls, ampl = 60, 0.9, 1.4
    t = np.sort(rng.uniform(0, 10, n))
    gate = np.empty((n, 1), order="F")
    gate[1:, 0] = -np.diff(t) / (2 * ls * ls)
    gate[0, 0] = -np.inf  # the first value is drawn from the stationary law itself
    x = np.asfortranarray(np.eye(n))
    h, _ = tctx.recurrence(gate, x, form="stationary")
    K = tctx.gram(("exponential", ls, ampl), t.reshape(-1, 1), t.reshape(-1, 1))
    assert np.max(np.abs(ampl * h @ h.T - K)) <= 40 * n * 2.0**-53 * ampl


def test_refusals(tctx):
    import torch
    from friedrich_amd import _capi as C
    from friedrich_amd.device import FriedrichError

    x = torch.zeros(8, 6, dtype=torch.float64, device="cuda").t()  # 6 x 8, column-major
    g = torch.zeros(8, 6, dtype=torch.float64, device="cuda").t()
    lib, h = tctx.lib, tctx.h

    def call(dtype=0, layout=0, form=1, n=6, d=8, gate=g.data_ptr(), cols=8, ldg=6, xp=x.data_ptr(), ldx=6, offsets=None, nseq=1, out=x.data_ptr(), ldh=6):
        return lib.fr_recurrence(h, dtype, layout, form, n, d, gate, cols, ldg, xp, ldx, offsets, nseq, None, 0, out, ldh, None, 0)

    assert call() == C.FR_OK
    for kw, status in [(dict(dtype=4), C.FR_INVALID_ARGUMENT), (dict(dtype=-1), C.FR_INVALID_ARGUMENT), (dict(layout=2), C.FR_INVALID_ARGUMENT),
                       (dict(form=3), C.FR_INVALID_ARGUMENT), (dict(n=-1), C.FR_SHAPE), (dict(cols=3), C.FR_SHAPE), (dict(cols=0), C.FR_SHAPE),
                       (dict(nseq=2), C.FR_INVALID_ARGUMENT), (dict(nseq=-1), C.FR_SHAPE), (dict(ldx=5), C.FR_SHAPE), (dict(ldg=5), C.FR_SHAPE), (dict(ldh=5), C.FR_SHAPE),
                       (dict(gate=None), C.FR_INVALID_ARGUMENT), (dict(xp=None), C.FR_INVALID_ARGUMENT), (dict(out=None), C.FR_INVALID_ARGUMENT),
                       (dict(xp=x.data_ptr() + 4), C.FR_INVALID_ARGUMENT)]:
        assert call(**kw) == status, kw
    for cuts in ([0, 7], [-1, 6], [0, 4, 3, 6]):
        off = np.array(cuts, dtype=np.int64)
        assert call(offsets=off.ctypes.data, nseq=len(cuts) - 1) == C.FR_SHAPE, cuts
    # offsets in device memory are kept inside the rows there are
    off = torch.tensor([-5, 3, 1 << 40], dtype=torch.int64, device="cuda")
    assert call(offsets=off.data_ptr(), nseq=2) == C.FR_OK
    torch.cuda.synchronize()
    with pytest.raises(FriedrichError) as e:
        tctx.markov_product(("matern1", 1.0, 1.0), np.arange(4.0), np.ones((4, 1), order="F"))
    assert e.value.status == C.FR_UNSUPPORTED_KERNEL
    with pytest.raises(FriedrichError) as e:
        tctx.markov_product(("exponential", 1.0, 1.0), np.array([0.0, 2.0, 1.0]), np.ones((3, 1), order="F"))
    assert e.value.status == C.FR_INVALID_ARGUMENT
    t = torch.tensor([0.0, 2.0, 1.0], dtype=torch.float64, device="cuda")
    assert torch.isnan(tctx.markov_product(("exponential", 1.0, 1.0), t, torch.ones(1, 3, dtype=torch.float64, device="cuda").t())).any()
