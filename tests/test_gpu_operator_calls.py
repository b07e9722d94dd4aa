"""What surrounds the operators past the cube: lost waits, workspaces, streams."""
import numpy as np
import pytest

from test_gpu_recurrence import host, problem, put, tctx, torch_types  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout,n,d", [("col", 60000, 2), ("row", 6000, 130)])
def test_a_lost_wait_is_an_error(monkeypatch, layout, n, d):
    """FRIEDRICH_AMD_TEST_WAIT_POLLS = 0: every tile that waits for others gives up at its first look.  The results are NaN, the kernels end as
    ever, and the call that waits for them says so -- the next one where the results stay on the device"""
    import torch
    from friedrich_amd import _capi as C
    from friedrich_amd.device import Context, FriedrichError

    rng = np.random.default_rng(63)
    gate, x, h0, _ = problem(rng, n, d, d, 1, "log", "f32", layout)
    monkeypatch.setenv("FRIEDRICH_AMD_TEST_WAIT_POLLS", "0")
    c = Context()
    monkeypatch.delenv("FRIEDRICH_AMD_TEST_WAIT_POLLS")
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    h, last = c.recurrence(gate, x, h0=h0)
    with pytest.raises(FriedrichError) as e:
        c.synchronize()
    assert e.value.status == C.FR_HIP_ERROR and torch.isnan(last).any()
    c.synchronize()  # (said once)
    c.recurrence(gate, x, h0=h0)
    torch.cuda.synchronize()
    with pytest.raises(FriedrichError) as e:  # the next operator's call
        c.route(torch.zeros(4, 4, device="cuda"), 1)
    assert e.value.status == C.FR_HIP_ERROR
    got, _ = c.route(torch.zeros(4, 4, device="cuda"), 1)
    assert (got == 0).all()
    with pytest.raises(FriedrichError) as e:  # host data: the call itself
        c.recurrence(*(np.array(host(t), dtype=np.float32, order="C" if layout == "row" else "F") for t in (gate, x)))
    assert e.value.status == C.FR_HIP_ERROR
    # calls whose rows lie in one tile (8 waves of 4 rows are the smallest) do not wait; a factorisation does not see the operators' word
    short = tuple(t[:32] for t in (gate, x))
    c.recurrence(*short)
    c.recurrence(gate, x, h0=h0)
    A = np.asfortranarray(rng.random((300, 3)))
    chol = c.cholesky_from_inputs(("squared_exp", 1.0, 1.0), A, 0.1)
    assert np.isfinite(chol.solve(np.ones(300))).all()
    chol.free()
    with pytest.raises(FriedrichError):
        c.synchronize()
    c.close()


def test_a_capture_leaves_buffers_of_other_sizes():
    """a captured call keeps its workspace for good: it takes one of about its size, not whatever is free"""
    import torch
    from friedrich_amd.device import Context, FriedrichError

    rng = np.random.default_rng(61)
    c, side = Context(), torch.cuda.Stream()
    gate, x, h0, _ = problem(rng, 9000, 2, 2, 1, "log", "f64", "col")
    out, last = torch.zeros_like(x), torch.zeros_like(h0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        c.set_stream(side.cuda_stream)
        A = np.asfortranarray(rng.random((3000, 200)))
        want = c.gram(("squared_exp", 1.0, 1.0), A, A)  # leaves buffers of 5 and 72 MB
        held = c.counter("pool_bytes")
        assert held > 70 << 20
        g = torch.cuda.CUDAGraph()
        refused = None
        with torch.cuda.graph(g, stream=side):
            try:
                c.recurrence(gate, x, h0=h0, out=out, last=last)
            except FriedrichError as e:
                refused = str(e)
        assert refused and "once outside" in refused
        c.recurrence(gate, x, h0=h0, out=out, last=last)
        side.synchronize()
        eager = out.clone()
        g2 = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g2, stream=side):
            c.recurrence(gate, x, h0=h0, out=out, last=last)
        for _ in range(3):
            out.zero_()
            g2.replay()
            side.synchronize()
            assert torch.equal(out, eager)
            assert np.array_equal(c.gram(("squared_exp", 1.0, 1.0), A, A), want)
        assert c.counter("pool_bytes") <= held + (2 << 20)  # (the large ones are free for calls of their size)
    torch.cuda.synchronize()
    del g, g2
    c.close()


def test_workspace_of_many_slots_and_few_points(tctx):  # noqa: F811
    """sums of pieces take about 256 MB at most, however many slots there are to an expert's few points"""
    import torch
    from friedrich_amd.device import Context

    rng = np.random.default_rng(62)
    c = Context()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    n, experts, m, k = 1000, 64, 1 << 19, 2
    X = put(rng.random((n, 1)), "col", torch.float64)
    Xq = put(rng.random((m, 1)), "col", torch.float64)
    offsets = torch.arange(experts + 1, device="cuda") * n // experts
    chosen = torch.randint(0, experts, (k, m), device="cuda", dtype=torch.int32).t()
    w = torch.rand(k, m, device="cuda", dtype=torch.float64).t()
    alpha = torch.randn(n, device="cuda", dtype=torch.float64)
    before = c.counter("pool_bytes")
    mean, slots = c.experts_predict(("squared_exp", 0.3, 1.0), X, alpha, offsets, Xq, chosen, w)
    own = 8 * m * k * (1 + 1 + 2)  # (query points packed, list and places, two pieces more than the bound)
    assert c.counter("pool_bytes") - before <= (256 << 20) + own + (4 << 20)
    # a sample against the definition: 16 points an expert and the exponential, 40 roundings in all at most
    for q in range(0, m, m // 50):
        for j in range(k):
            lo, hi = int(offsets[chosen[q, j]]), int(offsets[chosen[q, j] + 1])
            kx = torch.exp(-((X[lo:hi, 0] - Xq[q, 0]) ** 2) / (2 * 0.3 ** 2))
            assert abs(float(slots[q, j] - (kx * alpha[lo:hi]).sum())) <= 40 * 2.0**-52 * float((kx * alpha[lo:hi].abs()).sum())
    c.close()


def test_more_features_than_an_index_holds(tctx):  # noqa: F811
    """refused before anything is read"""
    import ctypes

    import torch
    from friedrich_amd import _capi as C

    z = torch.zeros(8, dtype=torch.float64, device="cuda")
    off = np.array([0, 1], dtype=np.int64)
    p, e = C.kprog(("squared_exp", 1.0, 1.0)), torch.zeros(1, dtype=torch.int32, device="cuda")
    at = z.data_ptr()
    d = (1 << 24) + 1
    st = tctx.lib.fr_experts_predict(tctx.h, ctypes.byref(p), at, 1, 1, d, at, off.ctypes.data, 1, at, 1, 1, e.data_ptr(), 1, at, 1, 1, None, at, None, 0)
    assert st == C.FR_SHAPE
    st = tctx.lib.fr_experts_backward(tctx.h, ctypes.byref(p), at, 1, 1, d, off.ctypes.data, 1, at, 1, 1, e.data_ptr(), 1, at, 1, 1, at, 1, at, at, 1, at)
    assert st == C.FR_SHAPE


def test_a_context_on_its_own_stream():
    """without set_stream: what torch has queued on its stream is there when the call reads it, and what the call wrote when torch does"""
    import torch
    from friedrich_amd.device import Context

    rng = np.random.default_rng(64)
    c = Context()
    gate, x, h0, _ = problem(rng, 20000, 3, 3, 4, "log", "f64", "row")
    offsets = torch.tensor([0, 100, 5000, 12000, 19000], dtype=torch.int64, device="cuda")
    z = put(rng.standard_normal((3000, 16)), "row", torch.float32)
    torch.cuda.synchronize()
    ref = Context()
    ref.set_stream(torch.cuda.current_stream().cuda_stream)
    want = ref.recurrence(gate, x, offsets=offsets, h0=h0)
    want_g = ref.recurrence_backward(gate, x, want[0], x, offsets=offsets, h0=h0)
    want_r = ref.route(z, 2)
    torch.cuda.synchronize()
    for _ in range(3):
        x2, z2 = torch.zeros_like(x), torch.zeros_like(z)
        torch.cuda._sleep(20_000_000)  # (clock ticks of a kernel that ends by itself: torch's stream is late)
        x2.copy_(x)
        z2.copy_(z)
        h, last = c.recurrence(gate, x2, offsets=offsets, h0=h0)
        h2, last2 = h + 0, last + 0
        assert torch.equal(h2, want[0]) and torch.equal(last2, want[1])
        torch.cuda._sleep(20_000_000)
        y = torch.zeros_like(x)
        y.copy_(x)
        got = c.recurrence_backward(gate, y, h, y, offsets=offsets, h0=h0)
        assert all(torch.equal(a + 0, b) for a, b in zip(got, want_g))
        e, w = c.route(z2, 2)
        assert torch.equal(e + 0, want_r[0]) and torch.equal(w + 0, want_r[1])
    c.close()
    ref.close()


@pytest.mark.parametrize("layout", ["row", "col"])
def test_states_are_not_carried_in_place(tctx, layout):  # noqa: F811
    """the states behind the sequences over those in front of them, and a product over its factor: memory that is read again after it
    has been written, so refused"""
    import torch
    from friedrich_amd import _capi as C
    from friedrich_amd.device import FriedrichError

    rng = np.random.default_rng(65)
    gate, x, h0, _ = problem(rng, 300, 5, 5, 1, "log", "f32", layout)
    V = put(rng.standard_normal((50, 2)), "col", torch.float64)
    t = torch.arange(50, dtype=torch.float64, device="cuda")
    refused = [lambda: tctx.recurrence(gate, x, h0=h0, last=h0), lambda: tctx.recurrence_backward(gate, x, x, x.clone(), dlast=h0, dh0=h0),
               lambda: tctx.markov_product(("exponential", 1.0, 1.0), t, V, out=V)]
    host_state = np.zeros((1, 5), np.float32, order="F")
    refused.append(lambda: tctx.recurrence(np.zeros((9, 5), np.float32, order="F"), np.ones((9, 5), np.float32, order="F"), h0=host_state, last=host_state))
    for call in refused:
        with pytest.raises(FriedrichError) as e:
            call()
        assert e.value.status == C.FR_INVALID_ARGUMENT
    before = h0.clone()
    _, last = tctx.recurrence(gate, x, h0=h0)
    assert torch.equal(h0, before) and not torch.equal(last, h0)
