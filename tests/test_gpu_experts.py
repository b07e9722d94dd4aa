"""fr_route, fr_route_backward, fr_experts_predict and fr_experts_backward against the plain statements in 64 bits.

Bounds.  u = 2^-53.  A score is an exponential (4 u with the library's exp) over a sum of E of them (E u) and the difference in front of it (exact to
u times the exponent, at most 60 here before the score itself vanishes against the sum): 80 u + E u; weights add a division and a sum over k.
Choices have to be equal.  f32 weights are rounded once, half a step 2^-24; 16-bit gradients half a step of theirs.
A covariance is worked out from d squared differences (d + 2 roundings of the exponent, which is at most `arg` on the inputs used) and an
exponential; a sum of c terms adds c u: (c + (d + 8)(1 + arg) + 16) u times the terms' size."""
import numpy as np
import pytest

import plain_operators as P
from test_gpu_recurrence import HALF_STEP, TINY, host, put, tctx, torch_types  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0**-53
# rows, experts, k, groups, kept groups
ROUTES = [(1, 1, 1, 1, 1), (3, 2, 2, 1, 1), (5, 64, 2, 1, 1), (7, 65, 3, 1, 1), (33, 16, 4, 4, 2), (64, 128, 8, 1, 1), (130, 256, 8, 8, 4), (9, 257, 5, 1, 1),
          (21, 300, 6, 3, 2), (17, 512, 8, 16, 3), (4, 1024, 64, 64, 7), (257, 24, 1, 24, 5), (66, 60, 20, 1, 1), (5, 7, 7, 7, 7)]


def weights_bound(dtype, experts, k, want, renormalise):
    half = 0.0 if dtype == "f64" else 2.0**-24
    return ((80 + experts + 2 * k) * 2 * U + half) * np.abs(want) + 1e-300 + (0.0 if dtype == "f64" else 2.0**-150)


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(tctx, score, dtype, layout):  # noqa: F811
    import torch

    rng = np.random.default_rng(21)
    for i, (n, experts, k, groups, kept) in enumerate(ROUTES):
        for biased in (False, True):
            renormalise, scale = bool(i & 1), 1.0 if i % 3 else 2.5
            z = 2.0 * rng.standard_normal((n, experts))
            if i % 4 == 1:
                z[rng.random((n, experts)) < 0.4] = -np.inf
            logits = put(z, layout, torch_types()[dtype], i % 3)
            bias = torch.from_numpy(0.2 * rng.standard_normal(experts)).cuda() if biased else None
            counts = torch.full((experts,), -1, dtype=torch.int64, device="cuda")
            got, w = tctx.route(logits, k, score=score, bias=bias, groups=groups, top_groups=kept, renormalise=renormalise, scale=scale, counts=counts)
            want, want_w, want_c = P.route(score, host(logits), None if bias is None else host(bias), groups, kept, k, renormalise, scale)
            assert np.array_equal(got.cpu().numpy(), want), (n, experts, k, biased)
            assert np.all(np.abs(host(w) - want_w) <= weights_bound(dtype, experts, k, want_w, renormalise)), (n, experts, k, biased)
            assert np.array_equal(counts.cpu().numpy(), want_c)


def test_route_many_rows(tctx):  # noqa: F811
    """the way of many rows: keys in 32 bits, rows that they do not decide in 64 -- ties of logits, of logits with a bias, biases that differ in
    their last bits only, values whose scores saturate, groups that are alike; choices checked against 64-bit scores by sorting"""
    import torch

    rng = np.random.default_rng(30)
    n = 20000
    for i, (experts, k, groups, kept, dtype, score) in enumerate([(256, 8, 8, 4, "f32", "sigmoid"), (64, 2, 1, 1, "bf16", "softmax"), (100, 5, 1, 1, "f64", "sigmoid"),
                                                                  (32, 8, 4, 2, "bf16", "sigmoid"), (512, 6, 1, 1, "f32", "softmax"), (16, 1, 2, 1, "f16", "softmax")]):
        z = rng.standard_normal((n, experts)) * np.where(np.arange(n) % 3 == 0, 0.0, np.where(np.arange(n) % 3 == 1, 2.0, 20.0))[:, None]
        z[5::7] = np.round(z[5::7])  # ties
        z[rng.random((n, experts)) < 0.02] = -np.inf
        z[11], z[12, 3] = -np.inf, np.nan
        if dtype == "f64":  # the type's lowest values are values: only -inf closes
            z[13], z[14, ::2], z[15, 1:] = np.finfo(np.float64).min, -1e300, -1e39
        flat = np.zeros(experts)
        close = 0.25 + 2.0**-40 * rng.integers(0, 4, experts)
        for bias in (None, flat, close, 0.1 * rng.standard_normal(experts)):
            for layout in ("row", "col"):
                logits = put(z, layout, torch_types()[dtype])
                b = None if bias is None else torch.from_numpy(bias).cuda()
                counts = torch.zeros(experts, dtype=torch.int64, device="cuda")
                got, w = tctx.route(logits, k, score=score, bias=b, groups=groups, top_groups=kept, renormalise=bool(i & 1), scale=1.5, counts=counts)
                x = host(logits)
                bad = np.isnan(x).any(1)
                p = P.scores(score, np.where(np.isnan(x), 0.0, x))
                rank = p + (0.0 if bias is None else bias)
                rank[np.isneginf(x)] = -np.inf
                key = np.where(np.isneginf(x), -np.inf, x if bias is None else rank)
                if kept < groups:
                    two = -np.sort(-rank.reshape(n, groups, -1), axis=2)[:, :, :2]
                    value = two[:, :, 0] + np.where(np.isneginf(two[:, :, 1]), 0.0, two[:, :, 1])
                    best = np.argsort(-value, axis=1, kind="stable")[:, :kept]
                    open_ = np.zeros((n, groups), bool)
                    np.put_along_axis(open_, best, True, 1)
                    key = np.where(np.repeat(open_, experts // groups, axis=1), key, -np.inf)
                order = np.argsort(-key, axis=1, kind="stable")[:, :k]
                want = np.where(np.isneginf(np.take_along_axis(key, order, 1)), -1, order)
                want[bad] = -1
                same = (got.cpu().numpy() == want).all(1)
                # numpy's exponential and the kernel's differ by an ulp: rows whose deciding 64-bit keys lie within 4 ulp may differ
                lead = -np.sort(-np.where(np.isneginf(key), -1e300, key), axis=1)[:, :k + 1]
                with np.errstate(invalid="ignore"):
                    gaps = lead[:, :-1] - lead[:, 1:]
                tight = ((gaps > 0) & (gaps < 1e-15 * (1 + np.abs(lead[:, :-1])))).any(1) if bias is not None else np.zeros(n, bool)
                if kept < groups:
                    v = -np.sort(-value, axis=1)
                    tight |= (v[:, kept - 1] - v[:, kept] < 1e-15 * 4) & (v[:, kept - 1] != v[:, kept])
                assert (same | tight).all(), (i, layout, bias is None, int((~(same | tight)).sum()))
                chosen = np.where(want < 0, 0, want)
                ww = np.where(want < 0, 0.0, np.take_along_axis(p, chosen, 1))
                if i & 1:
                    total = ww.sum(1, keepdims=True)
                    ww = np.where(total > 0, ww / np.where(total > 0, total, 1.0), 0.0)
                ww = 1.5 * ww
                ok = same & ~bad
                assert np.all((np.abs(host(w) - ww) <= weights_bound(dtype, experts, k, ww, bool(i & 1)))[ok])
                assert np.isnan(host(w)[bad]).all()
                c = got.cpu().numpy()
                assert np.array_equal(counts.cpu().numpy(), np.bincount(c[c >= 0], minlength=experts))


def test_route_ties_masks_and_rows_without_an_answer(tctx):  # noqa: F811
    import torch

    inf, low = np.inf, np.finfo(np.float32).min
    rows = np.array([
        [1.0, 1.0, 1.0, 1.0, 1.0, 1.0],       # all alike: the lowest indices
        [0.0, 3.0, 3.0, -1.0, 3.0, 0.0],      # three alike
        [-inf] * 6,                           # nothing open
        [-inf, 2.0, -inf, -inf, -inf, -inf],  # one open
        [low] * 6,                            # the type's lowest value is a value
        [low, 0.5, low, 0.2, low, low],
        [np.nan, 1.0, 0.0, 0.0, 0.0, 0.0],
        [inf, 1.0, 0.0, 0.0, 0.0, inf],
        [700.0, -700.0, 699.0, 0.0, 1.0, 2.0],
    ], dtype=np.float64)
    for score in ("softmax", "sigmoid"):
        for dtype in ("f64", "f32"):
            for renormalise in (True, False):
                logits = put(rows, "row", torch_types()[dtype])
                got, w = tctx.route(logits, 3, score=score, renormalise=renormalise)
                want, want_w, _ = P.route(score, host(logits), None, 1, 1, 3, renormalise, 1.0)
                assert np.array_equal(got.cpu().numpy(), want), (score, dtype)
                assert np.array_equal(np.isnan(host(w)), np.isnan(want_w)), (score, dtype)
                ok = ~np.isnan(want_w)
                # (scores below the smallest f32 round to 0 there: an absolute half step of the subnormals)
                assert np.all(np.abs(host(w) - want_w)[ok] <= weights_bound(dtype, 6, 3, want_w, renormalise)[ok]), (score, dtype)
    # a NaN bias closes its expert; an infinite one orders like any other
    logits = put(np.zeros((2, 4)), "row", torch_types()["f32"])
    bias = torch.tensor([np.nan, 0.0, inf, 1.0], dtype=torch.float64, device="cuda")
    got, _ = tctx.route(logits, 4, score="sigmoid", bias=bias)
    assert got.cpu().tolist() == [[2, 3, 1, -1]] * 2


@pytest.mark.parametrize("layout", ["row", "col"])
@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_backward(tctx, score, dtype, layout):  # noqa: F811
    rng = np.random.default_rng(22)
    wide = torch_types()["f64" if dtype == "f64" else "f32"]
    for i, (n, experts, k, _, _) in enumerate(ROUTES):
        for renormalise in (False, True):
            z = 2.0 * rng.standard_normal((n, experts))
            if i % 4 == 1:
                z[rng.random((n, experts)) < 0.4] = -np.inf
            logits = put(z, layout, torch_types()[dtype], i % 2)
            chosen, _ = tctx.route(logits, k, score=score, renormalise=renormalise)
            if i % 5 == 2:  # an expert named twice, and names that no expert has
                chosen[:, -1] = chosen[:, 0]
                chosen[0, 0] = experts + 3
            dw = put(rng.standard_normal((n, k)), layout, wide)
            got = tctx.route_backward(logits, chosen, dw, score=score, renormalise=renormalise, scale=1.7)
            want, size = P.route_backward(score, host(logits), chosen.cpu().numpy(), host(dw), renormalise, 1.7)
            bound = (80 + 2 * experts + 4 * k) * 4 * U * size + (HALF_STEP[dtype] or (2.0**-24 if dtype == "f32" else 0.0)) * np.abs(want) + TINY[dtype] + (2.0**-134 if dtype == "bf16" else 0.0)
            assert np.all(np.abs(host(got) - want) <= bound), (n, experts, k, renormalise)


def test_route_gradient_against_differences_and_without_an_answer(tctx):  # noqa: F811
    import torch

    rng = np.random.default_rng(23)
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            logits = put(rng.standard_normal((6, 12)), "col", torch.float64)
            chosen, _ = tctx.route(logits, 3, score=score, renormalise=renormalise)
            dw = put(rng.standard_normal((6, 3)), "col", torch.float64)
            g = tctx.route_backward(logits, chosen, dw, score=score, renormalise=renormalise, scale=1.3)

            def loss(z):
                p = P.scores(score, z)
                w = np.take_along_axis(p, chosen.cpu().numpy().astype(np.int64), 1)
                w = w / w.sum(1, keepdims=True) if renormalise else w
                return 1.3 * (w * host(dw)).sum()

            z = host(logits)
            for r in range(6):
                for e in range(12):
                    up, down = z.copy(), z.copy()
                    up[r, e] += 1e-6
                    down[r, e] -= 1e-6
                    assert abs((loss(up) - loss(down)) / 2e-6 - float(g[r, e])) <= 1e-8
            bad = logits.clone()
            bad[2, 5] = float("nan")
            out = tctx.route_backward(bad, chosen, dw, score=score, renormalise=renormalise)
            assert torch.isnan(out[2]).all() and not torch.isnan(out[[0, 1, 3, 4, 5]]).any()


def model(rng, n, d, experts, m, k, sizes=None, unused=0.0):
    X = np.asfortranarray(rng.random((n, d)))
    Xq = np.asfortranarray(rng.random((m, d)))
    if sizes is None:
        cuts = np.sort(rng.integers(0, n + 1, experts - 1)) if experts > 1 else np.zeros(0, np.int64)
        offsets = np.concatenate([[0], cuts, [n]]).astype(np.int64)
    else:
        offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
    chosen = np.asfortranarray(rng.integers(0, experts, (m, k)).astype(np.int32))
    chosen[rng.random((m, k)) < unused] = -1
    return X, Xq, offsets, chosen, np.asfortranarray(rng.standard_normal((m, k))), rng.standard_normal(n)


SPECS = [("squared_exp", 0.8, 1.3), ("exponential", 0.9, 0.7), ("matern1", 1.1, 0.9), ("matern2", 0.9, 1.2), ("rational_quadratic", 1.5, 0.8), ("linear", 0.7),
         ("sum", ("prod", ("squared_exp", 1.0, 1.0), ("matern1", 2.0, 0.5)), ("linear", 0.2))]
# points, features, experts, queries, slots, share of unused slots
MODELS = [(300, 11, 2, 400, 1, 0.0), (500, 20, 2, 300, 2, 0.1), (1, 1, 1, 1, 1, 0.0), (5, 2, 3, 4, 2, 0.0), (64, 3, 1, 64, 1, 0.0), (300, 5, 7, 65, 3, 0.3), (1000, 16, 8, 130, 2, 0.0), (513, 1, 2, 1, 2, 0.0), (2000, 8, 1000, 40, 4, 0.1),
          (700, 33, 3, 7, 1, 0.0), (4097, 4, 2, 257, 2, 0.5)]


def arg(d):
    return d / (2 * 0.8**2) + 1.0


def device(*arrays):
    import torch

    return [torch.from_numpy(np.ascontiguousarray(a.T)).cuda().t() if a.ndim == 2 else torch.from_numpy(a).cuda() for a in arrays]


@pytest.mark.parametrize("spec", SPECS, ids=lambda s: s[0])
def test_experts_forward_and_backward(tctx, spec):  # noqa: F811
    rng = np.random.default_rng(24)
    for n, d, experts, m, k, unused in MODELS:
        X, Xq, offsets, chosen, w, alpha = model(rng, n, d, experts, m, k, unused=unused)
        prior, dmean = rng.standard_normal(m), rng.standard_normal(m)
        want, want_s, size = P.experts_predict(spec, X, alpha, offsets, Xq, chosen, w, prior)
        most = int(np.max(np.diff(offsets)))
        rel = (most + (d + 8) * (1 + arg(d)) + 16) * 2 * U
        x, q, o, c, ww, a, pr, dm = device(X, Xq, offsets, chosen, w, alpha, prior, dmean)
        for args in ((X, alpha, offsets, Xq, chosen, w, prior), (x, a, o, q, c, ww, pr)):  # host and device memory
            mean, slots = tctx.experts_predict(spec, *args[:6], prior_q=args[6])
            mean, slots = (host(v) if hasattr(v, "cpu") else v for v in (mean, slots))
            assert np.all(np.abs(slots - want_s) <= rel * size + 1e-300), (n, d, experts, m, k)
            assert np.all(np.abs(mean - want) <= (rel + (k + 2) * U) * (np.abs(w) * size).sum(1) + (k + 2) * U * np.abs(prior)), (n, d, experts, m, k)
        want_w, want_a, size_a = P.experts_backward(spec, X, offsets, Xq, chosen, w, want_s, dmean)
        rel = (m * k + (d + 8) * (1 + arg(d)) + 16) * 2 * U
        for args in ((X, offsets, Xq, chosen, w, np.asfortranarray(want_s), dmean), (x, o, q, c, ww, device(want_s)[0], dm)):
            dw, da = (host(v) if hasattr(v, "cpu") else v for v in tctx.experts_backward(spec, *args))
            assert np.all(np.abs(dw - want_w) <= 2 * U * np.abs(want_w)), (n, d, experts, m, k)
            assert np.all(np.abs(da - want_a) <= rel * size_a + 1e-300), (n, d, experts, m, k)


@pytest.mark.parametrize("spec", SPECS[::3], ids=lambda s: s[0])
@pytest.mark.parametrize("per_expert", [31, 190, 200, 700])
def test_experts_on_either_side_of_many_slots(tctx, spec, per_expert):  # noqa: F811
    """slots an expert around the number from which a lane takes a slot, for features that stay in registers and more of them"""
    rng = np.random.default_rng(32)
    for n, d, experts in ((1200, 3, 3), (900, 8, 2), (700, 16, 5), (300, 33, 1)):
        m = per_expert * experts // 2
        X, Xq, offsets, chosen, w, alpha = model(rng, n, d, experts, m, 2, unused=0.05)
        want, want_s, size = P.experts_predict(spec, X, alpha, offsets, Xq, chosen, w, None)
        rel = (int(np.max(np.diff(offsets))) + (d + 8) * (1 + arg(d)) + 16) * 2 * U
        x, q, o, c, ww, a = device(X, Xq, offsets, chosen, w, alpha)
        mean, slots = (host(v) for v in tctx.experts_predict(spec, x, a, o, q, c, ww))
        assert np.all(np.abs(slots - want_s) <= rel * size + 1e-300), (n, d, experts, m)
        assert np.all(np.abs(mean - want) <= (rel + 4 * U) * (np.abs(w) * size).sum(1) + 1e-300), (n, d, experts, m)


def test_experts_of_thousands_of_slots(tctx):  # noqa: F811
    """lists of one expert on either side of what a workgroup holds, beside experts with none, one and few slots"""
    rng = np.random.default_rng(33)
    spec = ("matern2", 0.9, 1.2)
    for n, d, experts, m, k in ((60, 3, 1, 4096, 1), (60, 3, 1, 4097, 1), (90, 17, 4, 3000, 2), (40, 2, 2, 9001, 1)):
        X, Xq, offsets, chosen, w, alpha = model(rng, n, d, experts, m, k)
        chosen[chosen == experts - 1] = 0
        if experts > 1:
            chosen[5, 0] = experts - 1
        dmean = rng.standard_normal(m)
        want, want_s, size = P.experts_predict(spec, X, alpha, offsets, Xq, chosen, w, None)
        x, q, o, c, ww, a, dm, ws = device(X, Xq, offsets, chosen, w, alpha, dmean, np.asfortranarray(want_s))
        mean, slots = (host(v) for v in tctx.experts_predict(spec, x, a, o, q, c, ww))
        rel = (int(np.max(np.diff(offsets))) + (d + 8) * (1 + arg(d)) + 16) * 2 * U
        assert np.all(np.abs(slots - want_s) <= rel * size + 1e-300), (n, d, experts, m)
        assert np.all(np.abs(mean - want) <= (rel + 4 * U) * (np.abs(w) * size).sum(1) + 1e-300), (n, d, experts, m)
        want_w, want_a, size_a = P.experts_backward(spec, X, offsets, Xq, chosen, w, want_s, dmean)
        dw, da = (host(v) for v in tctx.experts_backward(spec, x, o, q, c, ww, ws, dm))
        assert np.all(np.abs(dw - want_w) <= 2 * U * np.abs(want_w)), (n, d, experts, m)
        assert np.all(np.abs(da - want_a) <= (m * k + (d + 8) * (1 + arg(d)) + 16) * 2 * U * size_a + 1e-300), (n, d, experts, m)


def test_covariances_that_vanish(tctx):  # noqa: F811
    """distances from none to beyond the smallest covariance, infinite and undefined ones: 0 and NaN as the Gram kernel has them, subnormals
    within the smallest step (half of it on either side), the exponent's error as in the other tests"""
    for name, reach in (("squared_exp", 40.0), ("exponential", 1600.0), ("matern1", 500.0), ("matern2", 400.0)):
        spec = (name, 1.0, 1.5)
        Xq = np.concatenate([np.linspace(0.0, reach, 400), [np.inf, np.nan]]).reshape(-1, 1)
        m = len(Xq)
        chosen, w = np.zeros((m, 1), np.int32, order="F"), np.ones((m, 1), order="F")
        got, _ = tctx.experts_predict(spec, np.zeros((1, 1)), np.ones(1), np.array([0, 1]), Xq, chosen, w)
        want = tctx.gram(spec, Xq, np.zeros((1, 1)))[:, 0]
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[-1])
        ok = ~np.isnan(want)
        assert np.all(np.abs(got - want)[ok] <= 16 * 800 * 2 * U * want[ok] + 2.0**-1074)


def test_one_expert_is_predict_mean(tctx):  # noqa: F811
    """each expert fitted by fr_chol_from_inputs on its own rows, alpha by fr_chol_solve: the mean of a query that names it alone is
    fr_predict_mean's"""
    rng = np.random.default_rng(25)
    kernel, noise, d = ("squared_exp", 0.8, 1.3), 0.1, 4
    sizes = [100, 1, 257, 64]
    X, Xq, offsets, _, _, _ = model(rng, sum(sizes), d, 4, 50, 1, sizes)
    y = rng.standard_normal(len(X))
    alpha, want = np.empty(len(X)), []
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        chol = tctx.cholesky_from_inputs(kernel, np.asfortranarray(X[lo:hi]), noise)
        alpha[lo:hi] = chol.solve(y[lo:hi])[:, 0]
        chol.set_targets(y[lo:hi])
        want.append(chol.predict_mean(kernel, None, Xq, np.full(50, 0.3)))
        chol.free()
    for e in range(4):
        mean, _ = tctx.experts_predict(kernel, X, alpha, offsets, Xq, np.full((50, 1), e, np.int32, order="F"), np.ones((50, 1), order="F"), prior_q=np.full(50, 0.3))
        size = np.abs(P.covariance(kernel, Xq, X[offsets[e]:offsets[e + 1]])) @ np.abs(alpha[offsets[e]:offsets[e + 1]]) + 0.3
        # the same covariances times the same coefficients; alpha itself is a solve of condition number up to c ampl / noise^2
        cond = sizes[e] * 1.3 / noise**2
        assert np.all(np.abs(mean - want[e]) <= (cond + 2 * sizes[e] + 200) * U * size)


def test_route_to_experts_and_back(tctx):  # noqa: F811
    """router and experts as they are used: logits from the distances to the experts' centres (a softmax of -|x - c|^2 / (2 ls^2), worked out by
    fr_gemm), the two best experts' means; gradients of a loss in the logits and the coefficients against differences"""
    import torch

    rng = np.random.default_rng(26)
    kernel, E, d, m, k = ("matern2", 0.9, 1.2), 6, 3, 40, 2
    X, Xq, offsets, _, _, alpha = model(rng, 240, d, E, m, k, [40] * E)
    centres = np.stack([X[a:b].mean(0) for a, b in zip(offsets[:-1], offsets[1:])])
    logits = np.asfortranarray(tctx.gemm(Xq, np.asfortranarray(centres), trans_b=True, alpha=4.0) - 2.0 * (centres**2).sum(1))
    dmean = rng.standard_normal(m)
    x, q, o, z, a, dm = device(X, Xq, offsets, logits, alpha, dmean)

    chosen, w = tctx.route(z, k)
    mean, slots = tctx.experts_predict(kernel, x, a, o, q, chosen, w)
    dw, da = tctx.experts_backward(kernel, x, o, q, chosen, w, slots, dm)
    dz = tctx.route_backward(z, chosen, dw)

    def loss(zz, aa):
        c, ww = tctx.route(zz, k)
        assert torch.equal(c, chosen)
        return float((tctx.experts_predict(kernel, x, aa, o, q, c, ww)[0] * dm).sum())

    for r, e in [(0, int(chosen[0, 0])), (3, int(chosen[3, 1])), (7, int(chosen[7, 0])), (11, 2)]:
        up, down = z.clone(), z.clone()
        up[r, e] += 1e-6
        down[r, e] -= 1e-6
        assert abs((loss(up, a) - loss(down, a)) / 2e-6 - float(dz[r, e])) <= 1e-6 * (1 + abs(float(dz[r, e])))
    for i in (0, 41, 239):
        up, down = a.clone(), a.clone()
        up[i] += 1e-3
        down[i] -= 1e-3
        assert abs((loss(z, up) - loss(z, down)) / 2e-3 - float(da[i])) <= 1e-8 * (1 + abs(float(da[i])))


def test_staged_inputs(tctx):  # noqa: F811
    """matrices that Context.inputs_to_device has put on the device are taken like arrays"""
    rng = np.random.default_rng(31)
    spec = ("matern1", 1.1, 0.9)
    X, Xq, offsets, chosen, w, alpha = model(rng, 200, 5, 3, 30, 2)
    x, q = tctx.inputs_to_device(np.ascontiguousarray(X)), tctx.inputs_to_device(Xq, "colmajor")
    got, slots = tctx.experts_predict(spec, x, alpha, offsets, q, chosen, w)
    want, _ = tctx.experts_predict(spec, X, alpha, offsets, Xq, chosen, w)
    assert np.array_equal(got, want)
    x.free(), q.free()


def test_experts_odd_offsets_and_names(tctx):  # noqa: F811
    """points of no expert, offsets in device memory that run out of range, names that no expert has: the places there are answer, nothing
    else is touched"""
    import torch

    rng = np.random.default_rng(27)
    spec = ("squared_exp", 0.8, 1.3)
    X, Xq, _, chosen, w, alpha = model(rng, 100, 3, 4, 30, 3)
    offsets = np.array([7, 20, 20, 66, 90], dtype=np.int64)
    chosen[0] = (-1, 4, 99)
    chosen[1] = (2, 2, 2)
    chosen[2] = (1, 1, 1)  # an expert without points
    x, q, o, c, ww, a = device(X, Xq, offsets, chosen, w, alpha)
    mean, slots = tctx.experts_predict(spec, x, a, o, q, c, ww)
    want, want_s, size = P.experts_predict(spec, X, alpha, offsets, Xq, chosen, w, None)
    assert np.all(np.abs(host(slots) - want_s) <= 200 * U * size) and np.all(host(mean)[[0, 2]] == 0.0)
    dm = torch.ones(30, dtype=torch.float64, device="cuda")
    dw, da = tctx.experts_backward(spec, x, o, q, c, ww, slots, dm)
    _, want_a, size_a = P.experts_backward(spec, X, offsets, Xq, chosen, w, host(slots), np.ones(30))
    assert np.all(np.abs(host(da) - want_a) <= 300 * U * size_a)
    assert np.all(host(da)[:7] == 0.0) and np.all(host(da)[90:] == 0.0) and np.all(host(dw)[0] == 0.0)
    wild = torch.tensor([-10, 20, 1 << 40, 1 << 41, 5], dtype=torch.int64, device="cuda")
    tctx.experts_predict(spec, x, a, wild, q, c, ww)
    tctx.experts_backward(spec, x, wild, q, c, ww, slots, dm)
    torch.cuda.synchronize()


def test_captured_and_repeated(tctx):  # noqa: F811
    """the same bits on every call, eager or replayed, with two graphs of one context alive"""
    import torch
    from friedrich_amd.device import Context

    rng = np.random.default_rng(28)
    side = torch.cuda.Stream()
    c = Context()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        c.set_stream(side.cuda_stream)
        calls, graphs = [], []
        for n, d, E, m, k in ((3000, 6, 12, 500, 2), (400, 3, 5, 9, 3)):
            X, Xq, offsets, _, _, alpha = model(rng, n, d, E, m, k)
            x, q, o, a, z, dm = device(X, Xq, offsets, alpha, np.asfortranarray(rng.standard_normal((m, E))), rng.standard_normal(m))
            out = [torch.empty(k, m, dtype=torch.int32, device="cuda").t(), *(torch.empty(k, m, dtype=torch.float64, device="cuda").t() for _ in range(3)),
                   *(torch.empty(v, dtype=torch.float64, device="cuda") for v in (m, n)), torch.empty(E, m, dtype=torch.float64, device="cuda").t(),
                   torch.empty(E, dtype=torch.int64, device="cuda")]

            def call(x=x, q=q, o=o, a=a, z=z, dm=dm, out=out, k=k):
                c.route(z, k, experts=out[0], weights=out[1], counts=out[7])
                c.experts_predict(("squared_exp", 0.8, 1.3), x, a, o, q, out[0], out[1], out=out[4], slots=out[2])
                c.experts_backward(("squared_exp", 0.8, 1.3), x, o, q, out[0], out[1], out[2], dm, dweights=out[3], dalpha=out[5])
                c.route_backward(z, out[0], out[3], dlogits=out[6])

            call()
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call()
            calls.append((call, z, out))
            graphs.append(g)
        for _ in range(4):
            for call, z, out in calls:
                z.copy_(torch.randn(z.shape, device="cuda", dtype=torch.float64))
                call()
                side.synchronize()
                eager = [t.clone() for t in out]
                for t in out:
                    t.zero_()
                for g in graphs:
                    g.replay()
                side.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(eager, out))
    torch.cuda.synchronize()
    del graphs, g
    c.close()


def test_refusals(tctx):  # noqa: F811
    import torch
    from friedrich_amd import _capi as C
    from friedrich_amd.device import FriedrichError

    z = torch.zeros(8, 6, dtype=torch.float64, device="cuda")
    for kw in (dict(k=0), dict(k=7), dict(k=2, groups=4), dict(k=2, groups=3, top_groups=0), dict(k=2, groups=3, top_groups=4), dict(k=5, groups=3, top_groups=2)):
        with pytest.raises(FriedrichError) as e:
            tctx.route(z, **kw)
        assert e.value.status == C.FR_SHAPE, kw
    with pytest.raises(FriedrichError):
        tctx.route(z, 2, scale=float("nan"))
    with pytest.raises(FriedrichError):
        tctx.route(torch.zeros(4, 1025, device="cuda"), 2)
    with pytest.raises(FriedrichError):
        tctx.route(torch.zeros(4, 200, device="cuda"), 65)
    with pytest.raises(ValueError):
        tctx.route(z, 2, bias=torch.zeros(6, device="cuda"))
    with pytest.raises(ValueError):
        tctx.route(z, 2, experts=torch.zeros(8, 2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        tctx.route(z.to(torch.int32), 2)
    rng = np.random.default_rng(29)
    X, Xq, offsets, chosen, w, alpha = model(rng, 20, 2, 3, 5, 2)
    for bad in ([0, 5, 4, 20], [0, 5, 6, 21], [-1, 5, 6, 20]):
        with pytest.raises(FriedrichError) as e:
            tctx.experts_predict(("squared_exp", 1.0, 1.0), X, alpha, np.array(bad, dtype=np.int64), Xq, chosen, w)
        assert e.value.status == C.FR_SHAPE
    with pytest.raises(FriedrichError) as e:
        tctx.experts_predict(("squared_exp", 1.0, 1.0), X[:, :0], alpha, offsets, Xq[:, :0], chosen, w)
    assert e.value.status == C.FR_SHAPE
    with pytest.raises(FriedrichError):
        tctx.experts_predict(("squared_exp", 1.0, 1.0), X, alpha, np.zeros(1026, dtype=np.int64), Xq, chosen, w)
    with pytest.raises(FriedrichError):
        tctx.experts_predict(("squared_exp", 1.0, 1.0), X, alpha[:19], offsets, Xq, chosen, w)
