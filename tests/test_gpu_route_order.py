"""The order of the experts over many rows, where 32-bit keys decide most of them: logits that 32 bits hold badly or not at all.  Choices
have to be those of the definition in 64 bits; only rows in which two 64-bit values that decide lie within the exponentials' own error
(numpy's and the kernel's, an ulp each: 1e-15 (1 + |value|)) may fall either way."""
import numpy as np
import pytest

import plain_operators as P
from test_gpu_recurrence import host, put, tctx, torch_types  # noqa: F401

pytestmark = pytest.mark.gpu


def expected(score, x, bias, groups, kept, k):
    """-> (experts n x k, rows that rounding may decide)"""
    n, experts = x.shape
    p = P.scores(score, x)
    rank = p + (0.0 if bias is None else bias)
    closed = np.isneginf(x) | (np.zeros(experts, bool) if bias is None else np.isneginf(bias))
    rank = np.where(closed, -np.inf, rank)
    key = np.where(closed, -np.inf, x) if bias is None else rank
    tight = np.zeros(n, bool)
    if kept < groups:
        two = -np.sort(-rank.reshape(n, groups, -1), axis=2)[:, :, :2]
        value = two[:, :, 0] + (0.0 if two.shape[2] == 1 else np.where(np.isneginf(two[:, :, 1]), 0.0, two[:, :, 1]))
        best = np.argsort(-value, axis=1, kind="stable")
        v = np.take_along_axis(value, best, 1)
        with np.errstate(invalid="ignore"):
            gap = v[:, kept - 1] - v[:, kept]
        tight |= (gap != 0) & (gap < 4e-15 * (1 + np.abs(v[:, kept - 1])))
        open_ = np.zeros((n, groups), bool)
        np.put_along_axis(open_, best[:, :kept], True, 1)
        key = np.where(np.repeat(open_, experts // groups, axis=1), key, -np.inf)
    order = np.argsort(-key, axis=1, kind="stable")
    lead = np.take_along_axis(key, order, 1)[:, :k + 1]
    if bias is not None:  # (logits order exactly)
        with np.errstate(invalid="ignore"):
            gaps = lead[:, :-1] - lead[:, 1:]
            tight |= ((gaps > 0) & (gaps < 2e-15 * (1 + np.abs(lead[:, :-1])))).any(1)
    return np.where(np.isneginf(lead[:, :k]), -1, order[:, :k]), tight


def compare(tctx, logits, bias, score, groups, kept, k, what):  # noqa: F811
    import torch

    got, w = tctx.route(logits, k, score=score, bias=None if bias is None else torch.from_numpy(bias).cuda(), groups=groups, top_groups=kept)
    want, tight = expected(score, host(logits), bias, groups, kept, k)
    same = (got.cpu().numpy() == want).all(1)
    assert (same | tight).all(), (what, int((~(same | tight)).sum()), np.nonzero(~(same | tight))[0][:3], int(tight.sum()))
    assert tight.sum() < len(want) / 100, (what, int(tight.sum()))
    return got, w


@pytest.mark.parametrize("offset", [-5000.0, 1e4, -1e5, 1e6])
@pytest.mark.parametrize("experts,k,groups,kept", [(8, 2, 1, 1), (64, 8, 1, 1), (64, 2, 8, 2), (256, 4, 4, 1)])
def test_far_logits(tctx, experts, k, groups, kept, offset):  # noqa: F811
    """a softmax does not change when every logit of a row moves by the same amount, as those of squared distances do"""
    rng = np.random.default_rng(41)
    n = 32768
    logits = put(offset + 2.0 * rng.standard_normal((n, experts)), "row", torch_types()["f64"])
    for bias in ([None] if groups > 1 else []) + [0.1 * rng.standard_normal(experts)]:
        compare(tctx, logits, bias, "softmax", groups, kept, k, (experts, k, groups, offset, bias is None))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [1, 2, 8])
def test_logits_beyond_32_bits(tctx, score, k):  # noqa: F811
    """64-bit logits larger than any of 32 bits, among the slots and just behind the last"""
    rng = np.random.default_rng(42)
    n, experts = 20000, 16
    z = rng.standard_normal((n, experts))
    huge = np.array([1e39, 2e39, 1e200, 1e300, np.finfo(np.float64).max])
    for r in range(0, n, 2):
        at = rng.permutation(experts)[:1 + r % 9]
        z[r, at] = huge[rng.integers(0, len(huge), len(at))]
    logits = put(z, "row", torch_types()["f64"])
    got, w = compare(tctx, logits, None, score, 1, 1, k, (score, k))
    assert np.isfinite(host(w)).all()
    if score == "softmax" and k == 1:
        assert np.all(host(w) == 1.0)  # (renormalised: the largest has all of it)
    compare(tctx, logits, None, score, 4, 2, k, (score, k, "groups"))
    compare(tctx, logits, 0.1 * rng.standard_normal(experts), score, 1, 1, k, (score, k, "bias"))


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16"])
def test_infinite_logits_in_groups(tctx, dtype):  # noqa: F811
    """a sigmoid of +inf is 1: an expert like any other, shut out with its group where that is not kept"""
    rng = np.random.default_rng(43)
    n, experts, groups, kept, k = 20000, 16, 4, 2, 4
    z = rng.standard_normal((n, experts))
    z[::2, 4:8] = -9.0
    z[::2, 5] = np.inf
    z[1::4, 9] = np.inf
    logits = put(z, "row", torch_types()[dtype])
    for layout in ("row", "col"):
        compare(tctx, put(z, layout, torch_types()[dtype]), None, "sigmoid", groups, kept, k, (dtype, layout))
    # (the rows do shut it out)
    want, _ = expected("sigmoid", host(logits), None, groups, kept, k)
    assert (want[::2] != 5).all(1).sum() > n // 8


@pytest.mark.parametrize("n", [50, 20000])
def test_a_bias_of_minus_infinity_closes(tctx, n):  # noqa: F811
    """as a NaN does: no slot, no part in its group's value, whatever else is left"""
    import torch

    rng = np.random.default_rng(44)
    experts = 12
    bias = 0.1 * rng.standard_normal(experts)
    bias[[0, 3, 4, 5, 6, 7, 9]] = -np.inf  # (the second group of four has none open)
    logits = put(rng.standard_normal((n, experts)), "row", torch_types()["f32"])
    for score in ("softmax", "sigmoid"):
        got, w = compare(tctx, logits, bias, score, 1, 1, 8, score)
        assert (got[:, 5:] == -1).all() and (w[:, 5:] == 0).all() and (got[:, :5] >= 0).all()
        got, w = compare(tctx, logits, bias, score, 3, 2, 8, (score, "groups"))
        assert (got[:, 5:] == -1).all() and (got[:, :5] >= 0).all()
        nan, _ = tctx.route(logits, 8, score=score, bias=torch.from_numpy(np.where(np.isinf(bias), np.nan, bias)).cuda(), groups=3, top_groups=2)
        assert torch.equal(nan, got)
