"""fr_experts_predict on either side of 256 slots an expert, where a lane takes a slot instead of a point.  Bounds as in
test_gpu_experts.py: (c + (d + 8)(1 + arg) + 16) 2 u of the terms' size for c points and d features."""
import numpy as np
import pytest

import plain_operators as P
from test_gpu_experts import U, arg, device, model
from test_gpu_recurrence import host, tctx  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [254, 256, 258, 300])
@pytest.mark.parametrize("spec", [("squared_exp", 0.8, 1.3), ("matern1", 1.1, 0.9), ("linear", 0.7)], ids=lambda s: s[0])
def test_around_the_slots_of_a_lane(tctx, spec, slots):  # noqa: F811
    rng = np.random.default_rng(71)
    for n, d, experts in ((1200, 3, 3), (900, 8, 2), (700, 16, 5), (300, 33, 1), (64, 1, 4)):
        m = slots * experts // 2
        X, Xq, offsets, chosen, w, alpha = model(rng, n, d, experts, m, 2, unused=0.05)
        want, want_s, size = P.experts_predict(spec, X, alpha, offsets, Xq, chosen, w, None)
        rel = (int(np.max(np.diff(offsets))) + (d + 8) * (1 + arg(d)) + 16) * 2 * U
        x, q, o, c, ww, a = device(X, Xq, offsets, chosen, w, alpha)
        mean, got = (host(v) for v in tctx.experts_predict(spec, x, a, o, q, c, ww))
        assert np.all(np.abs(got - want_s) <= rel * size + 1e-300), (n, d, experts, m)
        assert np.all(np.abs(mean - want) <= (rel + 4 * U) * (np.abs(w) * size).sum(1) + 1e-300), (n, d, experts, m)
