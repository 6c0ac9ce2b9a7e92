"""Sampling next to the borders of its tokens: how exact the weights are that decide the draw.

A row's weights are f64 exponentials, good to 4e-14 each, so a cumulative probability is off by less than 8e-14 + n 2^-53
for sums of n; a random number 2e-13 to either side of a border of up to 64 tokens decides as it does in the definition,
whose own error is n 2^-52."""
import numpy as np
import pytest

import strata_cuda as sc
from test_sample_gpu import check, draw

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("t", [1.0, 0.7, 2.5])
@pytest.mark.parametrize("vocab", [2, 7, 64])
def test_random_numbers_next_to_a_border(ctx, vocab, t):
    rng = np.random.default_rng(vocab)
    rows = 4096
    x = (rng.standard_normal((rows, vocab)) * 2 + rng.uniform(-15, 15, (rows, 1))).astype(np.float32)
    d = x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)
    c = np.cumsum(np.exp(d / np.float64(np.float32(t))), 1)
    at = rng.integers(0, vocab - 1, rows)
    border = c[np.arange(rows), at] / c[:, -1]
    xd = torch.from_numpy(x).cuda()
    for side, want in ((-1, at), (1, at + 1)):
        u = border * (1 + side * 2e-13)
        ids, _ = draw(ctx, xd, list(u), t=[t] * rows)
        off = np.nonzero(ids != want)[0]
        sure = (u < 1 - 1e-9) & (np.abs(u - border) > 1e-13)  # a border next to 0 or 1 leaves no room beside it
        assert not sure[off].any(), (len(off), x[off[0]], u[off[0]])


@pytest.mark.parametrize("center", [0.0, 10.0, -300.0, 9000.0])
def test_temperatures_that_leave_the_table(ctx, center):
    """A temperature times 600 within a few steps of the largest logit, where the weights' floor rounds; and very large ones."""
    rng = np.random.default_rng(7)
    for t in (1e-12, 1e-9, 1.7e-9, 2e-9, 3e-9, 1e-8, 1e-6, 3e-6, 1e-5, 1e-3, 1e5, 1e34, 4e35, 6e35, 1e38):
        x = (rng.standard_normal((6, 700)) * 2 + center).astype(np.float32)
        x[2:4] = np.round(x[2:4])  # several largest ones
        x[4:, ::3] = -np.inf
        for kw in ({}, dict(p=[0.9] * 6), dict(p=[0.3] * 6, m=[0.01] * 6)):
            check(ctx, x, list(rng.random(6)), t=[t] * 6, **kw)
