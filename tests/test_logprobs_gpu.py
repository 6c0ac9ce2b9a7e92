"""Log-probabilities, entropies and likeliest tokens (strata_cuda_logprobs_dev) against their formulas in 64 bits.

Ids must be equal. Tolerances, before any run: with d = x - max (rounded at 2^-24 of itself), an f32 weight e^d is off by
2^-22 + 2 |d| 2^-24 of itself, and what is below e^-30 of the largest does not count here: t = 2^-22 + 2^-18 (at the |d| of 15
and less that sums are made of, this leaves 2^-19 for eight maxima that moved, at 2^-22 each). Z = 1 + R:
log Z is off by t R / (1 + R), a log-probability by that and half a step of f32; the entropy is log Z - sum e d / Z, whose
sum is off by t and 16 roundings of 2^-24: t R / (1 + R) + (2 t + 2^-20) |sum e d| / Z and half a step. Z itself is an f64 sum of
1 and R: a thread that holds the 1 adds at most n / 512 + 4 more numbers to it and takes part in 9 joins, a rounding of 2^-53
of Z each, so log Z is off by (n / 512 + 16) 2^-53 more (all there is to it where R is next to nothing)."""
import math

import numpy as np
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
T = 2.0 ** -22 + 2.0 ** -18


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def expected(x, target, top):
    """One row: log p of the target, entropy, ids, their log p, each number with how far it may be off."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    m = x.max()
    order = np.argsort(-x, kind="stable")[:top]
    order = order[x[order] > -np.inf]
    if m == -np.inf:
        lp, h, th, tl = np.full_like(x, -np.inf), 0.0, 0.0, 0.0
    elif m == np.inf:
        z = np.isinf(x) & (x > 0)
        lp, h, th, tl = np.where(z, -math.log(z.sum()), -np.inf), math.log(z.sum()), 0.0, 0.0
    else:
        d = x - m
        e = np.exp(d)
        others = e.copy()
        others[np.argmax(x)] = 0
        rest = others.sum()
        z, ed = 1 + rest, (e[e > 0] * d[e > 0]).sum()
        lp, h = d - np.log1p(rest), np.log1p(rest) - ed / z
        tl = T * rest / z + (len(x) / 512 + 16) * 2.0 ** -53
        th = tl + (2 * T + 2.0 ** -20) * abs(ed) / z
    first = lp[target] if 0 <= target < len(x) else 0.0
    blank = top - len(order)
    return first, h, np.concatenate([order, np.full(blank, -1)]).astype(int), np.concatenate([lp[order], np.full(blank, -np.inf)]), tl, th


def check(ctx, x, targets, top, stride=0, entropy=True, lp=True):
    rows, vocab = x.shape
    base = torch.full((rows, stride or vocab), 1e4, device="cuda")
    base[:, :vocab] = x
    f = lambda *s: torch.full(s, 9.0, device="cuda")  # noqa: E731
    got, ent, tops = f(rows + 1), f(rows + 1), f(rows + 1, max(top, 1))
    ids = torch.full((rows + 1, max(top, 1)), 99, dtype=torch.int32, device="cuda")
    tg = torch.tensor(targets, dtype=torch.int32, device="cuda")
    ctx.logprobs_dev(base.data_ptr(), rows, vocab, tg.data_ptr() if lp else 0, got.data_ptr() if lp else 0, ent.data_ptr() if entropy else 0, top,
                     ids.data_ptr() if top else 0, tops.data_ptr() if top else 0, stride, stream())
    torch.cuda.synchronize()
    host = x.cpu().numpy()

    def close(a, b, tol, what):
        a = float(a)
        assert (a == b) or abs(a - b) <= tol + 2.0 ** -24 * abs(b) + 1e-45, (what, a, b, tol)

    for r in range(rows):
        first, h, order, lps, tl, th = expected(host[r].copy(), targets[r], top)
        if lp:
            close(got[r], first, tl, "target")
        if entropy:
            close(ent[r], h, th, "entropy")
        if top:
            assert ids[r].tolist() == order.tolist(), r
            for a, b in zip(tops[r].tolist(), lps):
                close(a, b, tl, "top")
    assert got[rows] == 9 and ent[rows] == 9 and (tops[rows] == 9).all() and (ids[rows] == 99).all()
    if not lp:
        assert (got == 9).all()
    if not entropy:
        assert (ent == 9).all()
    if not top:
        assert (ids == 99).all()


def logits(rows, vocab, seed, gain=2.5):
    return torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * gain


@pytest.mark.parametrize("top", [0, 1, 5, 32])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 511, 512, 513, 2047, 2048, 2049, 32003, 151936])
def test_vocabularies(ctx, vocab, top):
    for rows in (1, 5):
        x = logits(rows, vocab, vocab)
        check(ctx, x, [(r * 7919) % vocab for r in range(rows)], top)
        check(ctx, x, [(r * 7919) % vocab for r in range(rows)], top, stride=vocab + 3)
        check(ctx, x, [(r * 7919) % vocab for r in range(rows)], top, stride=(vocab + 7) // 4 * 4)


@pytest.mark.parametrize("rows", [1, 9, 18, 37, 74, 75, 150, 400])
def test_rows(ctx, rows):
    check(ctx, logits(rows, 5003, rows), [r % 5003 for r in range(rows)], 20)


def test_certain_tokens(ctx):
    """One token has nearly everything: its log-probability is the rest, to the rest's own precision."""
    x = logits(6, 40000, 3, 1.0)
    for r in range(6):
        x[r, 17 * r] = 14.0 + 4 * r
    check(ctx, x, [17 * r for r in range(6)], 3)


def test_wide_and_flat_rows(ctx):
    x = logits(6, 30011, 4)
    x[0], x[1], x[2] = 3.25, 0.0, torch.arange(30011, device="cuda") * -1e-3
    x[3] = torch.arange(30011, device="cuda") * 1e-3
    x[4] *= 1e37
    x[5] = torch.linspace(-3e38, 3e38, 30011, device="cuda")
    check(ctx, x, [0, 30010, 5, 30000, 77, 30010], 32)
    check(ctx, x, [0, 30010, 5, 30000, 77, 30010], 20, stride=30012)


def test_ties_go_to_the_lowest_index(ctx):
    x = torch.round(logits(8, 32003, 5))
    x[1] = torch.where(torch.arange(32003, device="cuda") % 2 == 0, 0.0, -0.0)  # equal zeros
    x[2, 5::512] = 50.0  # one thread's share, where threads take every 512th
    x[3, 4 * 9::2048] = 50.0
    x[4, :3000] = 20.0
    check(ctx, x, [0, 1, 5, 36, 2999, 6, 7, 8], 32)
    check(ctx, x, [0, 1, 5, 36, 2999, 6, 7, 8], 32, stride=32004)


def test_masked_rows(ctx):
    x = logits(9, 20011, 6)
    x[0] = -math.inf
    x[1], x[1, 500] = -math.inf, 1.0
    x[2, 1::2] = -math.inf
    x[3] = math.nan
    x[4, ::3] = math.nan
    x[5, 70], x[5, 9000] = math.inf, math.inf
    x[6, 3], x[6, 4] = math.inf, -math.inf
    x[7] = torch.finfo(torch.float32).min
    x[8], x[8, 19999:] = torch.finfo(torch.float32).min, 2.0
    targets = [3, 500, 1, 0, 0, 70, 3, 20010, 20010]
    check(ctx, x, targets, 8)
    check(ctx, x, [4, 1, 2, 1, 1, 71, 5, 0, 0], 32, stride=20012)


def test_targets_outside_and_outputs_left_out(ctx):
    x = logits(4, 1000, 7)
    check(ctx, x, [-1, 1000, 2 ** 31 - 1, -(2 ** 31)], 2)
    check(ctx, x, [1, 2, 3, 4], 2, entropy=False)
    check(ctx, x, [1, 2, 3, 4], 2, lp=False)
    check(ctx, x, [1, 2, 3, 4], 0, lp=False)
    ctx.logprobs_dev(0, 0, 1000, stream=stream())


def test_the_largest_vocabulary(ctx):
    check(ctx, logits(2, 1 << 22, 8), [5, (1 << 22) - 1], 20)


def test_captured_and_twice_the_same(ctx):
    x, t = logits(7, 9001, 9), torch.arange(7, dtype=torch.int32, device="cuda")
    lp, ent, ids, tops = torch.zeros(7, device="cuda"), torch.zeros(7, device="cuda"), torch.zeros(7, 4, dtype=torch.int32, device="cuda"), torch.zeros(7, 4, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def call():
        ctx.logprobs_dev(x.data_ptr(), 7, 9001, t.data_ptr(), lp.data_ptr(), ent.data_ptr(), 4, ids.data_ptr(), tops.data_ptr(), stream=stream())

    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        for i in range(3):
            x.copy_(logits(7, 9001, 20 + i))
            graph.replay()
            kept = [v.clone() for v in (lp, ent, ids, tops)]
            call()
            assert all(torch.equal(a, b) for a, b in zip(kept, (lp, ent, ids, tops)))


def test_refusals(ctx):
    x = logits(2, 100, 1)
    o = torch.zeros(400, device="cuda")
    p, q, s = x.data_ptr(), o.data_ptr(), stream()
    for kw in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(stride=99), dict(top=33, top_ids_ptr=q, top_logprobs_ptr=q + 800), dict(top=-1),
               dict(top=1), dict(top=1, top_ids_ptr=q + 800), dict(targets_ptr=0), dict(logprobs_ptr=0), dict(logprobs_ptr=p), dict(entropy_ptr=q + 100),
               dict(logits_ptr=0), dict(entropy_ptr=q + 402)):
        with pytest.raises(sc.BackendError):
            ctx.logprobs_dev(**{**dict(logits_ptr=p, rows=2, vocab=100, targets_ptr=q, logprobs_ptr=q + 100, stream=s), **kw})
    torch.cuda.synchronize()
