"""Sampling (strata_cuda_sample_dev) against its definition: the filters one after another on sorted f64 values.

Ids must be equal. A log-probability is a f64 value rounded once: 2^-24 of itself, and 1e-9 for sums taken in another order."""
import math

import numpy as np
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def expected(x, t, k, p, m, u):
    """One row by the definition in strata_sequence.h."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, -math.inf
    if not t > 0:
        return int(order[0]), 0.0
    top = x[order[0]]
    d = np.where(x == top, 0.0, x - top) if np.isfinite(top) else np.where(x == top, 0.0, -np.inf)
    if k > 0:
        order = order[:k]
    if p < 1:
        e = np.exp(d[order])
        before = np.concatenate([[0.0], np.cumsum(e)[:-1]])
        order = order[:max(1, int((before < p * e.sum()).sum()))]
    if m > 0:
        keep = np.exp(d[order]) >= m
        keep[0] = True
        order = order[keep]
    order = np.sort(order)
    with np.errstate(invalid="ignore"):
        w = np.where(d[order] == 0, 1.0, np.where(d[order] < -1e300, 0.0, np.exp(d[order] / t)))
    c = np.cumsum(w)
    u = u if u > 0 else 0.0
    hit = np.nonzero((c > u * c[-1]) & (w > 0))[0]
    at = hit[0] if len(hit) else np.nonzero(w)[0][-1]
    return int(order[at]), math.log(w[at] / c[-1])


def dev(v, dtype):
    return None if v is None else torch.tensor(v, dtype=dtype, device="cuda")


def draw(ctx, logits, u, t=None, k=None, p=None, m=None, stride=0, logprobs=True):
    rows, vocab = len(u), (logits.shape[1] if not stride else logits.shape[1])
    ids = torch.full((rows + 8,), -77, dtype=torch.int32, device="cuda")
    lps = torch.full((rows + 8,), 77.0, dtype=torch.float32, device="cuda")
    arrays = [dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(m, torch.float32)]
    ud = torch.tensor(u, dtype=torch.float64, device="cuda")
    at = [a.data_ptr() if a is not None else 0 for a in arrays]
    ctx.sample_dev(logits.data_ptr(), rows, vocab, ud.data_ptr(), ids.data_ptr(), lps.data_ptr() if logprobs else 0,
                   temperature_ptr=at[0], top_k_ptr=at[1], top_p_ptr=at[2], min_p_ptr=at[3], stride=stride, stream=stream())
    torch.cuda.synchronize()
    assert bool((ids[rows:] == -77).all()) and bool((lps[rows:] == 77).all())
    return ids[:rows].cpu().numpy(), lps[:rows].cpu().numpy()


def check(ctx, logits, u, t=None, k=None, p=None, m=None):
    """logits: rows x vocab f32 (numpy)."""
    rows = logits.shape[0]
    ids, lps = draw(ctx, torch.from_numpy(logits).cuda(), u, t, k, p, m)
    f32 = lambda v, off: [off] * rows if v is None else [float(np.float32(x)) for x in v]  # noqa: E731
    for r in range(rows):
        want, lp = expected(logits[r].copy(), f32(t, 1.0)[r], 0 if k is None else k[r], f32(p, 1.0)[r], f32(m, 0.0)[r], u[r])
        assert ids[r] == want, (r, ids[r], want)
        if math.isinf(lp):
            assert lps[r] == lp
        else:
            assert abs(lps[r] - lp) <= 2.0 ** -23 * abs(lp) + 1e-9, (r, lps[r], lp)


MODES = {"plain": {}, "greedy": dict(t=0.0), "top_k": dict(k=40), "top_p": dict(p=0.9), "min_p": dict(m=0.05),
         "all": dict(t=0.7, k=200, p=0.95, m=0.02), "wide": dict(t=1.5, k=5000, p=0.999), "one": dict(k=1), "hot": dict(t=4.0, p=0.99)}


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1024, 2049, 4097, 32003, 151936])
def test_vocabularies(ctx, vocab, mode):
    rng = np.random.default_rng(vocab)
    rows = 5 if vocab < 100000 else 3
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    check(ctx, x, list(rng.random(rows)), **{a: [v] * rows for a, v in MODES[mode].items()})


@pytest.mark.parametrize("mode", ["plain", "top_k", "top_p", "min_p", "all", "greedy"])
def test_a_row_too_long_for_shared_memory(ctx, mode):
    rng = np.random.default_rng(9)
    x = (rng.standard_normal((2, 700001)) * 2).astype(np.float32)
    check(ctx, x, [0.3, 0.999], **{a: [v] * 2 for a, v in MODES[mode].items()})


def test_settings_differ_by_row(ctx):
    rng = np.random.default_rng(1)
    rows = 70
    x = (rng.standard_normal((rows, 20011)) * 2.5).astype(np.float32)
    check(ctx, x, list(rng.random(rows)), t=list(rng.choice([0.0, 0.3, 1.0, 2.0], rows)), k=[int(v) for v in rng.choice([0, -1, 1, 7, 300, 50000], rows)],
          p=list(rng.choice([0.1, 0.5, 0.9, 0.999, 1.0, 2.0], rows)), m=list(rng.choice([0.0, 0.01, 0.2, 1.0], rows)))


@pytest.mark.parametrize("vocab", [50, 3000, 40000])
def test_equal_logits_rank_by_index(ctx, vocab):
    x = np.full((6, vocab), -1.25, np.float32)
    check(ctx, x, [0.0, 0.5, 0.999999, 0.25, 0.75, 0.5], k=[0, 10, 10, 0, 17, vocab - 1], p=[1.0, 1.0, 0.5, 0.25, 0.999, 0.5])
    rng = np.random.default_rng(vocab)
    y = (np.round(rng.standard_normal((12, vocab)) * 3) / 2).astype(np.float32)  # a dozen distinct values
    check(ctx, y, list(rng.random(12)), k=[0, 5, 40, 100, 333, 0] * 2, p=[0.3, 0.9, 1.0, 0.8, 0.5, 0.99] * 2)


def test_zero_of_either_sign_is_one_value(ctx):
    x = np.array([[-0.0, 0.0, -0.0, 0.0, -1.0]], np.float32)
    check(ctx, np.repeat(x, 4, 0), [0.0, 0.3, 0.6, 0.9], k=[2, 2, 3, 1])


def test_masked_rows(ctx):
    """-inf, NaN and the lowest float as masks; a row with one token, and rows with none."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((8, 5003)) * 2).astype(np.float32)
    x[0, rng.random(5003) < 0.999] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 100:] = np.finfo(np.float32).min
    x[4, :] = -np.inf
    x[4, 4999] = -3.0
    x[5, ::2] = np.nan
    x[6] = np.finfo(np.float32).min
    x[7, :5000] = -np.inf
    for kw in (dict(), dict(k=[50] * 8), dict(p=[0.9] * 8), dict(m=[0.1] * 8), dict(t=[0.0] * 8), dict(t=[0.6] * 8, k=[2] * 8, p=[0.7] * 8, m=[0.3] * 8)):
        check(ctx, x, list(rng.random(8)), **kw)


def test_infinite_logits_share_everything(ctx):
    x = np.zeros((4, 3001), np.float32)
    x[:, [5, 1700, 2999]] = np.inf
    check(ctx, x, [0.0, 0.4, 0.9, 0.99], p=[1.0, 0.9, 0.5, 1.0], k=[0, 0, 0, 2], t=[1.0, 0.5, 3.0, 1.0])


def test_far_logits(ctx):
    """Differences that f32 cannot hold, and tokens far below the first histogram's range."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((4, 9001)) * 200).astype(np.float32)
    x[1] *= 1e35
    x[2] = np.linspace(-300, 50, 9001, dtype=np.float32)
    check(ctx, x, [0.1, 0.5, 0.7, 0.999], k=[3000, 4000, 8000, 9000], p=[1.0, 1.0, 0.9, 1.0], t=[100.0, 1.0, 30.0, 2.0])
    x = (rng.standard_normal((3, 9001)) * 1e-20).astype(np.float32)  # all but equal, thousands of different keys
    check(ctx, x, [0.1, 0.5, 0.999], k=[0, 777, 5000], p=[0.5, 1.0, 0.3])


def test_edges_of_the_settings(ctx):
    nan, inf = float("nan"), float("inf")
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((1, 2500)) * 2).astype(np.float32)
    for kw in (dict(p=[0.0]), dict(p=[-1.0]), dict(p=[1e-30]), dict(p=[float(np.nextafter(np.float32(1), np.float32(0)))]), dict(m=[2.0]), dict(m=[1.0]),
               dict(m=[1e-44]), dict(t=[1e-30]), dict(t=[-2.0]), dict(t=[inf]), dict(k=[2**31 - 1]), dict(k=[-2**31]), dict(k=[2500]), dict(k=[2499])):
        for u in (0.0, 0.37, 1 - 2.0 ** -53):
            check(ctx, x, [u], **kw)
    for off, same in ((dict(p=[nan]), {}), (dict(m=[nan]), {}), (dict(t=[nan]), dict(t=[0.0]))):
        assert draw(ctx, torch.from_numpy(x).cuda(), [0.6], **off)[0][0] == draw(ctx, torch.from_numpy(x).cuda(), [0.6], **same)[0][0]


def test_random_numbers_outside_the_interval(ctx):
    x = np.zeros((1, 100), np.float32)
    x[0, 60:] = -np.inf
    xd = torch.from_numpy(x).cuda()
    for u, want in ((0.0, 0), (-5.0, 0), (float("nan"), 0), (1.0, 59), (7.0, 59), (float("inf"), 59)):
        assert draw(ctx, xd, [u])[0][0] == want


@pytest.mark.parametrize("vocab", [9000, 60001])
@pytest.mark.parametrize("kw", [dict(), dict(t=0.01), dict(p=0.9), dict(p=0.9, t=0.005), dict(p=0.99, t=3.0), dict(k=50), dict(m=0.1)], ids=str)
def test_the_ends_of_the_interval_pass_over_masked_stretches(ctx, vocab, kw):
    """The smallest and largest random numbers, with most of the row masked on the side that they point at."""
    rng = np.random.default_rng(vocab)
    near = 1 - 2.0 ** (-53 if kw.get("t", 1) >= 1 else -40)  # closer, and sums of tiny weights would decide by their order
    u = [0.0, 2.0 ** -53, 1e-300, near, 1.0, 5.0, 0.5]
    for masked in (slice(0, vocab * 3 // 4), slice(vocab // 4, vocab)):
        for mask in (-np.inf, np.nan, np.finfo(np.float32).min, -1e4):
            x = (rng.standard_normal((1, vocab)) * 2).astype(np.float32).repeat(len(u), 0)
            x[:, masked] = mask
            got = [int(v) for v in draw(ctx, torch.from_numpy(x).cuda(), u, **{a: [v] * len(u) for a, v in kw.items()})[0]]
            f32 = {a: float(np.float32(v)) if a != "k" else v for a, v in kw.items()}
            want = [expected(x[0].copy(), f32.get("t", 1.0), f32.get("k", 0), f32.get("p", 1.0), f32.get("m", 0.0), min(v, 1.0))[0] for v in u]
            assert got == want


@pytest.mark.parametrize("rows,vocab", [(1, 20000), (2, 120001), (40, 9001), (80, 5000), (150, 16384), (150, 16383)])
@pytest.mark.parametrize("sigma", [0.02, 0.1, 0.5])
def test_lists_of_every_length(ctx, rows, vocab, sigma):
    """Nearly flat rows: a border's bins hold hundreds to tens of thousands of tokens, for each number of blocks a row takes."""
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * sigma + 3).astype(np.float32)
    u = list(rng.random(rows))
    k = [int(v) for v in rng.choice([300, 900, 1500, 3900, 4500], rows)]
    for kw in (dict(k=k), dict(k=k, p=[0.4] * rows), dict(p=list(rng.choice([0.01, 0.1, 0.5, 0.98], rows))),
               dict(m=list(rng.choice([0.999, 0.9, 0.5], rows))), dict(k=k, p=[0.7] * rows, m=[0.8] * rows, t=[0.3] * rows)):
        check(ctx, x, u, **kw)


@pytest.mark.parametrize("rows,vocab", [(1, 3500), (3, 20000), (40, 3999), (160, 3600)])
def test_crowds_of_equal_and_nearly_equal_logits(ctx, rows, vocab):
    """Rounded logits (hundreds of one value), and thousands of different ones within a hair beside a few far above."""
    rng = np.random.default_rng(rows)
    u = list(rng.random(rows))
    k = [int(v) for v in rng.choice([100, 300, 700, 1500, 2500, 3400], rows)]
    p = list(rng.choice([0.2, 0.6, 0.9, 0.97], rows))
    rounded = np.round(rng.standard_normal((rows, vocab)) * 1.5 * 8) / 8
    close = rng.standard_normal((rows, vocab)) * 1e-5
    close[:, rng.integers(0, vocab, 3)] = 11.0
    halves = np.where(rng.random((rows, vocab)) < 0.1, rng.standard_normal((rows, vocab)), np.round(rng.standard_normal((rows, vocab))))
    for x in (rounded, close, halves):
        for kw in (dict(k=k), dict(p=p), dict(k=k, p=p), dict(k=k, p=p, m=[0.001] * rows, t=[1.7] * rows), dict(p=p, t=[0.5] * rows)):
            check(ctx, x.astype(np.float32), u, **kw)


def test_a_nearly_flat_row_too_long_for_shared_memory(ctx):
    rng = np.random.default_rng(21)
    x = (rng.standard_normal((2, 700001)) * 0.1).astype(np.float32)
    for kw in (dict(k=[300000, 2000]), dict(p=[0.5, 0.002]), dict(m=[0.9, 0.7])):
        check(ctx, x, [0.2, 0.8], **kw)


@pytest.mark.parametrize("center", [12345.0, -9990.0, -70000.0, 3e38])
def test_logits_far_from_zero(ctx, center):
    """f32 holds few steps between them: many tokens are equal, and all lie above or below the histogram's bins."""
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((6, 9000)) * (3 if center < 1e30 else 1e31) + center).astype(np.float32)
    u = list(rng.random(6))
    for kw in (dict(), dict(k=[5, 50, 700, 1500, 5000, 8999]), dict(p=[0.05, 0.3, 0.5, 0.9, 0.99, 0.999]), dict(m=[0.5, 0.1, 0.01] * 2)):
        check(ctx, x, u, **kw)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_that_start_anywhere(ctx, shift):
    rng = np.random.default_rng(shift)
    x = (rng.standard_normal((3, 8192)) * 2).astype(np.float32)
    whole = torch.full((shift + x.size,), 99.0, device="cuda")
    view = whole[shift:].view(3, 8192)
    view.copy_(torch.from_numpy(x))
    u = list(rng.random(3))
    ids, _ = draw(ctx, view, u, p=[0.9] * 3)
    assert [expected(x[r].copy(), 1.0, 0, float(np.float32(0.9)), 0.0, u[r])[0] for r in range(3)] == list(ids)


def test_every_random_number_lands_in_its_token(ctx):
    """The unit interval split by the cumulative probabilities: 4096 draws from one distribution."""
    w = np.array([1, 2, 0, 5, 3, 1, 4], np.float64)
    with np.errstate(divide="ignore"):
        x = np.repeat(np.log(w)[None].astype(np.float32), 4096, 0)
    u = (np.arange(4096) + 0.5) / 4096
    ids, _ = draw(ctx, torch.from_numpy(x).cuda(), list(u))
    assert np.array_equal(ids, np.searchsorted(np.cumsum(w) / w.sum(), u, side="right"))


def test_rows_apart_and_no_logprobs(ctx):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, 1500)).astype(np.float32)
    whole = torch.full((9, 1777), 50.0, device="cuda")  # what lies between the rows would win
    whole[:, :1500] = torch.from_numpy(x).cuda()
    u = list(rng.random(9))
    rows = torch.as_strided(whole, (9, 1500), (1777, 1))
    ids, lps = draw(ctx, rows, u, k=[30] * 9, stride=1777, logprobs=False)
    assert (lps == 77).all()
    assert [expected(x[r].copy(), 1.0, 30, 1.0, 0.0, u[r])[0] for r in range(9)] == list(ids)


def test_many_rows(ctx):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((1500, 257)) * 2).astype(np.float32)
    check(ctx, x, list(rng.random(1500)), p=[0.9] * 1500, k=[100] * 1500)


def test_the_same_bits_again_and_on_two_streams(ctx):
    logits = torch.randn(40, 50000, device="cuda") * 2.5
    u = torch.rand(40, dtype=torch.float64, device="cuda")
    p = torch.full((40,), 0.95, device="cuda")
    outs = []
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        ids, lps = torch.empty(40, dtype=torch.int32, device="cuda"), torch.empty(40, device="cuda")
        outs.append((ids, lps))
        torch.cuda.synchronize()
        ctx.sample_dev(logits.data_ptr(), 40, 50000, u.data_ptr(), ids.data_ptr(), lps.data_ptr(), top_p_ptr=p.data_ptr(), stream=streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1]) for a, b in outs)


def test_captured_and_replayed(ctx):
    logits, u = torch.empty(3, 7001, device="cuda"), torch.empty(3, dtype=torch.float64, device="cuda")
    k = torch.tensor([50, 0, 7], dtype=torch.int32, device="cuda")
    ids = torch.empty(3, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ctx.sample_dev(logits.data_ptr(), 3, 7001, u.data_ptr(), ids.data_ptr(), top_k_ptr=k.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        x, us = (rng.standard_normal((3, 7001)) * 2).astype(np.float32), rng.random(3)
        logits.copy_(torch.from_numpy(x))
        u.copy_(torch.from_numpy(us))
        g.replay()
        torch.cuda.synchronize()
        assert list(ids.cpu()) == [expected(x[r].copy(), 1.0, [50, 0, 7][r], 1.0, 0.0, us[r])[0] for r in range(3)]


def test_refusals(ctx):
    x = torch.zeros(1 << 16, device="cuda")
    p = x.data_ptr()

    def call(code, logits=p, rows=2, vocab=100, u=p + 4096, ids=p + 8192, **kw):
        with pytest.raises(sc.BackendError) as e:
            ctx.sample_dev(logits, rows, vocab, u, ids, stream=stream(), **kw)
        assert e.value.code == code and "sample" in str(e.value)

    call(sc.ERR_INVALID, logits=0)
    call(sc.ERR_INVALID, u=0)
    call(sc.ERR_INVALID, ids=0)
    call(sc.ERR_INVALID, rows=0)
    call(sc.ERR_INVALID, vocab=0)
    call(sc.ERR_INVALID, vocab=(1 << 22) + 1)
    call(sc.ERR_INVALID, stride=99)
    call(sc.ERR_INVALID, u=p + 4)
    call(sc.ERR_INVALID, ids=p)
    call(sc.ERR_INVALID, logprobs_ptr=p + 8192)
