"""Attention over a paged cache (strata_cuda_attention_dev) against its formula in 64 bits.

Tolerances, before any run. Let P = sum_j p_j |v_j| (the weights' own formula) and A = max_j scale sum_d |q_d k_jd|.
A score is a chain of f32 sums over products: off by at most 2^-23 a step of 16 elements, of A; its exponent's argument
rounds at 2^-23 of 1.45 A + 1, and the exponential is good to 2^-22. So a weight is off by
    w = 2 (A (D/16 + 8) 2^-23 + (1.45 A + 1) 2^-23) + 2^-22
of itself, in the sum of the weights as well; the sums over n keys add n/16 + 32 roundings of 2^-24 at most. f32 outputs:
(2 w + (n/16 + 32) 2^-23) P + 2^-24 |o|. With bf16 each weight is rounded once more, half a step of bf16 (2^-8), and so
is the output: 2^-8 P + 2^-8 |o| on top."""
import math

import numpy as np
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": (torch.float32, sc.F32), "bf16": (torch.bfloat16, sc.BF16)}


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


class Case:
    """Sequences with `past` tokens before the call and `lens` new ones in a cache of shuffled pages, whose unused rows
    and pages hold NaN. layout: "tokens" [page][token][head][dim], "heads" [page][head][token][dim], "both" one pool
    whose pages hold the keys' tokens, then the values'."""

    def __init__(self, lens, past, hq=4, hkv=2, d=64, page=16, dtype="bf16", window=0, sinks=0, scale=None, layout="tokens", seed=0,
                 offsets=None, q_pad=0, o_pad=0, spare=2, width=None, uniform=None, gain=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.lens, self.past, self.hq, self.hkv, self.d, self.page = lens, past, hq, hkv, d, page
        self.window, self.sinks, self.dtype = window, sinks, dtype
        self.scale = d ** -0.5 if scale is None else scale
        n = len(lens)
        self.offsets = [0] + [int(v) for v in np.cumsum(lens)] if offsets is None else offsets
        self.total = self.offsets[-1]
        self.kv = [a + b for a, b in zip(past, lens)]
        need = [-(-max(0, m) // page) for m in self.kv]
        width = max(1, max(need)) if width is None else width
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
        table, at = torch.full((n, width), -1, dtype=torch.int32), 0
        for i, m in enumerate(need):
            table[i, :m] = order[at:at + m]
            at += m
        self.table, self.len = table.cuda(), torch.tensor(self.kv, dtype=torch.int32, device="cuda")
        self.pages, self.width = pages, width
        nan = lambda *s: torch.full(s, math.nan, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        if layout == "tokens":
            self.pool = [nan(pages, page, hkv, d), nan(pages, page, hkv, d)]
            self.k, self.v, self.strides = self.pool[0], self.pool[1], {}
        elif layout == "heads":
            self.pool = [nan(pages, hkv, page, d), nan(pages, hkv, page, d)]
            self.k, self.v = (x.transpose(1, 2) for x in self.pool)
            self.strides = dict(token_stride=d, head_stride=page * d)
        else:
            self.pool = [nan(pages, 2, page, hkv, d)]
            self.k, self.v = self.pool[0][:, 0], self.pool[0][:, 1]
            self.strides = dict(page_stride=2 * page * hkv * d)
        for i, m in enumerate(self.kv):
            if m > 0:
                j = torch.arange(m, device="cuda")
                where = self.table[i].long()[j // page], j % page
                self.k[where] = rand(m, hkv, d).bfloat16()
                self.v[where] = rand(m, hkv, d).bfloat16()
        td, self.code = DT[dtype]
        self.qbuf = (rand(self.total + 3, hq * d + q_pad) * gain).to(td)
        self.obuf = torch.full((self.total + 3, hq * d + o_pad), 7.0, dtype=td, device="cuda")
        self.q = self.qbuf[: self.total, : hq * d].unflatten(1, (hq, d))
        self.cache = sc.KvCache(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.len.data_ptr(), n_pages=pages, page_size=page,
                                n_kv_head=hkv, head_dim=d, max_pages=width, **self.strides)
        how = dict(seq_len=uniform) if uniform is not None else dict(offsets=self.offsets)
        self.shape = sc.Attention(n, hq, self.scale, dtype=self.code, window=window, sinks=sinks, q_stride=hq * d + q_pad, o_stride=hq * d + o_pad, **how)
        self.work = torch.empty(max(16, sc.attention_work_bytes(self.shape, self.cache)), dtype=torch.uint8, device="cuda").fill_(0xFF)

    def run(self, ctx, s=None):
        ctx.attention_dev(self.shape, self.cache, self.qbuf.data_ptr(), self.obuf.data_ptr(), self.work.data_ptr(), self.work.numel(), stream() if s is None else s)
        return self.obuf

    def want(self):
        """o, and how far it may be off."""
        o = torch.zeros(self.total, self.hq, self.d, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(o)
        r = self.hq // self.hkv
        for i, (a, b) in enumerate(zip(self.offsets, self.offsets[1:])):
            n = b - a
            m = max(0, int(self.len[i]))
            if n == 0 or m == 0:
                continue
            j = torch.arange(min(m, self.width * self.page), device="cuda")
            pg = self.table[i].long()[j // self.page]
            placed = (pg >= 0) & (pg < self.pages)
            at = pg.clamp(0, self.pages - 1), j % self.page
            k, v = self.k[at].double(), self.v[at].double()
            for t in range(0, n, 256):
                u = min(n, t + 256)
                p = torch.arange(m - n + t, m - n + u, device="cuda")[:, None]
                seen = (j <= p) & placed
                if self.window:
                    seen &= (j > p - self.window) | (j < self.sinks)
                for h in range(self.hkv):
                    q = self.q[a + t:a + u, h * r:(h + 1) * r].double()
                    kh = torch.where(seen.any(0)[:, None], k[:, h], 0.0)
                    vh = torch.where(seen.any(0)[:, None], v[:, h], 0.0)
                    x = torch.where(seen[:, None], q @ kh.T * self.scale, -math.inf)
                    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
                    w = torch.where(seen[:, None], e / e.sum(-1, keepdim=True).clamp(min=1e-300), 0.0)
                    got = w @ vh
                    big = (q.abs() @ kh.abs().T * self.scale * seen[:, None]).amax(-1, keepdim=True)
                    off = 2 * (big * (self.d / 16 + 8) + 1.45 * big + 1) * 2.0 ** -23 + 2.0 ** -22
                    part = (2 * off + (len(j) / 16 + 32) * 2.0 ** -23) * (w @ vh.abs()) + 2.0 ** -24 * got.abs()
                    if self.dtype == "bf16":
                        part += 2.0 ** -8 * (w @ vh.abs() + got.abs())
                    o[a + t:a + u, h * r:(h + 1) * r], tol[a + t:a + u, h * r:(h + 1) * r] = got, part
        return o, tol

    def check(self, ctx):
        self.run(ctx)
        torch.cuda.synchronize()
        o, tol = self.want()
        got = self.obuf[: self.total, : self.hq * self.d].unflatten(1, (self.hq, self.d)).double()
        live = torch.zeros(self.total, dtype=torch.bool, device="cuda")
        for a, b in zip(self.offsets, self.offsets[1:]):
            live[a:b] = True
        bad = ~((got - o).abs() <= tol + 1e-30) & live[:, None, None]
        assert not bad.any(), (bad.nonzero()[:4].tolist(), (got - o).abs()[bad][:4].tolist(), tol[bad][:4].tolist())
        # nothing else is written
        assert (self.obuf[self.total:] == 7).all() and (self.obuf[:, self.hq * self.d:] == 7).all() and (got[~live] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(4, 2, 64), (1, 1, 8), (8, 1, 128), (9, 3, 80), (4, 4, 256), (20, 1, 72), (16, 2, 200), (40, 2, 16)], ids=str)
def test_single_tokens(ctx, heads, dtype):
    hq, hkv, d = heads
    past = [0, 1, 15, 16, 17, 63, 64, 65, 127, 500, 1037]
    Case([1] * len(past), past, hq, hkv, d, dtype=dtype, uniform=1).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256, 40])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_chunks(ctx, page, d, dtype):
    Case([1, 130, 0, 7, 64, 300], [5, 0, 9, 700, 129, 257], 6, 2, d, page, dtype, seed=page).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (16, 0), (64, 4), (100, 63), (100, 64), (100, 65), (129, 200), (4000, 2), (1 << 40, 1)])
def test_windows(ctx, window, sinks, dtype):
    Case([1, 1, 90, 33, 1], [0, 900, 100, 1500, 64], 6, 2, 64, 16, dtype, window, sinks).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,past,window", [(1500, 0, 0), (700, 1111, 0), (1025, 64, 200), (257, 8000, 1000)])
def test_long_chunks(ctx, n, past, window, dtype):
    Case([n], [past], 4, 1, 128, 64, dtype, window, 5 if window else 0).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["tokens", "heads", "both"])
def test_layouts_and_strides(ctx, layout, dtype):
    Case([3, 1, 200], [70, 40, 33], 4, 2, 64, 32, dtype, layout=layout, q_pad=5, o_pad=3).check(ctx)
    Case([3, 1, 200], [70, 40, 33], 4, 2, 64, 32, dtype, layout=layout, q_pad=64, o_pad=128).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_sequences(ctx, dtype):
    n = 700
    past = [(i * 37) % 200 for i in range(n)]
    Case([1] * n, past, 2, 1, 64, 16, dtype, uniform=1).check(ctx)
    Case([i % 3 for i in range(n)], past, 2, 1, 64, 16, dtype).check(ctx)


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (64, 4), (100, 65), (129, 200), (1 << 40, 1)])
def test_windows_in_tiles(ctx, window, sinks):
    """As test_windows, with rows enough for the tiles of 128 rows, one sequence with a single tile of them."""
    Case([1, 1, 190, 33, 430], [0, 900, 100, 1500, 64], 9, 3, 64, 16, "bf16", window, sinks).check(ctx)
    Case([333, 20], [700, 0], 8, 2, 128, 48, "bf16", window, sinks).check(ctx)


def test_lengths_and_pages_in_tiles(ctx):
    n = 300
    c = Case([n, n, n, n], [3, 0, 0, 50], 4, 2, 64, 16, "bf16")
    c.len.copy_(torch.tensor([n // 2, 0, -5, n + 50]))
    c.check(ctx)
    c = Case([n, n, n], [400, 400, 300], 4, 2, 128, 16, "bf16")
    c.table[0, 3], c.table[0, 7], c.table[0, 8] = -1, c.pages, -(2 ** 31)
    c.table[1, :] = 2 ** 31 - 1
    c.check(ctx)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_in_tiles(ctx, value):
    n, past = 700, 200
    for window, at in ((0, past + 400), (300, 20)):
        c = Case([n], [past], 4, 2, 64, 32, "bf16", window, 3 if window else 0)
        where = c.table[0, at // 32].long(), at % 32
        clean_k, clean_v = c.k[where].clone(), c.v[where].clone()
        want, tol = c.want()
        p = torch.arange(past, past + n, device="cuda")
        blind = (at > p) | (p - at >= window) if window else at > p
        for pool in (c.k, c.v):
            pool[where] = value
            c.run(ctx)
            torch.cuda.synchronize()
            got = c.obuf[:n, :4 * 64].unflatten(1, (4, 64)).double()
            assert blind.any() and ((got - want).abs() <= tol)[blind].all()
            if pool is c.v and not blind.all():
                assert not torch.isfinite(got[~blind]).any(-1).any()
            c.k[where], c.v[where] = clean_k, clean_v
    c = Case([n], [past], 4, 2, 64, 32, "bf16")
    want, tol = c.want()
    c.q[n - 1, 1, 5] = value
    c.run(ctx)
    got = c.obuf[:n].unflatten(1, (4, 64)).double()
    others = torch.ones(n, 4, dtype=torch.bool, device="cuda")
    others[n - 1, 1] = False
    assert ((got - want).abs() <= tol)[others].all() and torch.isnan(got[n - 1, 1]).all()


@pytest.mark.parametrize("lens,heads", [([512], (8, 1)), ([255], (8, 1)), ([40, 40], (32, 8)), ([17], (64, 4)), ([2100], (1, 1))], ids=str)
def test_few_blocks_of_rows_in_many_pieces(ctx, lens, heads):
    """One block of rows' keys cut over as many thread blocks as there are, behind long contexts."""
    Case(lens, [9000] * len(lens), *heads, 128, 64, "bf16").check(ctx)
    Case(lens, [3000] * len(lens), *heads, 72, 16, "bf16").check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_chunks(ctx, dtype):
    """More sequences than a launch holds, each long enough for tiles of rows; and as many of one length."""
    n = 260
    Case([16 + i % 9 for i in range(n)], [(i * 53) % 150 for i in range(n)], 4, 1, 64, 16, dtype).check(ctx)
    Case([50] * 7, [0, 1, 77, 78, 200, 300, 13], 8, 2, 128, 32, dtype, uniform=50).check(ctx)


@pytest.mark.parametrize("heads", [(20, 1, 72), (64, 1, 16), (7, 7, 104), (3, 1, 128)], ids=str)
def test_chunks_of_other_heads(ctx, heads):
    hq, hkv, d = heads
    Case([40, 1, 200], [100, 5, 0], hq, hkv, d, 16, "bf16").check(ctx)
    Case([40, 1, 200], [100, 5, 0], hq, hkv, d, 64, "bf16", window=77, sinks=20).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3.3e38])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(ctx, value, dtype):
    for n in (1, 150):
        c = Case([n, n], [30, 200], 4, 2, 64, 16, dtype)
        want, tol = c.want()
        c.q[n - 1, 1, 5] = value
        c.run(ctx)
        torch.cuda.synchronize()
        got = c.obuf[: c.total].unflatten(1, (4, 64)).double()
        others = torch.ones(c.total, 4, dtype=torch.bool, device="cuda")
        others[n - 1, 1] = False
        assert ((got - want).abs() <= tol)[others].all()
        assert torch.isnan(got[n - 1, 1]).all() or math.isfinite(value)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_between_and_behind_the_sequences_stay(ctx, dtype):
    Case([2, 3, 1], [4, 0, 9], 2, 2, 32, 16, dtype, offsets=[5, 7, 10, 11]).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(ctx, dtype):
    """Scores of some hundreds: one key has nearly all the weight."""
    c = Case([1, 60], [300, 100], 4, 2, 128, 16, dtype, gain=20.0)
    c.check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 20, 150])
def test_lengths_shorter_than_the_chunk(ctx, n, dtype):
    """Tokens at negative positions see nothing; a length of zero (or below) leaves no row a key."""
    c = Case([n, n, n, n], [3, 0, 0, 50], 4, 2, 64, 16, dtype)
    c.len.copy_(torch.tensor([n // 2, 0, -5, n + 50]))
    c.check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 150])
def test_pages_that_are_none(ctx, n, dtype):
    """Positions whose page number is none, or behind the table, are as masked."""
    c = Case([n, n, n], [400, 400, 300], 4, 2, 64, 16, dtype)
    c.table[0, 3], c.table[0, 7], c.table[0, 8] = -1, c.pages, -(2 ** 31)
    c.table[1, :] = 2 ** 31 - 1
    c.check(ctx)
    c.len[2] = c.width * c.page + 40  # the last tokens lie behind the table: they see all that is there
    c.k[c.table[2][: c.width].clamp(min=0).long()] = 0.5
    c.v[c.table[2][: c.width].clamp(min=0).long()] = 0.25
    c.check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_never_reaches_it(ctx, value, dtype):
    """NaN and infinities in later tokens' keys and values, and in keys outside the window."""
    n, past = 150, 200
    for window, at in ((0, past + 100), (100, 20)):
        c = Case([n], [past], 4, 2, 64, 16, dtype, window, 3 if window else 0)
        where = c.table[0, at // 16].long(), at % 16
        clean_k, clean_v = c.k[where].clone(), c.v[where].clone()
        want, tol = c.want()
        for pool in (c.k, c.v):
            pool[where] = value
            c.run(ctx)
            torch.cuda.synchronize()
            got = c.obuf[:n, :4 * 64].unflatten(1, (4, 64)).double()
            p = torch.arange(past, past + n, device="cuda")
            blind = (at > p) | ((window > 0) & (at <= p - window)) if window else at > p
            assert blind.any() and ((got - want).abs() <= tol)[blind].all()
            if pool is c.v and not blind.all():
                assert not torch.isfinite(got[~blind]).any(-1).any()
            c.k[where], c.v[where] = clean_k, clean_v


def test_a_long_cache(ctx):
    """Pages whose elements lie behind 2^32 of them (8 GiB a pool, one pool for both)."""
    page, hkv, d, n = 64, 8, 128, 1 << 16
    pool = torch.empty(n, 2, page, hkv, d, dtype=torch.bfloat16, device="cuda")
    assert (n - 100) * 2 * page * hkv * d > 2 ** 32
    for dtype, lens in (("bf16", [1, 200]), ("f32", [1, 20])):
        c = Case(lens, [300, 100], 8, 8, 128, page, dtype)
        far = torch.arange(n - c.pages, n, device="cuda")
        pool[far, 0], pool[far, 1] = c.k, c.v
        table = torch.where(c.table >= 0, c.table + (n - c.pages), -1)
        cache = sc.KvCache(pool.data_ptr(), pool[0, 1].data_ptr(), table.data_ptr(), c.len.data_ptr(), n_pages=n, page_size=page, n_kv_head=hkv,
                           head_dim=d, max_pages=c.width, page_stride=2 * page * hkv * d)
        near = c.run(ctx).clone()
        c.cache = cache
        c.obuf.fill_(7.0)
        assert torch.equal(c.run(ctx), near)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_captured_call_follows_lengths_and_pages(ctx, dtype):
    c = Case([1, 1, 40], [600, 0, 20], 4, 2, 64, 16, dtype, width=64)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.run(ctx)
        for lens in ([601, 1, 60], [13, 1, 55], [300, 1, 60]):
            c.len.copy_(torch.tensor(lens))
            c.table[0, :40] = c.table[0, :40].flip(0).contiguous()
            c.k[torch.isnan(c.k)], c.v[torch.isnan(c.v)] = 0.5, 0.25
            c.obuf.fill_(7.0)
            graph.replay()
            side.synchronize()
            o, tol = c.want()
            got = c.obuf[: c.total].unflatten(1, (4, 64)).double()
            assert ((got - o).abs() <= tol + 1e-30).all()
            again = c.obuf.clone()
            assert torch.equal(c.run(ctx), again)  # the same bits
            side.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_two_calls_at_once(ctx, dtype):
    cases = [Case([1] * 40 + [300], [500 + 7 * i for i in range(41)], 8, 2, 128, 16, dtype, seed=i) for i in range(2)]
    alone = []
    for c in cases:
        alone.append(c.run(ctx).clone())
        torch.cuda.synchronize()
        c.obuf.fill_(7.0)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(cases, streams):
            c.run(ctx, s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(c.obuf, a) for c, a in zip(cases, alone))


def test_nothing_to_do(ctx):
    c = Case([1, 1], [3, 4], 2, 1, 32)
    for how in (dict(seq_len=0), dict(offsets=[0, 0, 0]), dict(offsets=[9, 9, 9])):
        shape = sc.Attention(2, 2, 0.2, **how)
        assert sc.attention_work_bytes(shape, c.cache) == 0
        ctx.attention_dev(shape, c.cache, 0, 0, 0, 0, stream())
    torch.cuda.synchronize()


def test_refusals(ctx):
    c = Case([1, 1], [3, 4], 2, 1, 32)
    q, o, w, n, s = c.qbuf.data_ptr(), c.obuf.data_ptr(), c.work.data_ptr(), c.work.numel(), stream()
    for args in ((0, o, w, n), (q, 0, w, n), (q, o, 0, n), (q, o, w, 16), (q, q, w, n), (q, c.k.data_ptr(), w, n), (q, o, o, n), (q + 1, o, w, n), (q, o, w + 8, n)):
        with pytest.raises(sc.BackendError):
            ctx.attention_dev(c.shape, c.cache, *args, s)
    c.check(ctx)
