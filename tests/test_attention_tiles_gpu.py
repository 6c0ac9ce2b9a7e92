"""Attention (strata_cuda_attention_dev) of bf16 chunks in tiles of 128 rows: the cache's layouts, strides, far pages, captured
calls, running maxima that move late and long contexts, each over calls that the rule of attention.cu sends there. The cases,
the formula in 64 bits and the tolerances are test_attention_gpu.py's."""
import math
import re
from pathlib import Path

import pytest

import strata_cuda as sc
from test_attention_gpu import Case, ctx, torch  # noqa: F401

pytestmark = pytest.mark.gpu
SOURCE = (Path(sc.__file__).parent / "csrc" / "attention.cu").read_text()
ROWS, ALL = (int(n) for n in re.search(r"kTcRows = (\d+), kTcAll = (\d+);", SOURCE).groups())


def tiled(*args, **kw):
    """A case that the rule sends to the tiles: some sequence has rows enough, and those that have are enough together."""
    c = Case(*args, **kw)
    enough = -(-ROWS // (c.hq // c.hkv))
    assert c.dtype == "bf16" and c.d <= 128 and sum(n for n in c.lens if n >= enough) * c.hq >= ALL
    wide = [c.qbuf.data_ptr(), c.obuf.data_ptr(), c.qbuf.stride(0) * 2, c.obuf.stride(0) * 2]
    assert not any(v % 16 for v in wide)
    return c


@pytest.mark.parametrize("layout", ["tokens", "heads", "both"])
@pytest.mark.parametrize("d,page", [(64, 16), (64, 128), (128, 32), (128, 48), (72, 16), (8, 256)])
def test_layouts_and_strides(ctx, layout, d, page):  # noqa: F811
    tiled([600, 1, 200], [70, 40, 333], 4, 2, d, page, layout=layout).check(ctx)
    tiled([600, 1, 200], [70, 40, 333], 4, 2, d, page, layout=layout, q_pad=64, o_pad=128).check(ctx)
    tiled([130, 700], [333, 0], 6, 3, d, page, layout=layout, q_pad=8, o_pad=24, window=200, sinks=9).check(ctx)


def test_rows_between_and_behind_the_sequences_stay(ctx):  # noqa: F811
    tiled([300, 0, 5, 260], [4, 9, 0, 77], 4, 2, 128, 16, offsets=[7, 307, 307, 312, 572]).check(ctx)


@pytest.mark.parametrize("d", [64, 128])
def test_large_scores(ctx, d):  # noqa: F811
    """Scores of some hundreds, over several tiles of keys: one key has nearly all the weight, wherever it lies."""
    tiled([600, 300], [300, 1000], 4, 2, d, 16, gain=20.0).check(ctx)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("rising", [True, False])
def test_maxima_that_move_late(ctx, rising, window, d):  # noqa: F811
    """Keys that grow along the sequence: a row's maximum leaves what its first tiles gave by far more than 2^8, again and
    again, with outputs that are not zero by then. And the other way round."""
    n, past = 600, 1500
    c = tiled([n], [past], 4, 2, d, 32, window=window, sinks=4 if window else 0, gain=3.0)
    j = torch.arange(n + past, device="cuda")
    where = c.table[0].long()[j // 32], j % 32
    ramp = torch.exp2(torch.linspace(-4, 5, n + past, device="cuda"))
    c.k[where] = (c.k[where].float() * (ramp if rising else ramp.flip(0))[:, None, None]).bfloat16()
    if rising and not window:
        # the largest score of each tile of 128 keys that the last row sees, in powers of two, moves by 2^8 more than twice
        s = c.q[-1, 0].double() @ c.k[where][:, 0].double().T * c.scale * math.log2(math.e)
        top, moves = s[:128].max(), 0
        for t in range(128, n + past, 128):
            if s[t:t + 128].max() > top + 8:
                top, moves = s[t:t + 128].max(), moves + 1
        assert moves > 2
    c.check(ctx)


@pytest.mark.parametrize("lens,past,heads", [([1024], [20000], (8, 2, 128)), ([300], [60000], (8, 1, 64)), ([40, 700], [33000, 5], (12, 4, 96))], ids=str)
def test_long_contexts(ctx, lens, past, heads):  # noqa: F811
    tiled(lens, past, *heads, 64).check(ctx)


def test_a_long_cache(ctx):  # noqa: F811
    """Pages whose elements lie behind 2^32 of them (8 GiB a pool, one pool for both): the same bits as from near ones."""
    page, hkv, d, n = 64, 8, 128, 1 << 16
    pool = torch.empty(n, 2, page, hkv, d, dtype=torch.bfloat16, device="cuda")
    assert (n - 100) * 2 * page * hkv * d > 2 ** 32
    c = tiled([1, 300], [300, 100], 8, hkv, d, page)
    far = torch.arange(n - c.pages, n, device="cuda")
    pool[far, 0], pool[far, 1] = c.k, c.v
    table = torch.where(c.table >= 0, c.table + (n - c.pages), -1)
    near = c.run(ctx).clone()
    c.check(ctx)
    c.cache = sc.KvCache(pool.data_ptr(), pool[0, 1].data_ptr(), table.data_ptr(), c.len.data_ptr(), n_pages=n, page_size=page, n_kv_head=hkv,
                         head_dim=d, max_pages=c.width, page_stride=2 * page * hkv * d)
    c.obuf.fill_(7.0)
    assert torch.equal(c.run(ctx), near)
    torch.cuda.synchronize()


def test_a_captured_call_follows_lengths_and_pages(ctx):  # noqa: F811
    c = tiled([1, 300, 260], [600, 500, 20], 4, 2, 64, 16, width=64)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.run(ctx)
        for lens in ([601, 800, 280], [13, 300, 261], [300, 799, 100]):
            c.len.copy_(torch.tensor(lens))
            c.table[1, :50] = c.table[1, :50].flip(0).contiguous()
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


def test_two_calls_at_once(ctx):  # noqa: F811
    cases = [tiled([300, 1, 40, 700], [500, 77, 9, 300 + i], 8, 2, 128, 16, seed=i) for i in range(2)]
    alone = []
    for c in cases:
        c.check(ctx)
        alone.append(c.obuf.clone())
        c.obuf.fill_(7.0)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(cases, streams):
            c.run(ctx, s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(c.obuf, a) for c, a in zip(cases, alone))
