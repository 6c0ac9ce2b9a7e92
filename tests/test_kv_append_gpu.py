"""Appending to a paged cache (strata_cuda_kv_append_dev) against its formula in 64 bits.

Tolerances, before any run: sine and cosine are good to 2^-23, a product and a sum round at 2^-24 each, so a turned
element is off by at most 2^-22 (|a| + |b|); one that is rounded to bf16 by half a step more, 2^-8 of itself. What is not
turned is the input rounded once, bit for bit. Rows of the cache that no token of the call has are not touched."""
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


def turned(x, pos, rot, base, neighbours):
    """x [token][head][dim] in 64 bits, and how far f32 may be off."""
    y, tol = x.clone(), torch.zeros_like(x)
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    angle = (pos.double()[:, None] * base ** (-2 * i / rot))[:, None]
    ia, ib = (2 * i.long(), 2 * i.long() + 1) if neighbours else (i.long(), i.long() + rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    tol[..., ia] = tol[..., ib] = 2.0 ** -22 * (a.abs() + b.abs())
    return y, tol


def check(ctx, lens, past, hq=4, hkv=2, d=64, rot=64, page=16, dtype="f32", out="bf16", neighbours=False, base=10000.0, pads=(0, 0, 0, 0),
          layout="tokens", offsets=None, uniform=None, in_place=False, table_change=None, length_change=None):
    g = torch.Generator(device="cuda").manual_seed(d + rot + len(lens))
    n = len(lens)
    off = [0] + [int(v) for v in np.cumsum(lens)] if offsets is None else offsets
    total = off[-1]
    kv = [a + b for a, b in zip(past, lens)]
    need = [-(-m // page) for m in kv]
    width, pages = max(1, max(need)), sum(need) + 2
    order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int(), 0
    table = torch.full((n, width), -1, dtype=torch.int32)
    for i, m in enumerate(need):
        table[i, :m] = order[at:at + m]
        at += m
    if table_change:
        table_change(table, pages)
    length = torch.tensor(kv, dtype=torch.int32)
    if length_change:
        length_change(length)
    table, length = table.cuda(), length.cuda()
    td, code = DT[dtype]
    to, ocode = DT[out]
    buf = [torch.randn(total + 2, h * d + p, generator=g, device="cuda").to(td) for h, p in zip((hq, hkv, hkv), pads)]
    q, k, v = (x[:total, : h * d].unflatten(1, (h, d)) for x, h in zip(buf, (hq, hkv, hkv)))
    q0 = q.double()
    obuf = buf[0] if in_place else torch.full((total + 2, hq * d + pads[3]), 7.0, dtype=to, device="cuda")
    before = obuf.clone()
    shape = (pages, page, hkv, d) if layout == "tokens" else (pages, hkv, page, d)
    pools = [torch.randn(*shape, generator=g, device="cuda").bfloat16() for _ in range(2)]
    kc, vc = pools if layout == "tokens" else (x.transpose(1, 2) for x in pools)
    wk, wv, tk = kc.double(), vc.double(), torch.zeros(kc.shape, dtype=torch.float64, device="cuda")
    wq, tq = before[:total, : hq * d].unflatten(1, (hq, d)).double(), torch.zeros(total, hq, d, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(off, off[1:])):
        m = max(0, int(length[i]))
        pos = torch.arange(m - (b - a), m, device="cuda")
        wq[a:b], tq[a:b] = turned(q0[a:b], pos, rot, base, neighbours)
        kt, tol = turned(k[a:b].double(), pos, rot, base, neighbours)
        for t, p in enumerate(pos.tolist()):
            if 0 <= p < width * page and 0 <= int(table[i, p // page]) < pages:
                where = int(table[i, p // page]), p % page
                wk[where], tk[where], wv[where] = kt[t], tol[t], v[a + t].double()
    cache = sc.KvCache(pools[0].data_ptr(), pools[1].data_ptr(), table.data_ptr(), length.data_ptr(), n_pages=pages, page_size=page, n_kv_head=hkv,
                       head_dim=d, max_pages=width, **(dict(token_stride=d, head_stride=page * d) if layout == "heads" else {}))
    how = dict(seq_len=uniform) if uniform is not None else dict(offsets=off)
    desc = sc.KvAppend(n, hq, rot, base, dtype=code, q_dtype=ocode, neighbours=neighbours, q_stride=buf[0].shape[1], k_stride=buf[1].shape[1],
                       v_stride=buf[2].shape[1], q_out_stride=obuf.shape[1], **how)
    ctx.kv_append_dev(desc, cache, buf[0].data_ptr(), buf[1].data_ptr(), buf[2].data_ptr(), obuf.data_ptr(), stream())
    torch.cuda.synchronize()
    half = 2.0 ** -8
    got = obuf[:total, : hq * d].unflatten(1, (hq, d)).double()
    assert ((got - wq).abs() <= tq + (half * wq.abs() if out == "bf16" else 2.0 ** -24 * wq.abs())).all()
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, b in zip(off, off[1:]):
        live[a:b] = True
    still = torch.cat([torch.arange(rot, d, device="cuda")])
    assert torch.equal(got[live][..., still], q0[live][..., still].to(to).double())
    assert torch.equal(obuf[total:], before[total:]) and torch.equal(obuf[:, hq * d:], before[:, hq * d:]) and torch.equal(got[~live], before[:total, : hq * d].unflatten(1, (hq, d)).double()[~live])
    kd, vd = kc.double(), vc.double()
    assert ((kd - wk).abs() <= tk * (1 + half) + torch.where(tk > 0, half * wk.abs(), 0.0) + torch.where((tk == 0), (wk - wk.bfloat16().double()).abs(), 0.0)).all()
    assert torch.equal(vd, wv.bfloat16().double())


@pytest.mark.parametrize("dtype,out", [("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (128, 128), (80, 40), (256, 64), (8, 2), (72, 6), (64, 0), (200, 200)])
def test_types_and_turns(ctx, d, rot, neighbours, dtype, out):
    check(ctx, [1, 130, 0, 7, 33], [5, 0, 9, 700, 129], 6, 2, d, rot, dtype=dtype, out=out, neighbours=neighbours)


@pytest.mark.parametrize("n", [1, 64, 500])
def test_single_tokens(ctx, n):
    check(ctx, [1] * n, [(i * 37) % 300 for i in range(n)], 8, 2, 128, 128, uniform=1)
    check(ctx, [1] * n, [(i * 37) % 300 for i in range(n)], 8, 2, 128, 128)


@pytest.mark.parametrize("pads", [(0, 0, 0, 0), (3, 5, 1, 7), (64, 32, 64, 8)])
@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_strides(ctx, layout, pads):
    check(ctx, [40, 3], [10, 100], pads=pads, layout=layout)
    check(ctx, [40, 3], [10, 100], pads=pads, layout=layout, dtype="bf16", offsets=[2, 42, 45])


def test_a_long_prompt(ctx):
    check(ctx, [3000], [0], 2, 1, 128, 128, page=64)
    check(ctx, [2500], [77], 2, 1, 64, 32, page=48, dtype="bf16", neighbours=True)


def test_far_positions(ctx):
    """Angles of a million turns: the table covers the positions, only the last pages exist."""
    past = 1 << 20
    check(ctx, [9], [past], 2, 1, 64, 64, page=1 << 16, base=10.0)
    check(ctx, [9], [past + 3], 2, 1, 64, 64, page=1 << 16, base=1e7, neighbours=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(ctx, dtype):
    check(ctx, [40, 3], [10, 100], dtype=dtype, out=dtype, in_place=True)
    check(ctx, [40, 3], [10, 100], d=80, rot=40, dtype=dtype, out=dtype, in_place=True, neighbours=True, pads=(5, 0, 0, 0))


def test_tokens_without_a_place(ctx):
    def pages(table, n):
        table[0, 1], table[1, 2] = -1, n
    check(ctx, [40, 60, 5], [0, 0, 3], table_change=pages)

    def lengths(length):
        length[0], length[1], length[2] = 10, -3, 4000
    check(ctx, [40, 60, 5], [0, 0, 3], length_change=lengths)


def test_no_queries(ctx):
    k = torch.randn(5, 2, 64, device="cuda")
    kc, vc = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    table, length = torch.tensor([[2]], dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    cache = sc.KvCache(kc.data_ptr(), vc.data_ptr(), table.data_ptr(), length.data_ptr(), 4, 16, 2, 64, 1)
    ctx.kv_append_dev(sc.KvAppend(1, 0, 0, seq_len=5), cache, 0, k.data_ptr(), k.data_ptr(), 0, stream())
    torch.cuda.synchronize()
    assert torch.equal(kc[2, :5], k.bfloat16()) and torch.equal(vc[2, :5], k.bfloat16())
    kc[2, :5] = 0
    assert not kc.any()


def test_nothing_to_do(ctx):
    kc = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    ints = torch.zeros(4, dtype=torch.int32, device="cuda")
    cache = sc.KvCache(kc[0].data_ptr(), kc[1].data_ptr(), ints.data_ptr(), ints.data_ptr(), 4, 16, 2, 64, 1)
    for how in (dict(seq_len=0), dict(offsets=[0, 0, 0]), dict(offsets=[9, 9, 9])):
        ctx.kv_append_dev(sc.KvAppend(2, 4, 64, **how), cache, 0, 0, 0, 0, stream())
    with pytest.raises(sc.BackendError):
        ctx.kv_append_dev(sc.KvAppend(2, 4, 64), cache, 0, 0, 0, 0, stream())
    torch.cuda.synchronize()
    assert not kc.any()
