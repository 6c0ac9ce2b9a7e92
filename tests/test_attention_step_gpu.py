"""The attention operators as a model uses them: a prompt read in chunks and scored, then token after token, each step one
projection to q | k | v, the append to the cache, attention over it, the output projection, the head, the scored tokens and
the draw. Every stage is compared with its formula in 64 bits on what the stage before gave, with the tolerances that the
stages' own tests derive (the products': relative to the largest output, 1e-3 for the GEMV, 1e-2 for the GEMM)."""
import math

import numpy as np
import pytest

import strata_cuda as sc
import test_logprobs_gpu as lp
from synth import Q4_K, quant_matrix
from test_kv_append_gpu import turned

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EMBD, HQ, HKV, D, VOCAB, PAGE = 256, 8, 2, 64, 1003, 16
QKV = (HQ + 2 * HKV) * D
BASE, ROT, SCALE = 1e6, 32, D ** -0.5


class Layer:
    """One layer and its cache: sequences of up to 256 tokens, the queries handed from append to attention in `mid`."""

    def __init__(self, ctx, n_seq, mid, window):
        g = torch.Generator().manual_seed(n_seq)
        rand = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
        self.ctx, self.n, self.mid, self.window = ctx, n_seq, mid, window
        self.data = {}
        for i, (name, rows, cols) in enumerate((("in", QKV, EMBD), ("out", EMBD, HQ * D), ("head", VOCAB, EMBD))):
            q = quant_matrix(90 + i, Q4_K, rows, cols)
            w = ctx.upload(q, Q4_K, rows, cols)
            self.data[name] = (w, torch.from_numpy(ctx.dequant(w).reshape(rows, cols).astype(np.float64)).cuda())
        self.embed = rand(VOCAB, EMBD) * 0.05
        width = 256 // PAGE
        self.table = torch.randperm(n_seq * width + 3, generator=g)[: n_seq * width].int().reshape(n_seq, width).cuda()
        self.len = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.k, self.v = (torch.full((n_seq * width + 3, PAGE, HKV, D), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.cache = sc.KvCache(self.k.data_ptr(), self.v.data_ptr(), self.table.data_ptr(), self.len.data_ptr(), n_pages=len(self.k), page_size=PAGE,
                                n_kv_head=HKV, head_dim=D, max_pages=width)

    def buffers(self, lens):
        off = [0] + [int(v) for v in np.cumsum(lens)]
        rows = off[-1]
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        dt = torch.bfloat16 if self.mid == sc.BF16 else torch.float32
        b = dict(off=off, x=f(rows, EMBD), qkv=f(rows, QKV), q=torch.zeros(rows, HQ, D, dtype=dt, device="cuda"), o=torch.zeros(rows, HQ * D, dtype=dt, device="cuda"),
                 of=f(rows, HQ * D), y=f(rows, EMBD), logits=f(rows, VOCAB), lp=f(rows), ent=f(rows), ids=torch.zeros(rows, 3, dtype=torch.int32, device="cuda"),
                 tops=f(rows, 3), t=torch.full((rows,), 1e6, device="cuda"), next=torch.zeros(rows, dtype=torch.int32, device="cuda"), u=torch.zeros(rows, dtype=torch.float64, device="cuda"),
                 grow=torch.tensor(lens, dtype=torch.int32, device="cuda"))
        b["append"] = sc.KvAppend(self.n, HQ, ROT, BASE, offsets=off, q_dtype=self.mid, q_stride=QKV, k_stride=QKV, v_stride=QKV)
        b["att"] = sc.Attention(self.n, HQ, SCALE, offsets=off, dtype=self.mid, window=self.window, sinks=2 if self.window else 0)
        b["work"] = torch.zeros(sc.attention_work_bytes(b["att"], self.cache), dtype=torch.uint8, device="cuda")
        return b

    def step(self, b, tokens, targets):
        c, s, rows = self.ctx, torch.cuda.current_stream().cuda_stream or 1, b["x"].shape[0]

        def product(name, x, y):
            (c.gemv_dev if rows <= 8 else c.gemm_f32_dev)(self.data[name][0], x.data_ptr(), y.data_ptr(), rows, s)

        self.len.add_(b["grow"])
        torch.index_select(self.embed, 0, tokens, out=b["x"])
        product("in", b["x"], b["qkv"])
        p = b["qkv"].data_ptr()
        c.kv_append_dev(b["append"], self.cache, p, p + HQ * D * 4, p + (HQ + HKV) * D * 4, b["q"].data_ptr(), s)
        c.attention_dev(b["att"], self.cache, b["q"].data_ptr(), b["o"].data_ptr(), b["work"].data_ptr(), b["work"].numel(), s)
        b["of"].copy_(b["o"])
        product("out", b["of"], b["y"])
        product("head", b["y"], b["logits"])
        c.logprobs_dev(b["logits"].data_ptr(), rows, VOCAB, targets.data_ptr(), b["lp"].data_ptr(), b["ent"].data_ptr(), 3, b["ids"].data_ptr(), b["tops"].data_ptr(), stream=s)
        c.sample_dev(b["logits"].data_ptr(), rows, VOCAB, b["u"].data_ptr(), b["next"].data_ptr(), temperature_ptr=b["t"].data_ptr(), stream=s)

    def check(self, b, targets):
        torch.cuda.synchronize()
        rows = b["x"].shape[0]

        def close(got, want, tol, what):
            assert ((got.double() - want).abs() <= tol).all(), what

        def product(name, x, y):
            want = b[x].double() @ self.data[name][1].T
            close(b[y], want, (1e-3 if rows <= 8 else 1e-2) * want.abs().max(), name)

        product("in", "x", "qkv")
        half = 2.0 ** -8
        for i, (a, e) in enumerate(zip(b["off"], b["off"][1:])):
            n, m = e - a, int(self.len[i])
            pos = torch.arange(m - n, m, device="cuda")
            q, tq = turned(b["qkv"][a:e, : HQ * D].double().unflatten(1, (HQ, D)), pos, ROT, BASE, False)
            k, tk = turned(b["qkv"][a:e, HQ * D: (HQ + HKV) * D].double().unflatten(1, (HKV, D)), pos, ROT, BASE, False)
            close(b["q"][a:e], q, tq * 1.01 + (half if self.mid == sc.BF16 else 2.0 ** -24) * q.abs(), "q")
            at = self.table[i].long()[pos // PAGE], pos % PAGE
            close(self.k[at], k, tk * 1.01 + half * k.abs(), "k")
            assert torch.equal(self.v[at], b["qkv"][a:e, (HQ + HKV) * D:].unflatten(1, (HKV, D)).bfloat16())
            j = torch.arange(m, device="cuda")
            at = self.table[i].long()[j // PAGE], j % PAGE
            seen = j <= pos[:, None]
            if self.window:
                seen &= (j > pos[:, None] - self.window) | (j < 2)
            for h in range(HKV):
                kh, vh, qh = self.k[at][:, h].double(), self.v[at][:, h].double(), b["q"][a:e, h * 4:(h + 1) * 4].double()
                w = torch.softmax(torch.where(seen[:, None], qh @ kh.T * SCALE, -math.inf), -1)
                big = (qh.abs() @ kh.abs().T * SCALE * seen[:, None]).amax(-1, keepdim=True)
                off = 2 * (big * (D / 16 + 8) + 1.45 * big + 1) * 2.0 ** -23 + 2.0 ** -22
                want = w @ vh
                tol = (2 * off + (m / 16 + 32) * 2.0 ** -23) * (w @ vh.abs()) + 2.0 ** -24 * want.abs()
                if self.mid == sc.BF16:
                    tol += half * (w @ vh.abs() + want.abs())
                close(b["o"][a:e].unflatten(1, (HQ, D))[:, h * 4:(h + 1) * 4], want, tol, "o")
        product("out", "of", "y")
        product("head", "y", "logits")
        host = b["logits"].cpu().numpy()
        for r in range(rows):
            first, ent, order, lps, tl, th = lp.expected(host[r].copy(), int(targets[r]), 3)
            ulp = 2.0 ** -24
            assert abs(float(b["lp"][r]) - first) <= tl + ulp * abs(first) and abs(float(b["ent"][r]) - ent) <= th + ulp * abs(ent)
            assert b["ids"][r].tolist() == order.tolist()
            assert np.abs(b["tops"][r].cpu().numpy() - lps).max() <= tl + ulp * np.abs(lps).max()


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("mid", [sc.F32, sc.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lens,window", [([100], 0), ([37, 1, 70], 0), ([37, 1, 70], 20), ([5], 3)], ids=str)
def test_a_prompt_in_chunks_and_the_tokens_after_it(ctx, lens, window, mid):
    n = len(lens)
    layer = Layer(ctx, n, mid, window)
    rng = np.random.default_rng(sum(lens))
    second = [max(1, v // 3) for v in lens]
    for chunk in (lens, second, [1] * n, [1] * n, [1] * n):
        b = layer.buffers(chunk)
        tokens, targets = (torch.from_numpy(rng.integers(0, VOCAB, sum(chunk))).cuda() for _ in range(2))
        b["u"].copy_(torch.from_numpy(rng.random(sum(chunk))))
        layer.step(b, tokens, targets.int())
        layer.check(b, targets)


def test_one_chunk_or_several_give_the_same(ctx):
    """A prompt read whole and the same prompt read in pieces: the last token's attention, and its log-probabilities."""
    rng = np.random.default_rng(4)
    tokens = torch.from_numpy(rng.integers(0, VOCAB, 120)).cuda()
    outs = []
    for pieces in ([120], [64, 56], [100, 19, 1]):
        layer, at = Layer(ctx, 1, sc.F32, 0), 0
        for n in pieces:
            b = layer.buffers([n])
            part = tokens[at:at + n]
            layer.step(b, part, part.int())
            at += n
        torch.cuda.synchronize()
        outs.append((b["o"][-1].double(), b["lp"][-1].double()))
    for o, p in outs[1:]:
        # q, k and v come from the GEMM where a piece has more than 8 tokens and from the GEMV else: 1e-2 of the largest at most
        assert (o - outs[0][0]).abs().max() <= 0.05 * outs[0][0].abs().max()


def test_one_chunk_or_several_give_the_same_log_probabilities(ctx):
    """The last token's log-probability after a prompt read whole and in pieces. With |.| element by element and the products'
    own tolerances (1e-2 of the largest output at most, on either side): y differs by |W_out| |do| + 2e-2 max |y|, the logits x by
    |W_head| |dy| + 2e-2 max |x|, and a log-probability by |dx| of its token and the largest |dx| (the logarithm of a mean of
    exponentials moves by no more than they do), besides what each may be off from its own logits."""
    rng = np.random.default_rng(5)
    tokens = torch.from_numpy(rng.integers(0, VOCAB, 120)).cuda()
    outs = []
    for pieces in ([120], [64, 56], [100, 19, 1]):
        layer, at = Layer(ctx, 1, sc.F32, 0), 0
        for n in pieces:
            b = layer.buffers([n])
            part = tokens[at:at + n]
            layer.step(b, part, part.int())
            at += n
        torch.cuda.synchronize()
        outs.append({x: b[x][-1].double() for x in ("o", "y", "logits", "lp")})
    out, head, target, first = layer.data["out"][1].abs(), layer.data["head"][1].abs(), int(tokens[-1]), outs[0]

    def own(x):  # how far log p may be off from the logits it was computed from
        lp0, _, _, _, tl, _ = lp.expected(x["logits"].float().cpu().numpy(), target, 0)
        assert abs(float(x["lp"]) - lp0) <= tl + 2.0 ** -24 * abs(lp0)
        return tl + 2.0 ** -24 * abs(lp0)

    for x in outs[1:]:
        dy = out @ (x["o"] - first["o"]).abs() + 2e-2 * torch.maximum(x["y"].abs().max(), first["y"].abs().max())
        assert ((x["y"] - first["y"]).abs() <= dy).all()
        dx = head @ (x["y"] - first["y"]).abs() + 2e-2 * torch.maximum(x["logits"].abs().max(), first["logits"].abs().max())
        moved = (x["logits"] - first["logits"]).abs()
        assert (moved <= dx).all()
        assert abs(float(x["lp"] - first["lp"])) <= float(moved[target] + moved.max()) + own(x) + own(first)


@pytest.mark.parametrize("mid", [sc.F32, sc.BF16], ids=["f32", "bf16"])
def test_a_captured_step_gives_what_the_calls_give(ctx, mid):
    """Ten tokens of three sequences, each the last one's draw, by calls and by a captured graph that grows the lengths: the same bits."""
    layer = Layer(ctx, 3, mid, 6)
    b = layer.buffers([1, 1, 1])
    start = torch.tensor([1, 500, 1002], device="cuda")
    tokens, targets = start.clone(), torch.tensor([7, 8, 9], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    us = torch.rand(10, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).cuda()

    def run(advance):
        tokens.copy_(start)
        layer.len.zero_()
        layer.k.fill_(math.nan), layer.v.fill_(math.nan)
        seen = []
        for u in us:
            b["u"].copy_(u)
            advance()
            seen += [b[x].clone() for x in ("next", "o", "lp", "ent", "ids", "tops")]
        return seen + [torch.nan_to_num(layer.k), torch.nan_to_num(layer.v), layer.len.clone()]

    def step():
        layer.step(b, tokens, targets)
        tokens.copy_(b["next"])

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        eager = run(step)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        replayed = run(graph.replay)
        again = run(step)
    torch.cuda.synchronize()
    assert all(torch.equal(a, r) and torch.equal(a, e) for a, r, e in zip(eager, replayed, again))
    assert len({int(i) for i in torch.cat(eager[0:60:6])}) > 5  # the draws do differ
