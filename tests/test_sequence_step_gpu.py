"""The sequence operators as a model uses them: a prompt, then token after token, each step one projection, the short
convolution, the gated delta rule on columns of its output, a norm per head, the output projection, the head and the draw.

Every stage is compared with its formula in 64 bits on what the stage before gave. The products keep the library's own
bounds relative to the largest output (1e-3 for the GEMV, 1e-2 for the prompt's GEMM); the convolution and the delta rule
keep the tolerances that their own tests derive, a norm of n elements (n/2 + 4) 2^-24, and ids are equal."""
import numpy as np
import pytest

import strata_cuda as sc
from synth import Q4_K, quant_matrix
from test_sample_gpu import expected

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EMBD, HK, HV, D, TAPS, VOCAB = 256, 2, 4, 64, 4, 1003
QKV, PROJ = 2 * HK * D + HV * D, 2 * HK * D + HV * D + 2 * HV  # q, k, v, then the raw gates


class Layer:
    def __init__(self, ctx, n_seq):
        g = torch.Generator().manual_seed(n_seq)
        rand = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
        self.ctx, self.n = ctx, n_seq
        self.data = {}
        for i, (name, rows) in enumerate((("in", PROJ), ("out", EMBD), ("head", VOCAB))):
            q = quant_matrix(70 + i, Q4_K, rows, EMBD)
            w = ctx.upload(q, Q4_K, rows, EMBD)
            self.data[name] = (w, ctx.dequant(w).reshape(rows, EMBD).astype(np.float64))
        self.embed, self.cw, self.cb = rand(VOCAB, EMBD) * 0.05, rand(QKV, TAPS) * 0.5, rand(QKV)
        self.coef, self.shift, self.norm = -(0.05 + torch.rand(HV, generator=g)).cuda(), rand(HV), rand(D)
        self.fnorm = torch.full((EMBD,), 0.02, device="cuda")
        self.conv_state, self.state = torch.zeros(n_seq, TAPS - 1, QKV, device="cuda"), torch.zeros(n_seq, HV, D, D, device="cuda")
        self.temperature, self.top_p = torch.full((n_seq,), 0.8, device="cuda"), torch.full((n_seq,), 0.9, device="cuda")
        self.top_k = torch.tensor(([40, 0, 5] * n_seq)[:n_seq], dtype=torch.int32, device="cuda")

    def buffers(self, rows, offsets):
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        b = dict(x=f(rows, EMBD), proj=f(rows, PROJ), conv=f(rows, QKV), o=f(rows, HV * D), normed=f(rows, HV * D), y=f(rows, EMBD),
                 last=f(self.n, EMBD), logits=f(self.n, VOCAB), u=torch.zeros(self.n, dtype=torch.float64, device="cuda"),
                 ids=torch.zeros(self.n, dtype=torch.int32, device="cuda"), lps=f(self.n))
        b["tail"] = torch.tensor([e - 1 for e in offsets[1:]], device="cuda")
        b["offsets"] = offsets
        b["cs"] = sc.ShortConv(self.n, QKV, TAPS, offsets=offsets, x_stride=PROJ)
        b["ds"] = sc.GatedDelta(self.n, HK, HV, D, D, offsets=offsets, l2_eps=1e-6, raw_gates=True,
                                q_stride=QKV, k_stride=QKV, v_stride=QKV, gate_stride=PROJ, beta_stride=PROJ)
        b["work"] = torch.zeros(sc.gated_delta_work_bytes(b["ds"]) + 16, dtype=torch.uint8, device="cuda")
        return b

    def step(self, b, tokens):
        """tokens: int64 on the device, a row each."""
        c, s, rows = self.ctx, torch.cuda.current_stream().cuda_stream or 1, b["x"].shape[0]

        def product(name, x, y):
            (c.gemv_dev if x.shape[0] <= 8 else c.gemm_f32_dev)(self.data[name][0], x.data_ptr(), y.data_ptr(), x.shape[0], s)

        torch.index_select(self.embed, 0, tokens, out=b["x"])
        product("in", b["x"], b["proj"])
        p = b["proj"].data_ptr()
        c.short_conv_dev(b["cs"], p, self.cw.data_ptr(), self.cb.data_ptr(), self.conv_state.data_ptr(), b["conv"].data_ptr(), s)
        q = b["conv"].data_ptr()
        c.gated_delta_dev(b["ds"], q, q + HK * D * 4, q + 2 * HK * D * 4, p + QKV * 4, p + (QKV + HV) * 4, self.coef.data_ptr(), self.shift.data_ptr(),
                          self.state.data_ptr(), b["o"].data_ptr(), b["work"].data_ptr(), b["work"].numel(), s)
        b["normed"].copy_(b["o"])
        c.rms_norm_dev(b["normed"].data_ptr(), self.norm.data_ptr(), D, rows * HV, 1e-6, s)
        product("out", b["normed"], b["y"])
        torch.index_select(b["y"], 0, b["tail"], out=b["last"])
        c.rms_norm_dev(b["last"].data_ptr(), self.fnorm.data_ptr(), EMBD, self.n, 1e-6, s)
        product("head", b["last"], b["logits"])
        c.sample_dev(b["logits"].data_ptr(), self.n, VOCAB, b["u"].data_ptr(), b["ids"].data_ptr(), b["lps"].data_ptr(),
                     temperature_ptr=self.temperature.data_ptr(), top_k_ptr=self.top_k.data_ptr(), top_p_ptr=self.top_p.data_ptr(), stream=s)

    def check(self, b, conv0, state0):
        """The step just made against its formulas; conv0, state0: the states before it."""
        torch.cuda.synchronize()
        n = {k: v.cpu().double().numpy() for k, v in b.items() if isinstance(v, torch.Tensor)}

        def close(got, want, tol, what):
            assert np.abs(got - want).max() <= tol * np.abs(want).max(), what

        def product(name, x, y):
            close(n[y], n[x] @ self.data[name][1].T, 1e-3 if len(n[x]) <= 8 else 1e-2, name)

        def rms(x, w):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w.cpu().double().numpy()

        product("in", "x", "proj")
        w, bias = self.cw.cpu().double().numpy(), self.cb.cpu().double().numpy()
        o = np.empty_like(n["o"])
        for i, (a, e) in enumerate(zip(b["offsets"], b["offsets"][1:])):
            ext = np.concatenate([conv0[i].cpu().double().numpy(), n["proj"][a:e, :QKV]])
            prods = np.stack([ext[t:t + TAPS] * w.T for t in range(e - a)])
            z, mag = prods.sum(1) + bias, np.abs(prods).sum(1) + np.abs(bias)
            want = z / (1 + np.exp(-z))
            tol = 1.1 * (TAPS + 1) * 2.0 ** -24 * mag + (6 + 1.2 * np.abs(z)) * 2.0 ** -23 * np.abs(want) + 1e-37
            assert (np.abs(n["conv"][a:e] - want) <= tol).all()
            assert np.array_equal(self.conv_state[i].cpu().double().numpy(), ext[len(ext) - (TAPS - 1):])
            S = state0[i].cpu().double().numpy().copy()
            for t in range(a, e):
                q, k = (n["conv"][t, j * HK * D:(j + 1) * HK * D].reshape(HK, D) for j in (0, 1))
                q, k = (np.repeat(v / np.sqrt((v * v).sum(-1, keepdims=True) + 1e-6), HV // HK, 0) for v in (q, k))
                v = n["conv"][t, 2 * HK * D:].reshape(HV, D)
                gate, beta = n["proj"][t, QKV:QKV + HV], n["proj"][t, QKV + HV:]
                S *= np.exp(self.coef.cpu().double().numpy() * np.logaddexp(gate + self.shift.cpu().double().numpy(), 0))[:, None, None]
                S += k[:, :, None] * ((v - np.einsum("hij,hi->hj", S, k)) / (1 + np.exp(-beta))[:, None])[:, None]
                o[t] = (np.einsum("hij,hi->hj", S, q) * D ** -0.5).reshape(-1)
            spread = 8 * 2.0 ** -24 * np.sqrt(D * min(e - a, 256))
            close(n["o"][a:e], o[a:e], spread, "o")
            close(self.state[i].cpu().double().numpy(), S, spread, "state")
        close(n["normed"], rms(n["o"].reshape(-1, HV, D), self.norm).reshape(n["o"].shape), (D / 2 + 4) * 2.0 ** -24, "norm")
        product("out", "normed", "y")
        close(n["last"], rms(n["y"][b["tail"].cpu().numpy()], self.fnorm), (EMBD / 2 + 4) * 2.0 ** -24, "last norm")
        product("head", "last", "logits")
        for i in range(self.n):
            t, p = float(self.temperature[i]), float(self.top_p[i])
            want, lp = expected(b["logits"][i].cpu().numpy().copy(), t, int(self.top_k[i]), p, 0.0, float(b["u"][i]))
            assert int(b["ids"][i]) == want and abs(float(b["lps"][i]) - lp) <= 2.0 ** -23 * abs(lp) + 1e-9


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("lens", [[100], [5], [37, 1, 70], [3, 2]])
def test_a_prompt_and_the_tokens_after_it(ctx, lens):
    n = len(lens)
    layer = Layer(ctx, n)
    rng = np.random.default_rng(sum(lens))
    prompt = layer.buffers(sum(lens), [0] + [int(v) for v in np.cumsum(lens)])
    tokens = torch.from_numpy(rng.integers(0, VOCAB, sum(lens))).cuda()
    single = layer.buffers(n, list(range(n + 1)))
    for i in range(7):
        b = prompt if i == 0 else single
        b["u"].copy_(torch.from_numpy(rng.random(n)))
        before = layer.conv_state.clone(), layer.state.clone()
        layer.step(b, tokens)
        layer.check(b, *before)
        tokens = b["ids"].long()


def test_a_captured_step_gives_what_the_calls_give(ctx):
    """Ten tokens of three sequences, each the last one's draw, by calls and by a captured graph: the same bits."""
    layer = Layer(ctx, 3)
    b = layer.buffers(3, [0, 1, 2, 3])
    tokens = torch.tensor([1, 500, 1002], device="cuda")
    start = tokens.clone()
    side = torch.cuda.Stream()
    us = torch.rand(10, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).cuda()

    def run(advance):
        tokens.copy_(start)
        layer.conv_state.zero_(), layer.state.zero_()
        seen = []
        for u in us:
            b["u"].copy_(u)
            advance()
            seen += [b["ids"].clone(), b["lps"].clone(), b["logits"].clone()]
        return seen + [layer.conv_state.clone(), layer.state.clone()]

    def step():
        layer.step(b, tokens)
        tokens.copy_(b["ids"])

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
    assert len({int(i) for i in torch.cat(eager[0:30:3])}) > 5  # the draws do differ
