"""The gated delta rule (strata_gated_delta) against its recurrence in 64 bits.

Tolerance: a state or output element is a sum of k_dim products over a state that at most T updates made; each
f32 operation is off by at most half a step (2^-24 of its result), and the update is a contraction for the inputs
used here (decay <= 1, |k| <= 1, beta in [0, 1]), so earlier errors do not grow. The roundings are independent, so
their sum has a spread of 2^-24 sqrt(k_dim min(T, 256)) of the largest magnitudes (256 tokens back the decays leave
nothing); eight spreads cover the largest of the elements compared. A bf16 output rounds by 2^-8 of itself."""
import numpy as np
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

GUARD = 64


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


class Case:
    """Inputs of one call, its buffers on the device, and the recurrence in 64 bits."""

    def __init__(self, lens, hk=2, hv=4, dk=64, dv=64, dtype=sc.F32, raw=False, norm=True, tiled=False, first=0,
                 ragged=True, shift=0, gap=0, seed=0, shifted=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hk, self.hv, self.dk, self.dv, self.dtype = lens, hk, hv, dk, dv, dtype
        self.raw, self.norm, self.tiled, self.ragged = raw, norm, tiled, ragged
        self.off = [first]
        for n in lens:
            self.off.append(self.off[-1] + n)
        self.rows = self.off[-1] + 2
        self.dt = torch.bfloat16 if dtype == sc.BF16 else torch.float32
        self.width = 2 * hk * dk + hv * dv + gap
        qkv = torch.randn(self.rows, self.width, generator=g)
        if not norm:
            qkv[:, :2 * hk * dk] *= 0.8 / max(1.0, np.sqrt(dk) * 1.3)
        self.buf = torch.zeros(shift + qkv.numel(), dtype=self.dt, device="cuda")
        self.qkv = self.buf[shift:].view(self.rows, self.width)
        self.qkv.copy_(qkv.to(self.dt))
        if raw:
            self.gate, self.beta = (torch.randn(self.rows, hv + gap, generator=g).cuda() for _ in range(2))
            self.coef = -(0.1 + 2 * torch.rand(hv, generator=g)).cuda()
            self.bias = torch.randn(hv, generator=g).cuda() if shifted else None
        else:
            self.gate = -torch.rand(self.rows, hv + gap, generator=g).cuda() * 0.3
            self.beta = torch.rand(self.rows, hv + gap, generator=g).cuda()
            self.coef = self.bias = None
        self.gs = hv + gap
        self.state0 = torch.randn(len(lens), hv, dk, dv, generator=g) * 0.3
        self.swhole = torch.full((shift + self.state0.numel() + GUARD,), 7.0, device="cuda")
        self.state = self.swhole[shift: shift + self.state0.numel()].view(self.state0.shape)
        self.state.copy_(self.state0)
        self.os = hv * dv + gap
        self.owhole = torch.full((shift + self.rows * self.os + GUARD,), 7.0, dtype=self.dt, device="cuda")
        self.o = self.owhole[shift: shift + self.rows * self.os].view(self.rows, self.os)
        self.scale = dk ** -0.5
        self.shape = sc.GatedDelta(len(lens), hk, hv, dk, dv, seq_len=lens[0], offsets=self.off if ragged else None,
                                   dtype=dtype, l2_eps=1e-6 if norm else -1.0, tiled=tiled, raw_gates=raw,
                                   q_stride=self.width, k_stride=self.width, v_stride=self.width, o_stride=self.os,
                                   gate_stride=self.gs, beta_stride=self.gs)
        self.work = torch.full((sc.gated_delta_work_bytes(self.shape) + 256,), 0xFF, dtype=torch.uint8, device="cuda")

    def parts(self):
        a, b = self.hk * self.dk, 2 * self.hk * self.dk
        return self.qkv[:, :a], self.qkv[:, a:b], self.qkv[:, b:b + self.hv * self.dv]

    def run(self, ctx, s=None):
        q, k, v = self.parts()
        need = self.work.numel() - 256
        ctx.gated_delta_dev(self.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), self.gate.data_ptr(),
                            self.beta.data_ptr(), self.coef.data_ptr() if self.raw else 0,
                            self.bias.data_ptr() if self.bias is not None else 0, self.state.data_ptr(),
                            self.o.data_ptr(), self.work.data_ptr() if need else 0, need, s or stream())

    def reference(self):
        q, k, v = (x.cpu().double().reshape(self.rows, -1, d).numpy() for x, d in zip(self.parts(), (self.dk, self.dk, self.dv)))
        if self.norm:
            q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (q, k))
        h = np.arange(self.hv)
        h = h % self.hk if self.tiled else h // (self.hv // self.hk)
        g, b = self.gate.cpu().double().numpy()[:, :self.hv], self.beta.cpu().double().numpy()[:, :self.hv]
        if self.raw:
            z = g + (self.bias.cpu().double().numpy() if self.bias is not None else 0)
            g, b = self.coef.cpu().double().numpy() * np.logaddexp(z, 0), 1 / (1 + np.exp(-b))
        o = np.full((self.rows, self.hv, self.dv), 7.0)
        S = self.state0.double().numpy().copy()
        for i, (a, e) in enumerate(zip(self.off, self.off[1:])):
            for t in range(a, e):
                S[i] *= np.exp(g[t])[:, None, None]
                u = b[t][:, None] * (v[t] - np.einsum("hij,hi->hj", S[i], k[t, h]))
                S[i] += k[t, h][:, :, None] * u[:, None, :]
                o[t] = self.scale * np.einsum("hij,hi->hj", S[i], q[t, h])
        return o, S

    def check(self):
        torch.cuda.synchronize()
        want, S = self.reference()
        got = self.o.float().cpu().double().numpy()
        inside = slice(self.off[0], self.off[-1])
        spread = 8 * 2.0 ** -24 * np.sqrt(self.dk * min(max(self.lens + [1]), 256))
        if self.off[-1] > self.off[0]:
            w = want[inside].reshape(-1, self.hv * self.dv)
            tol = spread * max(np.abs(w).max(), 1e-30) + (2.0 ** -8 * np.abs(w) if self.dtype == sc.BF16 else 0)
            err = np.abs(got[inside, :self.hv * self.dv] - w)
            assert (err <= tol).all(), f"o off by {err.max():.3g} (largest {np.abs(w).max():.3g})"
        err = np.abs(self.state.cpu().double().numpy() - S)
        assert err.max() <= spread * max(np.abs(S).max(), 1e-30), f"state off by {err.max():.3g} (largest {np.abs(S).max():.3g})"
        for i, n in enumerate(self.lens):
            if n == 0:
                assert torch.equal(self.state[i].cpu(), self.state0[i])
        assert (got[:self.off[0]] == 7).all() and (got[self.off[-1]:] == 7).all() and (got[:, self.hv * self.dv:] == 7).all()
        assert bool((self.owhole[-GUARD:] == 7).all()) and bool((self.swhole[-GUARD:] == 7).all())
        assert bool((self.work[-256:] == 0xFF).all())


def check(ctx, *a, **kw):
    c = Case(*a, **kw)
    c.run(ctx)
    c.check()


DIMS = [(128, 128), (64, 64), (1, 1), (5, 3), (33, 40), (80, 52), (128, 36), (96, 160), (32, 256), (200, 72), (256, 130)]


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("dk,dv", DIMS)
def test_one_token_each(ctx, dk, dv, dtype):
    check(ctx, [1] * 5, dk=dk, dv=dv, dtype=dtype, ragged=False, seed=dk)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("dk,dv", DIMS)
def test_ragged_lengths(ctx, dk, dv, dtype):
    check(ctx, [1, 0, 2, 31, 32, 33, 64, 65, 0, 130], dk=dk, dv=dv, dtype=dtype, first=3, seed=dv)


@pytest.mark.parametrize("raw", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tiled", [False, True])
def test_gates_norms_and_head_orders(ctx, raw, norm, tiled):
    check(ctx, [1, 40, 300, 7], hk=3, hv=6, dk=48, dv=40, raw=raw, norm=norm, tiled=tiled)


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 8), (5, 5), (2, 6)])
def test_head_counts(ctx, hk, hv):
    check(ctx, [70, 1, 3], hk=hk, hv=hv, dk=32, dv=24, raw=True, shifted=False)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("shift,gap", [(1, 0), (2, 4), (0, 3), (4, 8), (0, 16)])
def test_strides_and_alignment(ctx, dtype, shift, gap):
    check(ctx, [2, 37, 100], dk=64, dv=128, dtype=dtype, shift=shift, gap=gap)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
def test_a_long_prompt(ctx, dtype):
    check(ctx, [1500], hk=1, hv=2, dk=128, dv=128, raw=True, dtype=dtype)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("n,length,dk,dv", [(1, 16, 64, 64), (3, 17, 128, 36), (2, 32, 80, 52), (5, 40, 128, 128), (20, 33, 128, 130), (9, 64, 33, 40), (250, 35, 16, 24)])
def test_uniform_lengths_without_offsets(ctx, n, length, dk, dv, dtype):
    check(ctx, [length] * n, hk=1, hv=2, dk=dk, dv=dv, dtype=dtype, ragged=False, seed=length)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
def test_many_sequences_in_chunks(ctx, dtype):
    check(ctx, [33 + i % 40 for i in range(230)], hk=2, hv=4, dk=64, dv=100, dtype=dtype)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
def test_single_tokens_beside_prompts(ctx, dtype):
    """Many short sequences in a call with long ones are read token by token, the others in chunks."""
    check(ctx, [1, 0, 3, 15] * 12 + [70, 0, 16, 33, 14], dk=64, dv=64, dtype=dtype, first=2)
    check(ctx, [200] + [1] * 40 + [0] + [17], hk=2, hv=4, dk=128, dv=36, raw=True, dtype=dtype, gap=3)
    check(ctx, [1 + (i % 9 == 0) * 40 for i in range(600)], hk=1, hv=2, dk=16, dv=8, dtype=dtype)


@pytest.mark.parametrize("lens,ragged", [([10500], False), ([4900, 4900], False), ([5200, 0, 33, 4700, 1], True)])
def test_prompts_beyond_one_filling_of_the_workspace(ctx, lens, ragged):
    """What is computed ahead of the scan is bounded, so that the longest calls run in pieces."""
    hk, hv, d = 16, 32, 128
    g = torch.Generator(device="cuda").manual_seed(sum(lens))
    rows, size = sum(lens), 2 * hk * d + hv * d
    qkv = torch.randn(rows, size, generator=g, device="cuda")
    gate, beta = -torch.rand(rows, hv, generator=g, device="cuda") * 0.2, torch.rand(rows, hv, generator=g, device="cuda")
    state0 = torch.randn(len(lens), hv, d, d, generator=g, device="cuda") * 0.3
    state, o = state0.clone(), torch.empty(rows, hv * d, device="cuda")
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    shape = sc.GatedDelta(len(lens), hk, hv, d, d, seq_len=lens[0], offsets=off if ragged else None, l2_eps=1e-6, q_stride=size, k_stride=size, v_stride=size)
    need = sc.gated_delta_work_bytes(shape)
    assert need <= 257 << 20
    work = torch.full((need + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    p = qkv.data_ptr()
    ctx.gated_delta_dev(shape, p, p + hk * d * 4, p + 2 * hk * d * 4, gate.data_ptr(), beta.data_ptr(), 0, 0, state.data_ptr(), o.data_ptr(), work.data_ptr(), need, stream())
    spread = 8 * 2.0 ** -24 * np.sqrt(d * 256)
    q, k, v = (x.reshape(rows, -1, d) for x in qkv.double().split([hk * d, hk * d, hv * d], 1))
    q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    q, k = (x.repeat_interleave(hv // hk, 1) for x in (q * d ** -0.5, k))
    decay, beta = gate.double().exp(), beta.double()
    want = torch.empty(rows, hv, d, dtype=torch.float64, device="cuda")
    for i, (a, e) in enumerate(zip(off, off[1:])):
        S = state0[i].double()
        for t in range(a, e):
            S *= decay[t, :, None, None]
            u = beta[t, :, None] * (v[t] - torch.bmm(k[t, :, None], S)[:, 0])
            S.baddbmm_(k[t, :, :, None], u[:, None])
            want[t] = torch.bmm(q[t, :, None], S)[:, 0]
        assert float((state[i].double() - S).abs().max()) <= spread * float(S.abs().max())
    assert float((o.view(rows, hv, d).double() - want).abs().max()) <= spread * float(want.abs().max())
    assert bool((work[need:] == 0xFF).all())


def test_more_sequences_than_one_launch_holds(ctx):
    check(ctx, [(i * 7) % 5 for i in range(600)], hk=1, hv=2, dk=16, dv=8)
    check(ctx, [40 * (i % 3 == 0) for i in range(300)], hk=1, hv=1, dk=32, dv=16)


def test_many_sequences_of_one_token(ctx):
    check(ctx, [1] * 1000, hk=1, hv=1, dk=16, dv=20, ragged=False)


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128)])
def test_a_prompt_in_pieces_equals_the_whole(ctx, dk, dv):
    """The state carries a sequence from call to call, whichever way each call is read."""
    c = Case([200], dk=dk, dv=dv, raw=True)
    q, k, v = c.parts()
    at, size = 0, 4
    for n in (1, 1, 64, 5, 100, 1, 28):
        part = sc.GatedDelta(1, c.hk, c.hv, dk, dv, seq_len=n, l2_eps=1e-6, raw_gates=True, q_stride=c.width, k_stride=c.width, v_stride=c.width)
        work = torch.empty(sc.gated_delta_work_bytes(part) + 16, dtype=torch.uint8, device="cuda")
        ctx.gated_delta_dev(part, q.data_ptr() + at * c.width * size, k.data_ptr() + at * c.width * size, v.data_ptr() + at * c.width * size,
                            c.gate.data_ptr() + at * c.gs * size, c.beta.data_ptr() + at * c.gs * size, c.coef.data_ptr(), c.bias.data_ptr(),
                            c.state.data_ptr(), c.o.data_ptr() + at * c.os * size, work.data_ptr(), work.numel(), stream())
        torch.cuda.synchronize()
        at += n
    assert at == 200
    c.check()


@pytest.mark.parametrize("length", [1, 20, 150])
def test_decay_that_forgets_everything(ctx, length):
    """g = -inf, or far below what exp resolves, empties the state; nothing turns into NaN."""
    c = Case([length], dk=64, dv=32)
    c.gate[::3] = -float("inf")
    c.gate[1::3] = -1e30
    c.gate[2::3] = -200.0
    c.run(ctx)
    c.check()


def test_beta_of_zero_leaves_the_decayed_state(ctx):
    c = Case([90], dk=64, dv=64)
    c.beta.zero_()
    c.gate.zero_()
    c.run(ctx)
    torch.cuda.synchronize()
    assert torch.equal(c.state.cpu(), c.state0)


def test_zero_keys_with_norm(ctx):
    """k = 0 and q = 0 normalise to 0 and write nothing."""
    c = Case([70], dk=64, dv=64)
    q, k, _ = c.parts()
    q[::2] = 0
    k[::2] = 0
    c.run(ctx)
    c.check()


@pytest.mark.parametrize("power", [-30, -12, 12, 30])
def test_scales_of_values_and_states(ctx, power):
    """Values and states of any magnitude keep their relative precision."""
    c = Case([150], dk=64, dv=64, raw=True)
    c.parts()[2].mul_(2.0 ** power)
    c.state0 *= 2.0 ** power
    c.state.copy_(c.state0)
    c.run(ctx)
    c.check()


def test_columns_of_different_scale(ctx):
    """Columns of the state are independent problems: a large one costs its neighbours nothing."""
    c = Case([140], hk=1, hv=1, dk=64, dv=64, raw=True)
    sizes = 2.0 ** (torch.arange(64) % 16 * 2.0 - 16)
    c.parts()[2].mul_(sizes.cuda())
    c.state0 *= sizes
    c.state.copy_(c.state0)
    c.run(ctx)
    torch.cuda.synchronize()
    o, S = c.reference()
    spread = 8 * 2.0 ** -24 * np.sqrt(64 * 140)
    got = c.o.cpu().double().numpy()[:140, :64]
    for j in range(64):
        assert np.abs(got[:, j] - o[:140, 0, j]).max() <= spread * np.abs(o[:140, 0, j]).max()
        assert np.abs(c.state.cpu().double().numpy()[0, 0, :, j] - S[0, 0, :, j]).max() <= spread * np.abs(S[0, 0, :, j]).max()


def test_nan_stays_in_its_sequence_and_head(ctx):
    c = Case([50, 100, 60], hk=2, hv=2, dk=64, dv=64)
    c.parts()[2][50 + 70, :64] = float("nan")  # sequence 1, token 70, head 0
    c.run(ctx)
    torch.cuda.synchronize()
    o = c.o[:210, :128].cpu()
    assert not o[:50].isnan().any() and not o[150:].isnan().any() and not o[:, 64:].isnan().any()
    assert o[120:150, :64].isnan().all()
    assert not o[50:50 + 64, :64].isnan().any()  # no chunk reaches further back than 32 tokens from its end


def test_repeated_calls_give_the_same_bits(ctx):
    c = Case([33, 400, 1], dk=128, dv=128, raw=True)
    c.run(ctx)
    torch.cuda.synchronize()
    o, s = c.o.clone(), c.state.clone()
    for _ in range(3):
        c.state.copy_(c.state0)
        c.run(ctx)
        torch.cuda.synchronize()
        assert torch.equal(c.o, o) and torch.equal(c.state, s)


def test_two_streams_at_once(ctx):
    cases = [Case([700, 33], dk=128, dv=128, raw=True, seed=i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                c.state.copy_(c.state0.cuda())
                c.run(ctx, s.cuda_stream)
    for c in cases:
        c.check()


@pytest.mark.parametrize("length", [1, 200])
def test_captured_and_replayed(ctx, length):
    c = Case([length] * 2, dk=64, dv=64, raw=True, ragged=length != 1)
    saved = c.state0.cuda()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.state.copy_(saved)
        c.run(ctx, torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        c.o.fill_(7)
        c.state.fill_(9)
        g.replay()
        c.check()


def test_refusals(ctx):
    c = Case([200], dk=64, dv=64, raw=True)
    q, k, v = (x.data_ptr() for x in c.parts())

    def call(code, shape=None, q=q, coef=c.coef.data_ptr(), state=c.state.data_ptr(), o=c.o.data_ptr(), work=c.work.data_ptr(), have=c.work.numel()):
        with pytest.raises(sc.BackendError) as e:
            ctx.gated_delta_dev(shape or c.shape, q, k, v, c.gate.data_ptr(), c.beta.data_ptr(), coef, 0, state, o, work, have, stream())
        assert e.value.code == code and "gated_delta" in str(e.value)

    call(sc.ERR_INVALID, q=0)
    call(sc.ERR_INVALID, coef=0)
    call(sc.ERR_INVALID, o=c.state.data_ptr())
    call(sc.ERR_INVALID, o=v)
    call(sc.ERR_INVALID, state=c.qkv.data_ptr())
    call(sc.ERR_INVALID, shape=sc.GatedDelta(1, 2, 4, 300, 64, seq_len=2))
    call(sc.ERR_INVALID, shape=sc.GatedDelta(1, 3, 4, 64, 64, seq_len=2))
    call(sc.ERR_UNSUPPORTED_QUANT, shape=sc.GatedDelta(1, 2, 4, 64, 64, seq_len=2, dtype=sc.F16))
    if sc.gated_delta_work_bytes(c.shape):
        call(sc.ERR_SCRATCH_LIMIT, work=0)
        call(sc.ERR_SCRATCH_LIMIT, have=sc.gated_delta_work_bytes(c.shape) - 1)
