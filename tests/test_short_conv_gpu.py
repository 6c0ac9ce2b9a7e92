"""The short causal convolution (strata_short_conv) against its definition in 64 bits.

Tolerance of an output, per element: the f32 sum of K products and the bias is off by at most
(K + 1) 2^-24 of the sum of their magnitudes m; SiLU's slope is at most 1.1, and its own exponential (2 ulp,
or 2 + 1.2 |z| ulp of 2^-23 in the approximate form that bf16 outputs take), addition and quick division (2 ulp)
add (6 + 1.2 |z|) 2^-23 of the result; a bf16 output rounds by 2^-8 of itself. States are copies: exact."""
import numpy as np
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

GUARD = 64  # elements around every output that must stay as they were


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def stream():
    return torch.cuda.current_stream().cuda_stream or 1


def guarded(n, dtype, shift=0):
    """A buffer with untouched margins; `shift` elements off 16-byte alignment."""
    whole = torch.full((n + 2 * GUARD + shift,), 7.0, dtype=dtype, device="cuda")
    return whole, whole[GUARD + shift: GUARD + shift + n]


def margins_kept(whole, n, shift=0):
    a = GUARD + shift
    return bool((whole[:a] == 7).all()) and bool((whole[a + n:] == 7).all())


def reference(x, w, b, state, offsets, silu):
    """f64: outputs of every row, new states, and the tolerance's magnitudes."""
    K = w.shape[1]
    y, mag, new = np.zeros(x.shape), np.zeros(x.shape), state.copy()
    for i, (a, e) in enumerate(zip(offsets, offsets[1:])):
        ext = np.concatenate([state[i], x[a:e]])
        for t in range(e - a):
            prod = ext[t:t + K] * w.T
            y[a + t], mag[a + t] = prod.sum(0) + b, np.abs(prod).sum(0) + np.abs(b)
        new[i] = ext[len(ext) - (K - 1):]
    z = y
    if silu:
        y = z / (1 + np.exp(-z))
    return y, new, mag, z


def run_case(ctx, lens, channels, taps, dtype, silu=True, bias=True, pad=(0, 0), shift=0, first=0, ragged=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    offsets = [first]
    for n in lens:
        offsets.append(offsets[-1] + n)
    rows = offsets[-1] + 3  # rows behind the last sequence
    dt = torch.bfloat16 if dtype == sc.BF16 else torch.float32
    xs, ys = channels + pad[0], channels + pad[1]
    xw, x = guarded(rows * xs, dt, shift)
    x.copy_(torch.randn(rows * xs, generator=g).to(dt))
    yw, y = guarded(rows * ys, dt, shift)
    y.fill_(7)
    w = torch.randn(channels, taps, generator=g) * 0.5
    b = torch.randn(channels, generator=g) if bias else torch.zeros(channels)
    st = torch.randn(len(lens), taps - 1, channels, generator=g).to(dt).float()
    wd, bd = w.cuda(), b.cuda()
    sw, sd = guarded(st.numel(), torch.float32, shift)
    sd.copy_(st.flatten())
    shape = sc.ShortConv(len(lens), channels, taps, seq_len=lens[0], offsets=offsets if ragged else None, dtype=dtype,
                         silu=silu, x_stride=xs, y_stride=ys)
    ctx.short_conv_dev(shape, x.data_ptr(), wd.data_ptr(), bd.data_ptr() if bias else 0, sd.data_ptr() if taps > 1 else 0,
                       y.data_ptr(), stream())
    torch.cuda.synchronize()
    xn = x.float().cpu().double().numpy().reshape(rows, xs)[:, :channels]
    want, new, mag, z = reference(xn, w.double().numpy(), b.double().numpy(), st.double().numpy(), offsets, silu)
    got = y.float().cpu().double().numpy().reshape(rows, ys)
    tol = 1.1 * (taps + 1) * 2.0 ** -24 * mag + (6 + 1.2 * np.abs(z)) * 2.0 ** -23 * np.abs(want) + 1e-37
    if dtype == sc.BF16:
        tol += 2.0 ** -8 * np.abs(want)
    inside = slice(offsets[0], offsets[-1])
    assert (np.abs(got[inside, :channels] - want[inside]) <= tol[inside]).all()
    if rows > offsets[-1]:
        assert (got[offsets[-1]:] == 7).all() and (got[:offsets[0]] == 7).all()
    assert (got[:, channels:] == 7).all()
    assert margins_kept(yw, rows * ys, shift) and margins_kept(sw, st.numel(), shift)
    assert np.array_equal(sd.cpu().double().numpy().reshape(st.shape), new)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 5, 6, 7, 8])
def test_every_number_of_taps(ctx, taps, dtype):
    run_case(ctx, [1, 0, 2, 3, 5, 7, 8, 15, 16, 17, 33, 70], 96, taps, dtype, seed=taps)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("channels", [1, 7, 8, 513, 1024, 2571])
def test_channel_counts(ctx, channels, dtype):
    run_case(ctx, [3, 40, 1], channels, 4, dtype, seed=channels)


@pytest.mark.parametrize("dtype", [sc.F32, sc.BF16])
@pytest.mark.parametrize("pad,shift", [((8, 16), 0), ((0, 0), 1), ((3, 5), 0), ((8, 8), 4)])
def test_strides_and_alignment(ctx, dtype, pad, shift):
    run_case(ctx, [5, 18, 2], 64, 4, dtype, pad=pad, shift=shift, first=2)


@pytest.mark.parametrize("silu,bias", [(False, False), (False, True), (True, False)])
def test_without_activation_or_bias(ctx, silu, bias):
    run_case(ctx, [21, 4], 40, 4, sc.F32, silu=silu, bias=bias)


def test_uniform_lengths_without_offsets(ctx):
    run_case(ctx, [1] * 300, 33, 4, sc.F32, ragged=False)
    run_case(ctx, [19] * 7, 128, 3, sc.BF16, ragged=False)


def test_more_sequences_than_one_launch_holds(ctx):
    run_case(ctx, [i % 4 for i in range(700)], 16, 4, sc.F32, seed=3)


def test_a_prompt_in_pieces_equals_the_whole(ctx):
    """Bit for bit: the state carries exactly what the next call needs."""
    c, n = 200, 61
    x, w = torch.randn(n, c, device="cuda"), torch.randn(c, 4, device="cuda")
    whole, s0 = torch.empty(n, c, device="cuda"), torch.randn(1, 3, c, device="cuda")
    s1 = s0.clone()
    ctx.short_conv_dev(sc.ShortConv(1, c, 4, seq_len=n), x.data_ptr(), w.data_ptr(), 0, s0.data_ptr(), whole.data_ptr(), stream())
    pieces, at = torch.empty(n, c, device="cuda"), 0
    for k in (1, 1, 2, 17, 1, 39):
        ctx.short_conv_dev(sc.ShortConv(1, c, 4, seq_len=k), x[at:].data_ptr(), w.data_ptr(), 0, s1.data_ptr(), pieces[at:].data_ptr(), stream())
        at += k
    torch.cuda.synchronize()
    assert at == n and torch.equal(whole, pieces) and torch.equal(s0, s1)


def test_all_sequences_empty_does_nothing(ctx):
    s = torch.randn(2, 3, 8, device="cuda")
    before = s.clone()
    y = torch.full((4, 8), 7.0, device="cuda")
    ctx.short_conv_dev(sc.ShortConv(2, 8, 4, offsets=[2, 2, 2]), y.data_ptr() + 4096, s.data_ptr() + 8192, 0, s.data_ptr(), y.data_ptr(), stream())
    torch.cuda.synchronize()
    assert torch.equal(s, before) and bool((y == 7).all())


def test_large_values_and_nan(ctx):
    """SiLU of far values is 0 or the value; a NaN stays in its channel and its taps."""
    x = torch.tensor([[1e30, -1e30, 100.0, -100.0, float("nan"), 0.0, 88.0, -88.0]], device="cuda").repeat(6, 1)
    x[1:, 4] = 1.0
    w = torch.zeros(8, 2, device="cuda")
    w[:, 0], w[:, 1] = 0.0, 1.0
    s, y = torch.zeros(1, 1, 8, device="cuda"), torch.empty(6, 8, device="cuda")
    ctx.short_conv_dev(sc.ShortConv(1, 8, 2, seq_len=6), x.data_ptr(), w.data_ptr(), 0, s.data_ptr(), y.data_ptr(), stream())
    torch.cuda.synchronize()
    y = y.cpu()
    assert y[3, 0] == np.float32(1e30) and y[3, 2] == 100 and abs(y[3, 1]) == 0 and abs(y[3, 3]) < 1e-40
    assert y[0, 4].isnan() and y[1, 4].isnan() and not y[2:, 4].isnan().any() and not y[:, :4].isnan().any()


def test_captured_and_replayed(ctx):
    c, w = 64, torch.randn(64, 4, device="cuda")
    x, y, s = torch.randn(2, c, device="cuda"), torch.empty(2, c, device="cuda"), torch.zeros(2, 3, c, device="cuda")
    shape = sc.ShortConv(2, c, 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.short_conv_dev(shape, x.data_ptr(), w.data_ptr(), 0, s.data_ptr(), y.data_ptr(), torch.cuda.current_stream().cuda_stream)
    inputs = [torch.randn(2, c, device="cuda") for _ in range(5)]
    for k in range(5):
        x.copy_(inputs[k])
        g.replay()
    torch.cuda.synchronize()
    ext = torch.stack(inputs[1:])  # the last four
    z = torch.einsum("kbc,ck->bc", ext.double(), w.double())
    assert (y - z / (1 + torch.exp(-z))).abs().max() < 1e-5
    assert torch.equal(s, torch.stack(inputs[2:], 1))


def test_refusals(ctx):
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()

    def call(code, xp=p, yp=p + 8192, sp=p + 4096, **over):
        with pytest.raises(sc.BackendError) as e:
            ctx.short_conv_dev(sc.ShortConv(**{**dict(n_seq=1, channels=16, taps=4, seq_len=2), **over}), xp, p + 2048, 0, sp, yp, stream())
        assert e.value.code == code and "short_conv" in str(e.value)

    call(sc.ERR_INVALID, xp=0)
    call(sc.ERR_INVALID, sp=0)
    call(sc.ERR_INVALID, yp=p)
    call(sc.ERR_INVALID, taps=9)
    call(sc.ERR_INVALID, channels=0)
    call(sc.ERR_INVALID, x_stride=8)
    call(sc.ERR_INVALID, offsets=[0, -3])
    call(sc.ERR_UNSUPPORTED_QUANT, dtype=sc.Q8_0)
