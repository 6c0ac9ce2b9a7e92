"""The gated delta rule over inputs whose sizes differ from token to token: growing states, outliers, keys of any norm.

Every output and every column of the state is compared on its own scale, made of what can have reached it: earlier tokens,
the same head, the same column. For column j of head h after token t,
  d_t = |S'| + |k| |u| + beta |k|^2 |S'| + beta |k| |v| + |S_t|,  S' = e^g S_{t-1}, 2-norms of columns,
is what the roundings of token t are relative to: products over k_dim carry 22 bits of the norms of their vectors (f16
limb pairs; 24 where sums are plain f32), everything else f32's 24. Where beta |k|^2 <= 2 the step is a contraction, so an
error of an earlier token is worth e^{g} of itself a token later. The roundings are independent, so that a column's error
has a spread of 2^-22 D_t at most with D_t^2 = (e^g D_{t-1})^2 + d_t^2, and an output's one of 2^-22 scale |q| D_t; eight
spreads cover the largest of the elements compared. A bf16 output rounds by 2^-8 of itself."""
import numpy as np
import pytest

import strata_cuda as sc
from test_gated_delta_gpu import Case, stream

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


def columns(x):
    return np.sqrt((x * x).sum(-2))


def reference(c):
    """f64: outputs and states with their tolerances, and the largest output of each token and head."""
    q, k, v = (x.cpu().double().reshape(c.rows, -1, d).numpy() for x, d in zip(c.parts(), (c.dk, c.dk, c.dv)))
    if c.norm:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-6) for x in (q, k))
    head = np.arange(c.hv) // (c.hv // c.hk)
    g, b = c.gate.cpu().double().numpy()[:, :c.hv], c.beta.cpu().double().numpy()[:, :c.hv]
    S = c.state0.double().numpy().copy()
    o, tol = np.zeros((c.rows, c.hv, c.dv)), np.zeros((c.rows, c.hv, c.dv))
    stol = np.zeros((len(c.lens), c.hv, c.dv))
    eps = 8 * 2.0 ** -22
    for i, (a, e) in enumerate(zip(c.off, c.off[1:])):
        D = np.zeros((c.hv, c.dv))
        for t in range(a, e):
            kt, qt, decay, beta = k[t, head], q[t, head], np.exp(g[t])[:, None], b[t][:, None]
            nk, nq = (np.sqrt((x * x).sum(-1))[:, None] for x in (kt, qt))
            assert (beta * nk * nk <= 2 * (1 + 1e-9)).all()
            S[i] *= decay[..., None]
            before = columns(S[i])
            u = beta * (v[t] - np.einsum("hij,hi->hj", S[i], kt))
            S[i] += kt[:, :, None] * u[:, None, :]
            d = before * (1 + beta * nk * nk) + nk * (np.abs(u) + beta * np.abs(v[t])) + columns(S[i])
            D = np.sqrt((decay * D) ** 2 + d ** 2)
            o[t] = c.scale * np.einsum("hij,hi->hj", S[i], qt)
            tol[t] = eps * c.scale * nq * D + (2.0 ** -8 * np.abs(o[t]) if c.dtype == sc.BF16 else 0)
        stol[i] = eps * D
    return o, tol, S, stol


def compare(c):
    torch.cuda.synchronize()
    o, tol, S, stol = reference(c)
    got = c.o.float().cpu().double().numpy()[:, :c.hv * c.dv].reshape(o.shape)
    for t in range(c.off[0], c.off[-1]):
        bad = ~(np.abs(got[t] - o[t]) <= tol[t] + 1e-37)
        assert not bad.any(), f"token {t}: {bad.sum()} outputs, off by {np.abs(got[t] - o[t]).max():.3g}, largest {np.abs(o[t]).max():.3g}"
    err = np.abs(c.state.cpu().double().numpy() - S).max(-2)
    assert (err <= stol + 1e-37).all(), f"state off by {(err / stol).max():.3g} tolerances"


def check(ctx, c):
    """In one call, and in calls of 15 tokens, which are read token by token."""
    c.run(ctx)
    compare(c)
    if len(c.lens) > 1:
        return
    c.state.copy_(c.state0)
    c.o.fill_(7)
    q, k, v = c.parts()
    size, fsize = c.qkv.element_size(), 4
    for a in range(c.off[0], c.off[-1], 15):
        part = sc.GatedDelta(1, c.hk, c.hv, c.dk, c.dv, seq_len=min(15, c.off[-1] - a), dtype=c.dtype, l2_eps=1e-6 if c.norm else -1.0,
                             q_stride=c.width, k_stride=c.width, v_stride=c.width, o_stride=c.os, gate_stride=c.gs, beta_stride=c.gs)
        assert sc.gated_delta_work_bytes(part) == 0
        ctx.gated_delta_dev(part, *(x.data_ptr() + a * c.width * size for x in (q, k, v)), *(x.data_ptr() + a * c.gs * fsize for x in (c.gate, c.beta)),
                            0, 0, c.state.data_ptr(), c.o.data_ptr() + a * c.os * size, 0, 0, stream())
    compare(c)


DTYPES = pytest.mark.parametrize("dtype", [sc.F32, sc.BF16], ids=["f32", "bf16"])


@DTYPES
@pytest.mark.parametrize("g,length", [(0.05, 15), (0.05, 200), (0.3, 64), (0.3, 200), (0.5, 150), (1.0, 64), (2.0, 15), (2.0, 40)])
def test_growing_states(ctx, g, length, dtype):
    """Gates above zero, as far as f32 holds what they grow (e^80)."""
    c = Case([length], dk=128, dv=64, dtype=dtype, seed=length)
    c.gate.fill_(g)
    check(ctx, c)


@DTYPES
@pytest.mark.parametrize("power", [20, 30, 40, 60])
@pytest.mark.parametrize("at", [31, 20, 63, 16])
def test_one_value_far_above_the_others(ctx, at, power, dtype):
    """What comes later costs earlier tokens nothing, nor does a column its neighbours."""
    c = Case([70], dk=64, dv=64, dtype=dtype, seed=at)
    c.parts()[2][at] *= 2.0 ** power
    check(ctx, c)
    c = Case([40, 1, 70], dk=128, dv=128, hk=1, hv=2, dtype=dtype, seed=at)
    c.parts()[2][at, 5::17] *= 2.0 ** power
    check(ctx, c)


@DTYPES
@pytest.mark.parametrize("power", [-60, -30, 30, 60])
def test_values_that_rise_and_fall_within_a_chunk(ctx, power, dtype):
    """From 1 to 2^power over 32 tokens, with decays that forget about as fast."""
    c = Case([96], dk=64, dv=48, dtype=dtype)
    steps = torch.arange(c.rows) % 32 * (power / 31)
    c.parts()[2].mul_((2.0 ** steps)[:, None].cuda())
    check(ctx, c)
    c.state.copy_(c.state0)
    c.gate.fill_(-abs(power) / 31 * 0.7)
    check(ctx, c)


@DTYPES
@pytest.mark.parametrize("power", [-40, -12, 12, 40, 62])
def test_normalised_keys_of_any_norm(ctx, power, dtype):
    """The norm of a key passes 2^power, its square stays within f32, and the update does not depend on either."""
    c = Case([50, 16], dk=128, dv=64, dtype=dtype, seed=power)
    q, k, _ = c.parts()
    for x, p in ((k, power), (q, -abs(power) // 4)):
        x.copy_((x.float() / x.float().reshape(c.rows, c.hk, c.dk).norm(dim=-1).repeat_interleave(c.dk, 1) * 2.0 ** p).to(c.dt))
    check(ctx, c)


@DTYPES
@pytest.mark.parametrize("power", [10, 25, 40])
def test_one_key_far_above_the_others(ctx, power, dtype):
    """Keys as they are, one of them long, with a step short enough for it."""
    c = Case([70], dk=64, dv=64, dtype=dtype, norm=False, seed=power)
    _, k, _ = c.parts()
    k[25] *= 2.0 ** power
    c.beta[25] *= 2.0 ** (-2 * power)
    check(ctx, c)


@DTYPES
@pytest.mark.parametrize("g", [-3.0, -0.5, 0.7, 2.7])
def test_one_token_seen_from_every_later_one(ctx, g, dtype):
    """o_t = scale e^{t g} beta (q_t . k_0) v_0 where nothing else is learnt: the decay of up to 31 tokens as one factor.
    Its own error is a few roundings (2^-21 in all, 2^-24 |g| a token where tokens multiply theirs); q . k carries 22 bits
    and a limb's 2^-40, f32 sums of 128 products another 2^-21 of the norms. Below f32's normal numbers (2^-126) that is absolute."""
    c = Case([32], hk=1, hv=1, dk=128, dv=32, dtype=dtype, norm=False)
    c.state0.zero_()
    c.state.zero_()
    q, k, v = c.parts()
    q.copy_(k[0:1].expand_as(q))
    v[1:] = 0
    c.beta[1:] = 0
    c.gate.fill_(g)
    c.run(ctx)
    torch.cuda.synchronize()
    q, k, v = (x.cpu().double().numpy() for x in (q, k, v))
    b, gate = float(c.beta[0, 0]), float(c.gate[0, 0])
    want = c.scale * np.exp(gate * np.arange(32))[:, None] * b * (k[0] @ k[0]) * v[0]
    got = c.o[:32, :32].float().cpu().double().numpy()
    rel = 2.0 ** -21 + 2.0 ** -21 + (2.0 ** -8 if dtype == sc.BF16 else 0)
    assert (np.abs(got - want) <= rel * np.abs(want) + 1e-37).all(), float((np.abs(got - want) / np.abs(want)).max())
