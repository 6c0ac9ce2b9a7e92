"""The sequence operators of a recurrent layer and of the token that follows it, as cases to be measured.

Three operators of the token step beside the quantized projections:

short_conv   the causal depthwise convolution (a few taps, SiLU) over the projected q | k | v channels, with
             the last taps - 1 inputs of every sequence as its state
gated_delta  the gated delta rule, a matrix state per value head: S <- exp(g) S + k (beta (v - exp(g) S^T k))^T,
             o = scale S^T q; one token per sequence when decoding, chunks of tokens when reading a prompt
sample       the next token of every row of logits: top-k, top-p, min-p, then temperature, from given
             random numbers

`own` False computes them with elementary torch operations, `own` True through strata_cuda.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one new token for each of 64 running sequences: the projected channels of 16 key heads and 32 value
        # heads of 128 (2 * 16 * 128 + 32 * 128 = 8192), 4 taps
        dict(name="conv decode 64", op="conv", lens=_even(64, 1), channels=8192, taps=4, dtype="f32", silu=True, bias=False),
        # a prompt of 8192 tokens read at once, activations in bf16
        dict(name="conv prompt 8192 bf16", op="conv", lens=_even(1, 8192), channels=8192, taps=4, dtype="bf16", silu=True, bias=False),
        # several prompts of odd lengths together, one of them empty, an odd channel count and a bias
        dict(name="conv ragged odd", op="conv", lens="513,1,0,2050,3,777,64,129", channels=2571, taps=4, dtype="f32", silu=True, bias=True),
        # one sequence answering: the latency of a single token
        dict(name="delta decode 1", op="delta", lens=_even(1, 1), hk=16, hv=32, dk=128, dv=128, dtype="f32", raw=True, norm=True, tiled=False),
        # 128 running sequences: the states (2 MiB a sequence) are the traffic
        dict(name="delta decode 128", op="delta", lens=_even(128, 1), hk=16, hv=32, dk=128, dv=128, dtype="f32", raw=True, norm=True, tiled=False),
        # a long prompt in one sequence
        dict(name="delta prompt 8192", op="delta", lens=_even(1, 8192), hk=16, hv=32, dk=128, dv=128, dtype="f32", raw=True, norm=True, tiled=False),
        # prompts of mixed lengths in one batch, activations in bf16
        dict(name="delta ragged bf16", op="delta", lens="1500,33,2049,700,1,1024,129,1600", hk=16, hv=32, dk=128, dv=128, dtype="bf16", raw=True, norm=True, tiled=False),
        # head sizes that fill no tile, value heads in tiled order, decay given as its logarithm
        dict(name="delta odd heads", op="delta", lens="257,5,0,600", hk=3, hv=9, dk=80, dv=52, dtype="f32", raw=False, norm=False, tiled=True),
        # one answer: every filter on, the vocabulary of the 2048 -> 151936 head
        dict(name="sample 1", op="sample", rows=1, vocab=151936, mode="mixed", masked=False),
        # a batch of requests, each with its own settings
        dict(name="sample 32 mixed", op="sample", rows=32, vocab=151936, mode="mixed", masked=False),
        # a large batch that shares its nucleus setting
        dict(name="sample 256 top-p", op="sample", rows=256, vocab=151936, mode="top_p", masked=False),
        # an odd vocabulary under grammar masks: most logits -inf, a row that leaves nothing, equal logits
        dict(name="sample 17 masked", op="sample", rows=17, vocab=32003, mode="mixed", masked=True),
    ]


def _even(n, length):
    return "%dx%d" % (n, length)


def _lens(text):
    if "x" in text:
        n, length = (int(v) for v in text.split("x"))
        return [length] * n
    return [int(v) for v in text.split(",")]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lens(rng, total):
    """One token for each of many sequences, one prompt, or several of mixed lengths: `total` tokens at most."""
    kind = rng.random()
    if kind < 0.35:
        return _even(_log(rng, 1, 128), 1)
    if kind < 0.6:
        return _even(1, _log(rng, 2, total))
    lens = []
    for _ in range(rng.randint(2, 9)):
        lens.append(rng.choice([0, 1, _log(rng, 2, max(2, total // 4)), _log(rng, 2, max(2, total // 4))]))
    lens.append(_log(rng, 1, max(1, total // 4)))
    while sum(lens) > total:
        lens[lens.index(max(lens))] //= 2
    return ",".join(str(v) for v in lens)


def draw(rng):
    op = rng.choice(["conv", "delta", "sample"])
    if op == "conv":
        return dict(op="conv", lens=_draw_lens(rng, 6000), channels=_log(rng, 96, 8192), taps=rng.choice([2, 3, 4, 4, 4]),
                    dtype=rng.choice(["f32", "bf16"]), silu=rng.random() < 0.8, bias=rng.random() < 0.5)
    if op == "delta":
        hk = _log(rng, 1, 16)
        usual = rng.random() < 0.5
        return dict(op="delta", lens=_draw_lens(rng, 5000), hk=hk, hv=hk * rng.choice([1, 2, 2]), dk=128 if usual else _log(rng, 16, 128),
                    dv=128 if usual else _log(rng, 16, 128), dtype=rng.choice(["f32", "bf16"]), raw=rng.random() < 0.7,
                    norm=rng.random() < 0.8, tiled=rng.random() < 0.3)
    return dict(op="sample", rows=_log(rng, 1, 200), vocab=_log(rng, 1000, 160000), mode=rng.choice(["mixed", "mixed", "top_k", "top_p", "min_p", "plain"]),
                masked=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "sample":
        return _prepare_sample(case, seed, normal, uniform)
    lens = _lens(case["lens"])
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    total, dt = offsets[-1], DTYPES[case["dtype"]]
    state = dict(case, offsets=offsets, total=total, n_seq=len(lens), seq_len=lens[0] if len(set(lens)) == 1 else -1, dt=dt)
    if case["op"] == "conv":
        c, k = case["channels"], case["taps"]
        state["x"] = normal(total, c).to(dt)
        state["w"] = normal(c, k) * 0.4
        state["b"] = normal(c) * 0.1 if case["bias"] else None
        state["s"] = normal(len(lens), k - 1, c).to(dt).float()  # what earlier calls left there
        return state
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    # q | k | v side by side, as the convolution leaves them
    qkv = normal(total, 2 * hk * dk + hv * dv)
    if not case["norm"]:
        qkv[:, : 2 * hk * dk] *= dk ** -0.5
    state["qkv"] = qkv.to(dt)
    if case["raw"]:
        # the gates as the projections give them, with the layer's decay rates (1 to 16) and time steps (0.001 to 0.1)
        state["gate"], state["beta"] = normal(total, hv), normal(total, hv)
        state["coef"] = -(1.0 + 15.0 * uniform(hv))
        step = torch.exp(uniform(hv) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        state["shift"] = torch.log(torch.expm1(step))
    else:
        state["gate"], state["beta"] = -0.2 * uniform(total, hv), uniform(total, hv)
        state["coef"] = state["shift"] = None
    state["s"] = normal(len(lens), hv, dk, dv) * 0.1
    return state


def _prepare_sample(case, seed, normal, uniform):
    rows, vocab, mode = case["rows"], case["vocab"], case["mode"]
    logits = normal(rows, vocab) * 2.5
    # a few tokens stand out, as they do after a trained head
    at = (uniform(rows, 12) * vocab).long().clamp_(max=vocab - 1)
    logits.scatter_(1, at, 8.0 + 5.0 * uniform(rows, 12))
    rng = random.Random(seed)
    temp, top_k, top_p, min_p = [], [], [], []
    for r in range(rows):
        m = mode if mode != "mixed" else ("all", "top_k", "top_p", "min_p", "plain", "greedy")[r % 6]
        temp.append(0.0 if m == "greedy" else rng.choice([0.6, 0.8, 1.0, 1.3]))
        top_k.append(rng.choice([20, 40, 200, 1000]) if m in ("all", "top_k") else 0)
        top_p.append(rng.choice([0.8, 0.9, 0.95]) if m in ("all", "top_p") else 1.0)
        min_p.append(rng.choice([0.02, 0.05, 0.1]) if m in ("all", "min_p") else 0.0)
    if case["masked"]:
        allowed = uniform(rows, vocab) < 0.01
        for r in range(rows):
            if r % 4 == 1:
                logits[r] = torch.where(allowed[r], logits[r], torch.full_like(logits[r], -math.inf))
            elif r % 4 == 2:
                logits[r] = torch.round(logits[r] * 2) / 2  # many equal values
            elif r == 3:
                logits[r] = -math.inf
    dev = dict(device="cuda")
    return dict(case, logits=logits, temperature=torch.tensor(temp, dtype=torch.float32, **dev), top_k=torch.tensor(top_k, dtype=torch.int32, **dev),
                top_p=torch.tensor(top_p, dtype=torch.float32, **dev), min_p=torch.tensor(min_p, dtype=torch.float32, **dev),
                u=torch.tensor([rng.random() for _ in range(rows)], dtype=torch.float64, **dev))


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return {"conv": _conv_own, "delta": _delta_own, "sample": _sample_own}[state["op"]](state)
    return {"conv": _conv_plain, "delta": _delta_plain, "sample": _sample_plain}[state["op"]](state)


def _padded(state):
    """[sequence, position] -> row of the packed tokens, and where there is a token."""
    off = torch.tensor(state["offsets"], device="cuda")
    lens = off[1:] - off[:-1]
    pos = torch.arange(max(b - a for a, b in zip(state["offsets"], state["offsets"][1:])), device="cuda")
    there = pos[None, :] < lens[:, None]
    return torch.where(there, off[:-1, None] + pos[None, :], 0), there, lens


def _conv_plain(s):
    at, there, lens = _padded(s)
    k = s["taps"]
    x = torch.cat([s["s"], s["x"].float()[at] * there[..., None]], 1)  # the state's rows before each sequence
    n = at.shape[1]
    y = sum(x[:, j:j + n] * s["w"][:, j] for j in range(k))
    if s["b"] is not None:
        y = y + s["b"]
    if s["silu"]:
        y = y / (1 + torch.exp(-y))
    last = lens[:, None] + torch.arange(k - 1, device="cuda")[None, :]
    s["s"].copy_(torch.gather(x, 1, last[..., None].expand(-1, -1, x.shape[2])))
    return {"y": y[there].to(s["dt"]), "state": s["s"]}


def _delta_inputs(s):
    hk, hv, dk, dv = s["hk"], s["hv"], s["dk"], s["dv"]
    return s["qkv"][:, : hk * dk].unflatten(1, (hk, dk)), s["qkv"][:, hk * dk: 2 * hk * dk].unflatten(1, (hk, dk)), s["qkv"][:, 2 * hk * dk:].unflatten(1, (hv, dv))


def _delta_plain(s):
    at, there, _ = _padded(s)
    q, k, v = (x.float() for x in _delta_inputs(s))
    if s["norm"]:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q = q * s["dk"] ** -0.5
    r = s["hv"] // s["hk"]
    q, k = (x.repeat(1, r, 1) if s["tiled"] else x.repeat_interleave(r, 1) for x in (q, k))
    g, beta = s["gate"], s["beta"]
    if s["raw"]:
        g = s["coef"] * torch.logaddexp(g + s["shift"], torch.zeros((), device="cuda"))
        beta = 1 / (1 + torch.exp(-beta))
    # [sequence, head, position, ...], a whole number of chunks of 64 (of one token when decoding): what is no token has k, beta and g of zero
    c = min(64, 1 << (at.shape[1] - 1).bit_length())
    pad = -at.shape[1] % c
    at, m = torch.nn.functional.pad(at, (0, pad)), torch.nn.functional.pad(there, (0, pad))
    q, k, v = ((x[at] * m[..., None, None]).transpose(1, 2).unflatten(2, (-1, c)) for x in (q, k, v))
    g, beta = ((x[at] * m[..., None]).transpose(1, 2).unflatten(2, (-1, c)) for x in (g, beta))
    gs = torch.cumsum(g.double(), -1)
    low = torch.ones(c, c, device="cuda").tril()
    decay = torch.exp(torch.where(low > 0, gs[..., :, None] - gs[..., None, :], 0.0)).float() * low
    a = beta[..., None] * decay * (k @ k.transpose(-1, -2)) * low.tril(-1)
    eye = torch.eye(c, device="cuda")
    t, p = eye - a, a @ a
    for _ in range(5):  # (I + a)^-1 = (I - a)(I + a^2)(I + a^4) ...: a^64 = 0
        t, p = t + t @ p, p @ p
    qk = (q @ k.transpose(-1, -2)) * decay
    up, total = torch.exp(gs).float()[..., None], torch.exp(gs[..., -1]).float()[..., None, None]
    down = torch.exp(gs[..., -1:] - gs).float()[..., None]
    u0, w0 = t @ (beta[..., None] * v), t @ (beta[..., None] * up * k)
    state, out = s["s"], []
    for i in range(q.shape[2]):
        u = u0[:, :, i] - w0[:, :, i] @ state
        out.append((up[:, :, i] * q[:, :, i]) @ state + qk[:, :, i] @ u)
        state = total[:, :, i] * state + (down[:, :, i] * k[:, :, i]).transpose(-1, -2) @ u
    s["s"].copy_(state)
    o = torch.stack(out, 2).flatten(2, 3).transpose(1, 2)[:, : there.shape[1]]
    return {"o": o[there].to(s["dt"]), "state": s["s"]}


def _sample_plain(s):
    x = s["logits"].double()
    v = x.shape[1]
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(1, keepdim=True)
    d = torch.where(x == top, 0.0, x - top)
    e = torch.where(x == -math.inf, 0.0, torch.exp(d))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    es, pos = e.gather(1, order), torch.arange(v, device="cuda")[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], v)[:, None]
    keep = (pos < k) & (x.gather(1, order) > -math.inf)
    es = es * keep
    before = torch.cumsum(es, 1) - es
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (before < p * es.sum(1, keepdim=True)) | (pos == 0)
    keep &= (es >= s["min_p"].double()[:, None]) | (pos == 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    t = s["temperature"].double()[:, None]
    w = torch.where(kept & (e > 0), torch.exp(d / torch.where(t > 0, t, 1.0)), 0.0)
    cum = torch.cumsum(w, 1)
    z = cum[:, -1:]
    pick = torch.searchsorted(cum, s["u"][:, None] * z, right=True)[:, 0].clamp(max=v - 1)
    greedy = s["temperature"] <= 0
    pick = torch.where(greedy, order[:, 0], pick)
    logp = torch.where(greedy, 0.0, torch.log(w.gather(1, pick[:, None]) / z)[:, 0])
    none = top[:, 0] == -math.inf
    return {"ids": torch.where(none, -1, pick).int(), "logprobs": torch.where(none, -math.inf, logp).float()}


# ---------------------------------------------------------------- the framework's calls

_context = []


def _ctx():
    if not _context:
        if str(ROOT / "strata-rs_b200") not in sys.path:
            sys.path.insert(0, str(ROOT / "strata-rs_b200"))
        import strata_cuda
        _context.extend([strata_cuda, strata_cuda.Context(torch.cuda.current_device())])
    return _context


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1  # 1: CUDA's handle of the default stream


def _lengths(s):
    return dict(seq_len=s["seq_len"]) if s["seq_len"] >= 0 else dict(offsets=s["offsets"])


def _conv_own(s):
    sc, ctx = _ctx()
    if "desc" not in s:
        s["desc"] = sc.ShortConv(n_seq=s["n_seq"], channels=s["channels"], taps=s["taps"], silu=s["silu"],
                                 dtype=sc.BF16 if s["dtype"] == "bf16" else sc.F32, **_lengths(s))
    y = torch.empty(s["total"], s["channels"], dtype=s["dt"], device="cuda")
    ctx.short_conv_dev(s["desc"], s["x"].data_ptr(), s["w"].data_ptr(), s["b"].data_ptr() if s["b"] is not None else 0,
                       s["s"].data_ptr(), y.data_ptr(), stream=_stream())
    return {"y": y, "state": s["s"]}


def _delta_own(s):
    sc, ctx = _ctx()
    if "desc" not in s:
        width = s["qkv"].shape[1]
        s["desc"] = sc.GatedDelta(n_seq=s["n_seq"], n_k_head=s["hk"], n_v_head=s["hv"], k_dim=s["dk"], v_dim=s["dv"],
                                  dtype=sc.BF16 if s["dtype"] == "bf16" else sc.F32, q_stride=width, k_stride=width, v_stride=width,
                                  tiled=s["tiled"], raw_gates=s["raw"], scale=s["dk"] ** -0.5, l2_eps=1e-6 if s["norm"] else -1.0, **_lengths(s))
        s["work"] = torch.empty(max(16, sc.gated_delta_work_bytes(s["desc"])), dtype=torch.uint8, device="cuda")
    q, k, v = _delta_inputs(s)
    o = torch.empty(s["total"], s["hv"], s["dv"], dtype=s["dt"], device="cuda")
    ctx.gated_delta_dev(s["desc"], q.data_ptr(), k.data_ptr(), v.data_ptr(), s["gate"].data_ptr(), s["beta"].data_ptr(),
                        s["coef"].data_ptr() if s["raw"] else 0, s["shift"].data_ptr() if s["raw"] else 0, s["s"].data_ptr(), o.data_ptr(),
                        s["work"].data_ptr(), s["work"].numel(), stream=_stream())
    return {"o": o, "state": s["s"]}


def _sample_own(s):
    _, ctx = _ctx()
    rows, vocab = s["logits"].shape
    ids = torch.empty(rows, dtype=torch.int32, device="cuda")
    logprobs = torch.empty(rows, dtype=torch.float32, device="cuda")
    ctx.sample_dev(s["logits"].data_ptr(), rows, vocab, s["u"].data_ptr(), ids.data_ptr(), logprobs_ptr=logprobs.data_ptr(),
                   temperature_ptr=s["temperature"].data_ptr(), top_k_ptr=s["top_k"].data_ptr(), top_p_ptr=s["top_p"].data_ptr(),
                   min_p_ptr=s["min_p"].data_ptr(), stream=_stream())
    return {"ids": ids, "logprobs": logprobs}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # every logit once; a maximum and an exponential's worth of products for each
        return {"bytes": rows * (vocab * 4 + 32), "flops": rows * vocab * 12}
    lens = _lens(case["lens"])
    total, size = sum(lens), 2 if case["dtype"] == "bf16" else 4
    live = sum(n > 0 for n in lens)
    if case["op"] == "conv":
        c, k = case["channels"], case["taps"]
        return {"bytes": total * c * 2 * size + c * k * 4 + live * (k - 1) * c * 8 + (c * 4 if case["bias"] else 0), "flops": total * c * (2 * k + 4)}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    # q, k, v and o once, the gates, the state read and written; S^T k, S^T q and the rank-1 update a token
    return {"bytes": total * ((2 * hk * dk + 2 * hv * dv) * size + hv * 8) + live * hv * dk * dv * 8, "flops": total * hv * dk * dv * 6}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _conv_exact, "delta": _delta_exact, "sample": _sample_exact}[case["op"]](s)


def _conv_exact(s):
    """Sequence by sequence, the state's rows in front of the inputs."""
    k, ys, states = s["taps"], [], []
    for i, (a, b) in enumerate(zip(s["offsets"], s["offsets"][1:])):
        x = torch.cat([s["s"][i].double(), s["x"][a:b].double()])
        y = torch.einsum("tck,ck->tc", x.unfold(0, k, 1), s["w"].double()) if b > a else x[:0]
        y = y + (s["b"].double() if s["b"] is not None else 0)
        ys.append(y * torch.sigmoid(y) if s["silu"] else y)
        states.append(x[x.shape[0] - (k - 1):])
    return {"y": torch.cat(ys), "state": torch.stack(states)}


def _delta_exact(s):
    """Token by token over all sequences at once; where a sequence has ended its state stays."""
    q, k, v = (x.double() for x in _delta_inputs(s))
    if s["norm"]:
        q, k = (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    head = torch.arange(s["hv"], device="cuda")
    head = head % s["hk"] if s["tiled"] else head // (s["hv"] // s["hk"])
    g, beta = s["gate"].double(), s["beta"].double()
    if s["raw"]:
        g = s["coef"].double() * torch.nn.functional.softplus(g + s["shift"].double(), threshold=200.0)
        beta = torch.sigmoid(beta)
    off = torch.tensor(s["offsets"], device="cuda")
    state, o = s["s"].double(), torch.zeros(s["total"], s["hv"], s["dv"], dtype=torch.float64, device="cuda")
    lens = [b - a for a, b in zip(s["offsets"], s["offsets"][1:])]
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    sorted_state = state[order].contiguous()
    starts = off[:-1][torch.tensor(order, device="cuda")]
    for t in range(max(lens)):
        n = sum(x > t for x in lens)
        rows, live = starts[:n] + t, sorted_state[:n]
        kt, qt = k[rows][:, head], q[rows][:, head]
        live *= torch.exp(g[rows])[..., None, None]
        err = beta[rows][..., None] * (v[rows] - torch.einsum("nhij,nhi->nhj", live, kt))
        live += kt[..., :, None] * err[..., None, :]
        o[rows] = torch.einsum("nhij,nhi->nhj", live, qt) * s["dk"] ** -0.5
    state[order] = sorted_state
    return {"o": o, "state": state}


def _sample_exact(s):
    """Row by row: the candidates in falling order, cut by each filter in turn."""
    ids, logps = [], []
    for r in range(s["rows"]):
        x = s["logits"][r].double()
        cand = torch.argsort(-x, stable=True)
        cand = cand[: int((x > -math.inf).sum())]
        if not len(cand):
            ids.append(-1), logps.append(-math.inf)
            continue
        temp, k, p, m = float(s["temperature"][r]), int(s["top_k"][r]), float(s["top_p"][r]), float(s["min_p"][r])
        if temp <= 0:
            ids.append(int(cand[0])), logps.append(0.0)
            continue
        cand = cand[:k] if k > 0 else cand
        prob = torch.softmax(x[cand], 0)
        if p < 1:
            prob = prob[: int((torch.cumsum(prob, 0) < p).sum()) + 1]
        cand = cand[: max(1, int((prob >= m * prob[0]).sum()))].sort().values
        weight = torch.softmax(x[cand] / temp, 0)
        at = min(int((torch.cumsum(weight, 0) <= float(s["u"][r])).sum()), len(cand) - 1)
        ids.append(int(cand[at])), logps.append(math.log(float(weight[at])))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "logprobs": torch.tensor(logps, dtype=torch.float64)}
