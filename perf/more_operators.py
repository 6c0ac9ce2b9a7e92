"""The attention of a layer that keeps a cache, and the scoring of tokens, as cases to be measured.

Three operators of the token step beside the quantized projections:

append       a call's new keys and values into a paged cache, bf16, with the position rotation of the keys and
             of the queries on the way
attention    the queries of new tokens over that cache: one token of many sequences when decoding, chunks of a
             prompt behind what is there already; causal, with a sliding window and first tokens that stay
logprobs     the log probability of a given token in every row of logits, the row's entropy and its likeliest
             tokens

`own` False computes them with elementary torch operations, `own` True through strata_cuda.
"""
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one new token for each of 64 running sequences: f32 projections, the queries handed on in bf16
        dict(name="append decode 64", op="append", lens="64x1", past="0-8000", hq=32, hkv=8, d=128, page=16, rot=128, pairs="halves", dtype="f32", out="bf16"),
        # a prompt of 8192 tokens written at once
        dict(name="append prompt 8192", op="append", lens="1x8192", past="0", hq=32, hkv=8, d=128, page=64, rot=128, pairs="halves", dtype="f32", out="bf16"),
        # chunks of odd lengths, one of them empty, a head size that fills no tile, part of it rotated in neighbouring pairs, far positions
        dict(name="append ragged odd", op="append", lens="513,1,0,1030,3,777", past="100000,7,5,0,90001,33", hq=9, hkv=3, d=80, page=16, rot=40, pairs="neighbours", dtype="bf16", out="bf16"),
        # one sequence answering: the latency of a single token
        dict(name="attention decode 1", op="attention", lens="1x1", past="4100", hq=32, hkv=8, d=128, page=16, window=0, sinks=0, dtype="bf16"),
        # 64 running sequences of mixed lengths: the cache is the traffic
        dict(name="attention decode 64", op="attention", lens="64x1", past="100-16000", hq=32, hkv=8, d=128, page=16, window=0, sinks=0, dtype="bf16"),
        # f32 activations, as the quantized products give them; far contexts under a window with first tokens that stay
        dict(name="attention decode 32 window f32", op="attention", lens="32x1", past="1000-60000", hq=16, hkv=2, d=256, page=32, window=4096, sinks=4, dtype="f32"),
        # a prompt of 8192 tokens read at once
        dict(name="attention prompt 8192", op="attention", lens="1x8192", past="0", hq=32, hkv=8, d=128, page=64, window=0, sinks=0, dtype="bf16"),
        # the next chunk of a long prompt
        dict(name="attention chunk 1024 over 20000", op="attention", lens="1x1024", past="20000", hq=32, hkv=8, d=128, page=16, window=0, sinks=0, dtype="bf16"),
        # chunks and single tokens in one batch, a head size that fills no tile, three queries a key head, window
        dict(name="attention mixed odd", op="attention", lens="700,1,0,1301,1,64,5,1", past="0,3001,9,2000,64,129,8191,15", hq=9, hkv=3, d=80, page=16, window=1000, sinks=7, dtype="bf16"),
        # one answer of the 2048 -> 151936 head, with 20 alternatives
        dict(name="logprobs 1", op="logprobs", rows=1, vocab=151936, top=20, masked=False),
        # a prompt's chunk scored
        dict(name="logprobs 1024", op="logprobs", rows=1024, vocab=151936, top=5, masked=False),
        # an odd vocabulary under grammar masks: most logits -inf, a row that leaves nothing, equal logits
        dict(name="logprobs 33 masked", op="logprobs", rows=33, vocab=32003, top=20, masked=True),
    ]


def _lens(text):
    if "x" in text:
        n, length = (int(v) for v in text.split("x"))
        return [length] * n
    return [int(v) for v in text.split(",")]


def _past(text, n):
    """What n sequences hold before the call: one number for all, one for each, or spread over a range (as their logarithms)."""
    if "-" in text:
        lo, hi = (int(v) for v in text.split("-"))
        return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (((i * 37) % n) / max(1, n - 1)))) - 1 for i in range(n)]
    each = [int(v) for v in text.split(",")]
    return each if len(each) == n else each * n


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lens(rng, longest, pairs):
    """Single tokens of many sequences, one chunk, or several of mixed lengths, with what is there before: `pairs` of
    a query and a key at most."""
    kind = rng.random()
    if kind < 0.4:
        n, lo = _log(rng, 1, 128), rng.choice([0, 100])
        return "%dx1" % n, "%d-%d" % (lo, lo + _log(rng, 16, 16000))
    if kind < 0.65:
        n = _log(rng, 2, longest)
        past = rng.choice([0, 0, _log(rng, 1, 20000)])
        return "1x%d" % n, str(min(past, pairs // n))
    lens, past = [], []
    for _ in range(rng.randint(2, 9)):
        lens.append(rng.choice([0, 1, _log(rng, 2, longest // 4), _log(rng, 2, longest // 4)]))
        past.append(min(rng.choice([0, _log(rng, 1, 9000)]), pairs // 8 // max(1, lens[-1])))
    if not any(lens):
        lens[0] = 1
    return ",".join(map(str, lens)), ",".join(map(str, past))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "logprobs"])
    if op == "logprobs":
        rows = _log(rng, 1, 800)
        return dict(op="logprobs", rows=rows, vocab=_log(rng, 1000, 160000), top=rng.choice([0, 1, 5, 20, 32]), masked=rng.random() < 0.3)
    hkv = _log(rng, 1, 8)
    heads = dict(hq=hkv * rng.choice([1, 2, 3, 4, 4, 8]), hkv=hkv, d=rng.choice([64, 128, 128, 256, 8 * _log(rng, 2, 32)]), page=rng.choice([16, 16, 32, 64, 128, 48]))
    dtype = rng.choice(["f32", "bf16", "bf16"])
    if op == "append":
        lens, past = _draw_lens(rng, 6000, 1 << 40)
        return dict(op="append", lens=lens, past=past, **heads, rot=rng.choice([heads["d"], 2 * _log(rng, 1, heads["d"] // 2)]),
                    pairs=rng.choice(["halves", "neighbours"]), dtype=dtype, out=dtype if dtype == "bf16" else rng.choice(["f32", "bf16"]))
    if heads["hq"] * heads["d"] > 4096:
        heads["hq"] = hkv
    lens, past = _draw_lens(rng, 6000, 16000000)
    window = rng.choice([0, 0, _log(rng, 1, 4096)])
    return dict(op="attention", lens=lens, past=past, **heads, window=window, sinks=rng.choice([0, rng.randint(1, 16)]) if window else 0, dtype=dtype)


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if case["op"] == "logprobs":
        return _prepare_logprobs(case, normal, uniform)
    lens = _lens(case["lens"])
    past = _past(case["past"], len(lens))
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    total = offsets[-1]
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    dt = DTYPES[case["dtype"]]
    state = dict(case, offsets=offsets, total=total, n_seq=len(lens), seq_len=lens[0] if len(set(lens)) == 1 else -1, dt=dt,
                 kv=[p + n for p, n in zip(past, lens)])
    # every sequence has the pages it needs, in any order in the pool; the rest of its row of the table is no page
    need = [-(-n // page) for n in state["kv"]]
    width, pages = max(1, max(need)), sum(need) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    state["table"], state["width"], state["pages"] = table, width, pages
    state["len"] = torch.tensor(state["kv"], dtype=torch.int32, device="cuda")
    state["k"], state["v"] = (normal(pages, page, hkv, d).bfloat16() for _ in range(2))
    if case["op"] == "append":
        # q | k | v side by side, as one projection leaves them
        state["qkv"] = normal(total, (hq + 2 * hkv) * d).to(dt)
        return state
    state["q"] = (normal(total, hq, d) * 1.5).to(dt)
    return state


def _prepare_logprobs(case, normal, uniform):
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab) * 2.5
    # a few tokens stand out, as they do after a trained head, and the scored token is often one of them
    at = (uniform(rows, 12) * vocab).long().clamp_(max=vocab - 1)
    logits.scatter_(1, at, 8.0 + 5.0 * uniform(rows, 12))
    target = torch.where(uniform(rows) < 0.7, at[:, 0], (uniform(rows) * vocab).long().clamp_(max=vocab - 1)).int()
    if case["masked"]:
        allowed = uniform(rows, vocab) < 0.01
        for r in range(rows):
            if r % 4 == 1:
                logits[r] = torch.where(allowed[r], logits[r], torch.full_like(logits[r], -math.inf))
            elif r % 4 == 2:
                logits[r] = torch.round(logits[r] * 2) / 2  # many equal values
            elif r == 3:
                logits[r] = -math.inf
    return dict(case, logits=logits, target=target)


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return {"append": _append_own, "attention": _attention_own, "logprobs": _logprobs_own}[state["op"]](state)
    return {"append": _append_plain, "attention": _attention_plain, "logprobs": _logprobs_plain}[state["op"]](state)


def _qkv(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    return s["qkv"][:, : hq * d].unflatten(1, (hq, d)), s["qkv"][:, hq * d: (hq + hkv) * d].unflatten(1, (hkv, d)), s["qkv"][:, (hq + hkv) * d:].unflatten(1, (hkv, d))


def _where(s):
    """Per token of the call: its position, and its page and row there."""
    off = torch.tensor(s["offsets"], device="cuda")
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(off[1:], row, right=True)
    pos = s["len"][seq] - (off[seq + 1] - row)
    return pos, s["table"][seq, pos // s["page"]].long(), pos % s["page"]


def _append_plain(s):
    q, k, v = (x.float() for x in _qkv(s))
    pos, page, slot = _where(s)
    rot, half = s["rot"], s["rot"] // 2
    theta = 10000.0 ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / rot)
    angle = pos.double()[:, None] * theta
    c, sn = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(x):
        x = x.clone()
        ia, ib = (slice(0, half), slice(half, rot)) if s["pairs"] == "halves" else (slice(0, rot, 2), slice(1, rot, 2))
        a, b = x[..., ia].clone(), x[..., ib].clone()
        x[..., ia], x[..., ib] = a * c - b * sn, a * sn + b * c
        return x

    s["k"][page, slot] = turn(k).bfloat16()
    s["v"][page, slot] = v.bfloat16()
    return {"q": turn(q).to(DTYPES[s["out"]]), "k": s["k"], "v": s["v"]}


def _attention_plain(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    o = torch.zeros(s["total"], hq, d, device="cuda")
    for i, (a, b) in enumerate(zip(s["offsets"], s["offsets"][1:])):
        n, m = b - a, s["kv"][i]
        if n == 0:
            continue
        pages = s["table"][i, : -(-m // s["page"])].long()
        k, v = (s[x][pages].flatten(0, 1)[:m].float() for x in ("k", "v"))
        p = torch.arange(m - n, m, device="cuda")[:, None, None]
        j = torch.arange(m, device="cuda")
        seen = j <= p
        if s["window"]:
            seen = seen & ((j > p - s["window"]) | (j < s["sinks"]))
        for h in range(hkv):
            g = slice(h * hq // hkv, (h + 1) * hq // hkv)
            x = torch.where(seen, (s["q"][a:b, g].float() @ k[:, h].T) * d ** -0.5, -math.inf)
            e = torch.exp(x - x.amax(-1, keepdim=True))
            o[a:b, g] = (e @ v[:, h]) / e.sum(-1, keepdim=True)
    return {"o": o.to(s["dt"])}


def _logprobs_plain(s):
    x = torch.where(s["logits"].isnan(), -math.inf, s["logits"])
    top = x.amax(1, keepdim=True)
    d = torch.where(x == top, 0.0, x - top).double()  # a row's sum is next to 1 where one token has nearly everything
    e = torch.where(x == -math.inf, 0.0, torch.exp(d))
    z = e.sum(1, keepdim=True)
    logz = torch.log(z)
    logp = torch.where(x == -math.inf, -math.inf, d - logz)
    entropy = logz - (e * torch.where(e > 0, d, 0.0)).sum(1, keepdim=True) / z
    out = {"logprobs": logp.gather(1, s["target"].long()[:, None])[:, 0].float(),
           "entropy": torch.where(z > 0, entropy, 0.0)[:, 0].float()}
    if s["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : s["top"]]
        lp = logp.gather(1, ids)
        out["ids"] = torch.where(lp == -math.inf, -1, ids).int()
        out["top"] = lp.float()
    return out


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


def _cache(sc, s):
    return sc.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["len"].data_ptr(), n_pages=s["pages"], page_size=s["page"],
                      n_kv_head=s["hkv"], head_dim=s["d"], max_pages=s["width"])


def _append_own(s):
    sc, ctx = _ctx()
    if "desc" not in s:
        width = s["qkv"].shape[1]
        s["cache"] = _cache(sc, s)
        s["desc"] = sc.KvAppend(n_seq=s["n_seq"], n_head=s["hq"], n_rot=s["rot"], freq_base=10000.0, neighbours=s["pairs"] == "neighbours",
                                dtype=sc.BF16 if s["dtype"] == "bf16" else sc.F32, q_dtype=sc.BF16 if s["out"] == "bf16" else sc.F32,
                                q_stride=width, k_stride=width, v_stride=width, **_lengths(s))
    q, k, v = _qkv(s)
    out = torch.empty(s["total"], s["hq"], s["d"], dtype=DTYPES[s["out"]], device="cuda")
    ctx.kv_append_dev(s["desc"], s["cache"], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stream=_stream())
    return {"q": out, "k": s["k"], "v": s["v"]}


def _attention_own(s):
    sc, ctx = _ctx()
    if "desc" not in s:
        s["cache"] = _cache(sc, s)
        s["desc"] = sc.Attention(n_seq=s["n_seq"], n_head=s["hq"], window=s["window"], sinks=s["sinks"], scale=s["d"] ** -0.5,
                                 dtype=sc.BF16 if s["dtype"] == "bf16" else sc.F32, **_lengths(s))
        s["work"] = torch.empty(max(16, sc.attention_work_bytes(s["desc"], s["cache"])), dtype=torch.uint8, device="cuda")
    o = torch.empty(s["total"], s["hq"], s["d"], dtype=s["dt"], device="cuda")
    ctx.attention_dev(s["desc"], s["cache"], s["q"].data_ptr(), o.data_ptr(), s["work"].data_ptr(), s["work"].numel(), stream=_stream())
    return {"o": o}


def _logprobs_own(s):
    _, ctx = _ctx()
    rows, vocab, n = s["rows"], s["vocab"], s["top"]
    f32 = dict(dtype=torch.float32, device="cuda")
    out = {"logprobs": torch.empty(rows, **f32), "entropy": torch.empty(rows, **f32)}
    if n:
        out["ids"], out["top"] = torch.empty(rows, n, dtype=torch.int32, device="cuda"), torch.empty(rows, n, **f32)
    ctx.logprobs_dev(s["logits"].data_ptr(), rows, vocab, s["target"].data_ptr(), out["logprobs"].data_ptr(), entropy_ptr=out["entropy"].data_ptr(),
                     top=n, top_ids_ptr=out["ids"].data_ptr() if n else 0, top_logprobs_ptr=out["top"].data_ptr() if n else 0, stream=_stream())
    return out


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # every logit once; an exponential, two sums and a comparison's worth for each
        return {"bytes": rows * (vocab * 4 + 12 + 8 * case["top"]), "flops": rows * vocab * 12}
    lens = _lens(case["lens"])
    kv = [p + n for p, n in zip(_past(case["past"], len(lens)), lens)]
    total, hq, hkv, d, size = sum(lens), case["hq"], case["hkv"], case["d"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "append":
        out = 2 if case["out"] == "bf16" else 4
        # q, k and v once, the rotated queries and both rows of the cache once; six products and sums a rotated pair
        return {"bytes": total * ((hq + 2 * hkv) * d * size + hq * d * out + 2 * hkv * d * 2), "flops": total * (hq + hkv) * case["rot"] * 3}
    w, sinks, keys, pairs = case["window"], case["sinks"], 0, 0
    for n, m in zip(lens, kv):
        if n == 0:
            continue
        first = m - n  # the first query's position
        if not w:
            keys += m
            pairs += n * first + n * (n + 1) // 2
            continue
        begin = max(0, first - w + 1)
        keys += m - begin + min(sinks, begin)
        pairs += sum(min(p + 1, w) + max(0, min(sinks, p + 1 - w)) for p in range(first, m))
    # the keys and values that some query sees, q and o once; q k and p v for every visible pair
    return {"bytes": keys * 2 * hkv * d * 2 + total * 2 * hq * d * size, "flops": pairs * hq * d * 4}


# ---------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attention": _attention_exact, "logprobs": _logprobs_exact}[case["op"]](s)


def _append_exact(s):
    """Sequence by sequence; a pair is a complex number that is turned by its angle."""
    q, k, v = (x.double() for x in _qkv(s))
    kc, vc, qo = s["k"].double(), s["v"].double(), q.clone()
    freq = torch.exp(torch.arange(s["rot"] // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(10000.0) / s["rot"]))
    for i, (a, b) in enumerate(zip(s["offsets"], s["offsets"][1:])):
        if a == b:
            continue
        pos = torch.arange(s["kv"][i] - (b - a), s["kv"][i], device="cuda")
        unit = torch.polar(torch.ones_like(freq).expand(b - a, -1).contiguous(), pos.double()[:, None] * freq)[:, None]
        turned = []
        for x in (q[a:b], k[a:b]):
            y, front = x.clone(), x[..., : s["rot"]]
            pair = front.unflatten(-1, (2, -1)).transpose(-1, -2) if s["pairs"] == "halves" else front.unflatten(-1, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * unit)
            y[..., : s["rot"]] = (z.transpose(-1, -2) if s["pairs"] == "halves" else z).flatten(-2)
            turned.append(y)
        at = s["table"][i].long()[pos // s["page"]], pos % s["page"]
        qo[a:b], kc[at], vc[at] = turned[0], turned[1], v[a:b]
    return {"q": qo, "k": kc, "v": vc}


def _attention_exact(s):
    """Blocks of queries over the keys that some of them see."""
    r, d = s["hq"] // s["hkv"], s["d"]
    o = torch.zeros(s["total"], s["hq"], d, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(s["offsets"], s["offsets"][1:])):
        first = s["kv"][i] - (b - a)
        for t in range(a, b, 512):
            u = min(b, t + 512)
            p = torch.arange(first + t - a, first + u - a, device="cuda")
            j = torch.arange(int(first + u - a), device="cuda")
            if s["window"]:
                j = j[(j > first + t - a - s["window"]) | (j < s["sinks"])]
            at = s["table"][i].long()[j // s["page"]], j % s["page"]
            k, v = s["k"][at].double(), s["v"][at].double()
            hidden = j[None] > p[:, None]
            if s["window"]:
                hidden |= (p[:, None] - j[None] >= s["window"]) & (j[None] >= s["sinks"])
            score = torch.einsum("thrd,jhd->hrtj", s["q"][t:u].double().unflatten(1, (-1, r)), k) / math.sqrt(d)
            prob = torch.softmax(score.masked_fill_(hidden, -math.inf), -1)
            o[t:u] = torch.einsum("hrtj,jhd->thrd", prob, v).flatten(1, 2)
    return {"o": o}


def _logprobs_exact(s):
    """Row by row: a log softmax over the candidates that are left, in falling order."""
    logp, entropy, ids, top = [], [], [], []
    for r in range(s["rows"]):
        x = s["logits"][r].double()
        cand = torch.argsort(-x, stable=True)
        cand = cand[: int((x > -math.inf).sum())]
        lp = torch.full_like(x, -math.inf)
        if len(cand):
            lp[cand] = torch.log_softmax(x[cand], 0)
        logp.append(lp[int(s["target"][r])])
        entropy.append(-(torch.exp(lp[cand]) * lp[cand]).sum())
        first = cand[: s["top"]]
        blank = s["top"] - len(first)
        ids.append(torch.nn.functional.pad(first, (0, blank), value=-1))
        top.append(torch.nn.functional.pad(lp[first], (0, blank), value=-math.inf))
    out = {"logprobs": torch.stack(logp), "entropy": torch.stack(entropy)}
    if s["top"]:
        out["ids"], out["top"] = torch.stack(ids).int(), torch.stack(top)
    return out
