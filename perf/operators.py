"""Linear attention with a decay per head and the log probabilities of given
tokens, over packed sequences: timed cases, plain forms and 64-bit results.

``listed()`` gives the fixed cases, ``draw(rng)`` one more of the ranges they
stand for, ``prepare(case, seed)`` the inputs on the GPU, ``run(state)`` one
pass, ``exact(case, seed)`` its outputs in 64 bits and ``work(case)`` the bytes
and operations a pass cannot do without.  With ``own`` false ``run`` computes
the plain form from elementary torch operations in 32 bits; with ``own`` true
it makes the calls a user makes of this package.

Linear attention, per sequence and K/V head with decay ``lam = exp(log_decay)``:
``S_t = lam S_{t-1} + k_t v_t^T`` and ``o_t = scale q_t S_t``; the single-token
step is one turn of that recurrence for every sequence of a batch.  The log
probabilities are ``x_y - logsumexp(x)`` of each row's given token, with the
row's entropy and its most likely tokens.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"
CHUNK = 64


# ------------------------------------------------------------------- cases
def _linear(name, *, dtype, heads, kv_heads, k_dim, v_dim, seqs, mean_len, sigma, len_seed, train,
            state, total=0):
    # state: an initial state comes in and the final state goes out
    return {"name": name, "kind": "linear", "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "k_dim": k_dim, "v_dim": v_dim, "seqs": seqs, "mean_len": mean_len, "sigma": sigma,
            "len_seed": len_seed, "total": total, "train": train, "state": state}


def _step(name, *, dtype, heads, kv_heads, k_dim, v_dim, seqs):
    return {"name": name, "kind": "step", "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "k_dim": k_dim, "v_dim": v_dim, "seqs": seqs}


def _logp(name, *, dtype, rows, vocab, top_k, train, masked):
    # masked: the share of the vocabulary that is ruled out (-inf) in each row
    return {"name": name, "kind": "logp", "dtype": dtype, "rows": rows, "vocab": vocab,
            "top_k": top_k, "train": train, "masked": masked}


def listed():
    return [
        # A short request batch of a small model: 16 sequences of mean 128, 4
        # heads of 32, forward only.  Latency.
        _linear("linear_fwd_small_fp16", dtype="fp16", heads=4, kv_heads=4, k_dim=32, v_dim=32,
                seqs=16, mean_len=128, sigma=0.6, len_seed=0, train=False, state=False),
        # Prefill of a mixed batch of prompts, 32 query heads on 8 K/V heads of
        # 128, the states going on to decoding.
        _linear("linear_prefill_gqa_bf16", dtype="bf16", heads=32, kv_heads=8, k_dim=128, v_dim=128,
                seqs=8, mean_len=1024, sigma=0.6, len_seed=0, train=False, state=True),
        # One long document on 16 heads of 128, continued from a state: few
        # rows, a long axis.
        _linear("linear_prefill_long_bf16", dtype="bf16", heads=16, kv_heads=16, k_dim=128,
                v_dim=128, seqs=1, mean_len=65536, sigma=0.0, len_seed=0, train=False, state=True,
                total=65536),
        # A training step of the benchmark's batch: 12,160 tokens, 16 heads of 64.
        _linear("linear_train_fp16_16x64", dtype="fp16", heads=16, kv_heads=16, k_dim=64, v_dim=64,
                seqs=16, mean_len=760, sigma=0.6, len_seed=0, train=True, state=False, total=12160),
        # Long-context pretraining: 32 sequences up to 16k tokens, 32 heads of
        # 128 (the largest case).
        _linear("linear_train_bf16_32x128", dtype="bf16", heads=32, kv_heads=32, k_dim=128,
                v_dim=128, seqs=32, mean_len=2048, sigma=1.2, len_seed=0, train=True, state=False),
        # Training in fp32: 16 sequences of mean 256, 8 heads of 64.
        _linear("linear_train_fp32_8x64", dtype="fp32", heads=8, kv_heads=8, k_dim=64, v_dim=64,
                seqs=16, mean_len=256, sigma=0.6, len_seed=0, train=True, state=False),
        # One decoding step of a single request, 16 heads of 128.  Latency.
        _step("step_1_bf16", dtype="bf16", heads=16, kv_heads=16, k_dim=128, v_dim=128, seqs=1),
        # One decoding step of a full serving batch with grouped query heads.
        _step("step_256_gqa_bf16", dtype="bf16", heads=32, kv_heads=8, k_dim=128, v_dim=128, seqs=256),
        # Log probabilities of 16 sampled tokens with 20 alternatives each, a
        # tenth of the vocabulary ruled out: one decoding step.
        _logp("logp_decode_top20_bf16", dtype="bf16", rows=16, vocab=128000, top_k=20, train=False,
              masked=0.1),
        # Scoring a batch of given texts with 5 alternatives, odd vocabulary.
        _logp("logp_score_top5_fp16", dtype="fp16", rows=1980, vocab=50021, top_k=5, train=False,
              masked=0.0),
        # The loss of the benchmark's batch with an entropy term: 12,160 rows of
        # 32,000, forward and backward.
        _logp("logp_train_bf16", dtype="bf16", rows=12160, vocab=32000, top_k=0, train=True,
              masked=0.0),
        # The same loss on logits kept in fp32, fewer rows, odd vocabulary.
        _logp("logp_train_fp32", dtype="fp32", rows=986, vocab=50257, top_k=0, train=True, masked=0.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "step", "logp", "logp"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if kind == "logp":
        vocab, rows = _log_int(rng, 1000, 160000), _log_int(rng, 1, 12160)
        train = rng.random() < 0.5
        top_k = 0 if train else rng.randrange(0, 33)
        rows = max(1, min(rows, (400 << 20) // DTYPES[dtype].itemsize // vocab))
        return _logp(None, dtype=dtype, rows=rows, vocab=vocab, top_k=top_k, train=train,
                     masked=rng.choice([0.0, 0.0, 0.1, 0.9]))
    k_dim = rng.choice([32, 64, 64, 96, 128, 128, 256])
    v_dim = k_dim if rng.random() < 0.7 else rng.choice([32, 64, 96, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    if kind == "step":
        seqs = _log_int(rng, 1, 512)
        seqs = max(1, min(seqs, (1 << 27) // (kv_heads * k_dim * v_dim)))
        return _step(None, dtype=dtype, heads=heads, kv_heads=kv_heads, k_dim=k_dim, v_dim=v_dim,
                     seqs=seqs)
    seqs = _log_int(rng, 1, 96)
    tokens = _log_int(rng, 64, 65536)
    while tokens * heads * max(k_dim, v_dim) > 1 << 26:
        tokens = tokens * 2 // 3
    return _linear(None, dtype=dtype, heads=heads, kv_heads=kv_heads, k_dim=k_dim, v_dim=v_dim,
                   seqs=seqs, mean_len=max(1, tokens // seqs), sigma=round(rng.uniform(0.2, 1.2), 2),
                   len_seed=rng.randrange(1 << 20), train=rng.random() < 0.5,
                   state=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Log-normal sequence lengths, as the benchmark's sampler draws them;
    rescaled to ``total`` tokens when that is set."""
    rng = np.random.default_rng(case["len_seed"])
    x = rng.lognormal(mean=np.log(case["mean_len"]), sigma=case["sigma"], size=case["seqs"])
    if case["total"]:
        x = x * (case["total"] / x.sum())
    n = [max(1, int(v)) if case["total"] else min(16384, max(1, int(v))) for v in x]
    if case["total"]:
        n[int(np.argmax(n))] += case["total"] - sum(n)
    return n


def _offsets(lengths):
    off = np.zeros(len(lengths) + 1, dtype=np.int32)
    off[1:] = np.cumsum(lengths)
    return torch.from_numpy(off).to(DEVICE)


def _randn(gen, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32)
    return (x * scale).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "logp":
        n, v = case["rows"], case["vocab"]
        t = {"logits": _randn(gen, (n, v), dt, 2.5)}
        t["targets"] = torch.randint(0, v, (n,), generator=gen, device=DEVICE)
        if case["masked"]:
            out = torch.rand((n, v), generator=gen, device=DEVICE) < case["masked"]
            out.scatter_(1, t["targets"][:, None], False)  # a sampled token is never ruled out
            t["logits"].masked_fill_(out, -math.inf)
        if case["train"]:
            # the weight of each token's log probability (advantages) and of its entropy
            t["dlogp"] = _randn(gen, (n,), torch.float32)
            t["dentropy"] = _randn(gen, (n,), torch.float32, 0.1)
        return t
    h, hk, dk, dv = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"]
    n = case["seqs"] if case["kind"] == "step" else sum(_lengths(case))
    t = {"q": _randn(gen, (n, h, dk), dt), "k": _randn(gen, (n, hk, dk), dt),
         "v": _randn(gen, (n, hk, dv), dt)}
    # decays from 1 - 2^-4 to 1 - 2^-8 over the heads, so that their memories
    # reach from tens to hundreds of tokens
    reach = torch.arange(hk, device=DEVICE, dtype=torch.float64) / hk
    t["log_decay"] = torch.log1p(-torch.exp2(-4 - 4 * reach)).float()
    if case["kind"] == "step" or case["state"]:
        b = case["seqs"]
        t["state"] = _randn(gen, (b, hk, dk, dv), torch.float32, 4.0)
    if case["kind"] == "linear" and case["train"]:
        t["do"] = _randn(gen, (n, h, dv), dt)
        if case["state"]:
            t["dstate"] = _randn(gen, (case["seqs"], hk, dk, dv), torch.float32)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    st = {"case": case, "t": t}
    if case["kind"] == "linear":
        st["lengths"] = _lengths(case)
        st["cu"] = _offsets(st["lengths"])
    if case["kind"] == "step":
        st["new_state"] = torch.empty_like(t["state"])
    if own and case.get("train"):
        for name in ("q", "k", "v", "state", "logits"):
            if name in t:
                t[name].requires_grad_(True)
    return st


# -------------------------------------------------------------- plain forms
def _rows_of_chunks(lengths, reverse):
    """Rows (chunks, CHUNK) of every sequence's chunks, -1 past a sequence's
    end, each sequence's first chunk, chunk count and each chunk's row count;
    ``reverse`` runs every sequence from its last row."""
    n = np.asarray(lengths, dtype=np.int64)
    start = np.concatenate([[0], np.cumsum(n)])[:-1]
    counts = (n + CHUNK - 1) // CHUNK
    first = np.concatenate([[0], np.cumsum(counts)])[:-1]
    seq = np.repeat(np.arange(len(n)), counts)
    pos = (np.arange(counts.sum()) - first[seq])[:, None] * CHUNK + np.arange(CHUNK)
    row = start[seq][:, None] + (n[seq][:, None] - 1 - pos if reverse else pos)
    row = np.where(pos < n[seq][:, None], row, -1)
    return torch.from_numpy(row).to(DEVICE), first, counts, np.minimum(n[seq] - pos[:, 0], CHUNK)


def _decayed(x, y, z, log_decay, lengths, reverse, state, zscale):
    """``out_i = sum_{j <= i} lam^{i-j} (x_i . y_j) z_j * zscale + x_i . A_i`` with
    the state's share ``A_i``, and the last state; rows x, y, z (n, heads,
    groups, dim) run from each sequence's end when ``reverse``.  Forward the
    state comes in from before the first row (its share is lam^{i+1}), reversed
    it joins at the last row (lam^i)."""
    n, hk, gx, dx = x.shape
    gy, dz = y.shape[2], z.shape[3]
    e = 0 if reverse else 1
    rows, first, counts, lens = _rows_of_chunks(lengths, reverse)
    ok = (rows >= 0).view(*rows.shape, 1, 1, 1)

    def chunks(t, g):  # (n, hk, g, d) -> (chunks, hk, g * CHUNK, d) in 32 bits
        c = t.float()[rows.clamp(min=0)] * ok
        return c.permute(0, 2, 3, 1, 4).reshape(len(rows), hk, g * CHUNK, -1)

    xc, yc, zc = chunks(x, gx), chunks(y, gy), chunks(z, gy) * zscale
    step = torch.arange(CHUNK, device=DEVICE)
    lag = step[:, None] - step[None, :]
    lam = torch.where(lag >= 0, torch.exp(log_decay.view(-1, 1, 1) * lag.clamp(min=0)), 0.0)
    p = torch.matmul(xc, yc.transpose(2, 3).contiguous()) * lam.repeat(1, gx, gy)
    out = torch.matmul(p, zc)
    del p
    count = torch.from_numpy(lens).to(DEVICE)
    left = (count[:, None] - e - step).clamp(min=0).float()
    w = torch.exp(log_decay.view(1, -1, 1) * left[:, None, :]).repeat(1, 1, gy)
    u = torch.matmul((yc * w[..., None]).transpose(2, 3).contiguous(), zc)
    keep = torch.exp(log_decay[None, :] * count[:, None].float())[..., None, None]
    a = state.clone() if state is not None else torch.zeros((len(lengths), hk, dx, dz), device=DEVICE)
    came = torch.empty_like(u)
    order = np.argsort(-counts, kind="stable")
    for j in range(int(counts.max())):
        live = order[:int((counts > j).sum())]
        at, seq = torch.from_numpy(first[live] + j).to(DEVICE), torch.from_numpy(live).to(DEVICE)
        cur = a[seq]
        came[at] = cur
        a[seq] = cur * keep[at] + u[at]
    inter = torch.exp(log_decay.view(-1, 1) * (step + e)).repeat(1, gx)
    out = out + torch.matmul(xc, came) * inter[None, :, :, None]
    out = out.view(len(rows), hk, gx, CHUNK, dz).permute(0, 3, 1, 2, 4)
    res = torch.zeros((n, hk, gx, dz), device=DEVICE)
    live = rows >= 0
    res[rows[live]] = out[live]
    return res, a


def _plain_linear(st):
    case, t, lengths = st["case"], st["t"], st["lengths"]
    n, hk = t["k"].shape[:2]
    scale = 1.0 / math.sqrt(case["k_dim"])
    q, k, v = t["q"].view(n, hk, -1, case["k_dim"]), t["k"][:, :, None], t["v"][:, :, None]
    g = t["log_decay"]
    dt = t["q"].dtype
    o, last = _decayed(q, k, v, g, lengths, False, t.get("state"), 1.0)
    out = [(o * scale).to(dt).view(n, -1, case["v_dim"])]
    if case["state"]:
        out.append(last)
    if not case["train"]:
        return tuple(out)
    do = t["do"].view(n, hk, -1, case["v_dim"])
    s0 = t["state"].transpose(2, 3).contiguous() if case["state"] else None
    dq, _ = _decayed(do, v, k, g, lengths, False, s0, 1.0)
    out.append((dq * scale).to(dt).view(n, -1, case["k_dim"]))
    ds = t.get("dstate")
    dst = ds.transpose(2, 3).contiguous() if ds is not None else None
    dk, _ = _decayed(v, do, q, g, lengths, True, dst, scale)
    dv, d0 = _decayed(k, q, do, g, lengths, True, ds, scale)
    out += [dk.to(dt)[:, :, 0], dv.to(dt)[:, :, 0]]
    if case["state"]:
        out.append(d0)
    return tuple(out)


def _plain_step(st):
    case, t = st["case"], st["t"]
    b, hk = t["k"].shape[:2]
    lam = torch.exp(t["log_decay"]).view(1, hk, 1, 1)
    s = t["state"] * lam + t["k"].float()[..., :, None] * t["v"].float()[..., None, :]
    q = t["q"].float().view(b, hk, -1, case["k_dim"])
    o = torch.matmul(q, s) * (1.0 / math.sqrt(case["k_dim"]))
    return o.view(b, -1, case["v_dim"]).to(t["q"].dtype), s


def _plain_top(x, k):
    """Values and places of the k largest of each row, the lowest place first
    among equals: one integer key holds the value's order and the place."""
    vals, places = [], []
    for c in x.split(max(1, (1 << 26) // x.shape[1])):
        bits = (c + 0.0).contiguous().view(torch.int32).long()  # + 0.0: -0.0 equals 0.0
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = key * (1 << 31) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=DEVICE))
        place = x.shape[1] - 1 - (torch.topk(key, k, dim=1).values & 0x7FFFFFFF)
        places.append(place)
        vals.append(c.gather(1, place))
    return torch.cat(vals), torch.cat(places)


def _plain_logp(st):
    case, t = st["case"], st["t"]
    x = t["logits"].detach().float()
    m = x.max(dim=1, keepdim=True).values
    ex = torch.exp(x - m)
    z = ex.sum(1, keepdim=True)
    p = ex / z
    lp = x - m - torch.log(z)
    logp = lp.gather(1, t["targets"][:, None])[:, 0]
    plogp = torch.where(p > 0, p * lp, 0.0)
    ent = -plogp.sum(1)
    out = [logp, ent]
    if case["top_k"]:
        vals, places = _plain_top(x, case["top_k"])
        out += [vals - m - torch.log(z), places]
    if case["train"]:
        glp, gh = t["dlogp"][:, None], t["dentropy"][:, None]
        dx = -p * glp - gh * (plogp + p * ent[:, None])
        dx.scatter_add_(1, t["targets"][:, None], glp)
        out.append(dx.to(t["logits"].dtype))
    return tuple(out)


# --------------------------------------------------------------------- run
def _own_linear(st):
    from scree_amd.kernels import hip

    case, t = st["case"], st["t"]
    res = hip.varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["log_decay"], st["cu"],
                                          initial_state=t.get("state"), return_state=case["state"])
    out = res if case["state"] else (res,)
    if not case["train"]:
        return tuple(out)
    leaves = [t[x] for x in ("q", "k", "v", "state") if x in t]
    grads = torch.autograd.grad(out, leaves, (t["do"], t["dstate"]) if case["state"] else (t["do"],))
    return tuple(o.detach() for o in out) + tuple(grads)


def _own_step(st):
    from scree_amd.kernels import hip

    t = st["t"]
    o = hip.linear_attention_step_hip(t["q"], t["k"], t["v"], t["log_decay"], t["state"],
                                      state_out=st["new_state"])
    return o, st["new_state"]


def _own_logp(st):
    from scree_amd.kernels import hip

    case, t = st["case"], st["t"]
    res = hip.varlen_token_logprobs_hip(t["logits"], t["targets"], top_k=case["top_k"])
    out = [res.logprob, res.entropy]
    if case["top_k"]:
        out += [res.top_logprob, res.top_index]
    if not case["train"]:
        return tuple(out)
    dx, = torch.autograd.grad(out, [t["logits"]], (t["dlogp"], t["dentropy"]))
    return tuple(o.detach() for o in out) + (dx,)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "step": _own_step, "logp": _own_logp}[kind](state)
    return {"linear": _plain_linear, "step": _plain_step, "logp": _plain_logp}[kind](state)


# -------------------------------------------------------------------- work
def work(case):
    s = DTYPES[case["dtype"]].itemsize
    if case["kind"] == "logp":
        x = s * case["rows"] * case["vocab"]
        # train: the logits once and their gradient once
        return {"bytes": (2 if case["train"] else 1) * x + case["rows"] * (16 + 12 * case["top_k"]),
                "flops": 0}
    h, hk, dk, dv = case["heads"], case["kv_heads"], case["k_dim"], case["v_dim"]
    states = 4 * case["seqs"] * hk * dk * dv
    n = case["seqs"] if case["kind"] == "step" else sum(_lengths(case))
    qo, kv = s * n * h * (dk + dv), s * n * hk * (dk + dv)
    # one update of the state and one product with it for every token
    flops = 2.0 * n * (h + hk) * dk * dv
    if case["kind"] == "step":
        return {"bytes": qo + kv + 2 * states, "flops": flops}
    moved = qo + kv + (2 * states if case["state"] else 0)
    if not case["train"]:
        return {"bytes": moved, "flops": flops}
    # q, k, v, do in, o, dq, dk, dv out; the backward has the states of both
    # directions (S again, and its gradient from every query head), dq, dk and dv
    flops += 2.0 * n * (2 * h + 3 * hk) * dk * dv
    return {"bytes": 2 * (qo + kv) + (4 * states if case["state"] else 0), "flops": flops}


# ------------------------------------------------------------------- exact
def _recurrence(x, y, z, log_decay, lengths, reverse, state):
    """The recurrence token by token: ``A = lam A + sum_groups y z^T`` then
    ``out = x A``, sequences side by side, the longest first; reversed, the
    state joins undecayed at the last row.  Returns out and the final A
    (decayed once more when reversed: the gradient of the state before)."""
    n, hk, gx, dx = x.shape
    dz = z.shape[3]
    lens = np.asarray(lengths)
    order = np.argsort(-lens, kind="stable")
    start = np.concatenate([[0], np.cumsum(lens)])[:-1][order]
    lens = lens[order]
    o = torch.from_numpy(order).to(DEVICE)
    base = torch.from_numpy(start + (lens - 1 if reverse else 0)).to(DEVICE)
    lam = torch.exp(log_decay.double()).view(1, hk, 1, 1)
    a = torch.zeros((len(lens), hk, dx, dz), dtype=torch.float64, device=DEVICE)
    if state is not None:
        a.copy_(state.double()[o])
    out = torch.zeros((n, hk, gx, dz), dtype=torch.float64, device=DEVICE)
    live_at = [int((lens > i).sum()) for i in range(int(lens.max()))]
    for i, live in enumerate(live_at):
        rows = base[:live] + (-i if reverse else i)
        s = a[:live]
        if not (reverse and i == 0):
            s.mul_(lam)
        yr = y[rows].double().flatten(0, 1).transpose(1, 2).contiguous()
        zr = z[rows].double().flatten(0, 1)
        s.view(-1, dx, dz).baddbmm_(yr, zr)
        out[rows] = torch.matmul(x[rows].double(), s)
    if reverse:
        a.mul_(lam)
    last = torch.empty_like(a)
    last[o] = a
    return out, last


def _exact_linear(case, seed):
    t = _inputs(case, seed)
    lengths = _lengths(case)
    n, hk = t["k"].shape[:2]
    scale = 1.0 / math.sqrt(case["k_dim"])
    q, k, v = t["q"].view(n, hk, -1, case["k_dim"]), t["k"][:, :, None], t["v"][:, :, None]
    o, last = _recurrence(q, k, v, t["log_decay"], lengths, False, t.get("state"))
    out = [(o * scale).view(n, -1, case["v_dim"])] + ([last] if case["state"] else [])
    if not case["train"]:
        return tuple(out)
    do = t["do"].view(n, hk, -1, case["v_dim"])
    s0 = t["state"].transpose(2, 3) if case["state"] else None
    dq, _ = _recurrence(do, v, k, t["log_decay"], lengths, False, s0)
    out.append((dq * scale).view(n, -1, case["k_dim"]))
    # R / scale: the state's gradient comes in divided by it
    ds = t["dstate"].double() / scale if case["state"] else None
    dst = ds.transpose(2, 3) if ds is not None else None
    dk, _ = _recurrence(v, do, q, t["log_decay"], lengths, True, dst)
    dv, d0 = _recurrence(k, q, do, t["log_decay"], lengths, True, ds)
    out += [dk[:, :, 0] * scale, dv[:, :, 0] * scale]
    if case["state"]:
        out.append(d0 * scale)
    return tuple(out)


def _exact_step(case, seed):
    t = _inputs(case, seed)
    group = case["heads"] // case["kv_heads"]
    s = torch.einsum("bhi,bhj->bhij", t["k"].double(), t["v"].double())
    s += t["log_decay"].double().exp()[None, :, None, None] * t["state"].double()
    q = t["q"].double() / math.sqrt(case["k_dim"])
    o = torch.stack([(q[:, j, :, None] * s[:, j // group]).sum(1) for j in range(case["heads"])], 1)
    return o, s


def _exact_logp(case, seed):
    t = _inputs(case, seed)
    parts = []
    step = max(1, (1 << 27) // case["vocab"])
    for a in range(0, case["rows"], step):
        rows = slice(a, a + step)
        lp = torch.log_softmax(t["logits"][rows].double(), dim=1)
        y = t["targets"][rows]
        p = lp.exp()
        each = torch.nan_to_num(p * lp, nan=0.0)
        ent = -each.sum(1)
        out = [lp[torch.arange(len(y), device=DEVICE), y], ent]
        if case["top_k"]:
            order = torch.sort(t["logits"][rows].float(), dim=1, descending=True, stable=True).indices
            order = order[:, :case["top_k"]].contiguous()
            out += [lp.gather(1, order), order]
        if case["train"]:
            hot = torch.zeros_like(p)
            hot[torch.arange(len(y), device=DEVICE), y] = 1.0
            dx = t["dlogp"][rows].double()[:, None] * (hot - p)
            dx -= t["dentropy"][rows].double()[:, None] * (each + p * ent[:, None])
            out.append(dx)
        parts.append(out)
    return tuple(torch.cat(c) for c in zip(*parts))


def exact(case, seed):
    # the recurrence runs token by token: past these steps it takes too long
    if case["kind"] == "linear":
        if max(_lengths(case)) * (4 if case["train"] else 1) > 100000:
            return None
        return _exact_linear(case, seed)
    return (_exact_step if case["kind"] == "step" else _exact_logp)(case, seed)
