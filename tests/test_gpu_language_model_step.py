"""The operators of a packed language-model step together, as they are used: a
training step (RMSNorm, linear attention, fused residual add + RMSNorm, the
log probabilities of the next tokens with an entropy term, backward) against
the same model in fp64 on the CPU, and the same model decoding token by token
from its prompts' states.

fp32 throughout.  Bound: with e = 2^-24, every stage's result is off by a few
hundred e of the sums it is made of (dots of 64 to 96, chunks of 64, rows of
211 logits), and six stages follow one another, each passing errors on with a
factor of order one (the norms keep the activations at unit size); 2^-24 x
2,000 = 1.2e-4 of the largest value of each compared tensor covers them.
"""

from __future__ import annotations

import math

import pytest
import torch

from parity import cu_of, say

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, HIDDEN, VOCAB = 4, 2, 24, 96, 211
LENGTHS = [70, 1, 0, 200, 33]
REL = 2000 * 2.0 ** -24


def _model(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).float()  # noqa: E731
    return {"emb": r(VOCAB, HIDDEN), "n1": 1 + 0.1 * r(HIDDEN), "wq": r(HIDDEN, HEADS * DIM) / math.sqrt(HIDDEN),
            "wk": r(HIDDEN, KV * DIM) / math.sqrt(HIDDEN), "wv": r(HIDDEN, KV * DIM) / math.sqrt(HIDDEN),
            "wo": r(HEADS * DIM, HIDDEN) / math.sqrt(HEADS * DIM), "n2": 1 + 0.1 * r(HIDDEN),
            "head": r(HIDDEN, VOCAB) / math.sqrt(HIDDEN)}


DECAY = torch.tensor([-0.02, -0.3])


def _tokens():
    n = sum(LENGTHS)
    tokens = torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(3))
    targets = torch.full((n,), -1)
    a = 0
    for length in LENGTHS:
        if length:
            targets[a:a + length - 1] = tokens[a + 1:a + length]  # a sequence's last token has none
        a += length
    return tokens, targets


def _qkv(p, h):
    return ((h @ p["wq"]).view(-1, HEADS, DIM), (h @ p["wk"]).view(-1, KV, DIM), (h @ p["wv"]).view(-1, KV, DIM))


def _reference(p, tokens, targets, weights):
    """Logits and the loss's gradients in fp64 on the CPU."""
    p = {k: v.double().requires_grad_(True) for k, v in p.items()}
    rms = lambda x, w: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    x = p["emb"][tokens]
    q, k, v = _qkv(p, rms(x, p["n1"]))
    lam = DECAY.double().exp()[:, None, None]
    outs, a = [], 0
    for length in LENGTHS:
        s = torch.zeros(KV, DIM, DIM, dtype=torch.float64)
        for t in range(a, a + length):
            s = lam * s + k[t][:, :, None] * v[t][:, None, :]
            outs.append((q[t].view(KV, -1, DIM) @ s).reshape(HEADS * DIM) / math.sqrt(DIM))
        a += length
    h = x + torch.stack(outs) @ p["wo"]
    logits = rms(h, p["n2"]) @ p["head"]
    lp = torch.log_softmax(logits, dim=-1)
    picked = torch.where(targets >= 0, lp.gather(1, targets.clamp(min=0)[:, None])[:, 0], torch.zeros(()).double())
    entropy = -(lp.exp() * lp).sum(-1)
    loss = -(weights.double() * picked).sum() - 0.01 * entropy.sum()
    loss.backward()
    return logits.detach(), loss.detach(), {k: v.grad for k, v in p.items()}


def _forward(p, x, mix):
    from scree_amd.kernels.hip import varlen_add_rmsnorm_hip, varlen_rmsnorm_hip

    o = mix(*_qkv(p, varlen_rmsnorm_hip(x, p["n1"], 1e-6)))
    _, y = varlen_add_rmsnorm_hip(x, o.reshape(-1, HEADS * DIM) @ p["wo"], p["n2"], 1e-6)
    return y @ p["head"]


def _close(name, got, want):
    want = want.double()
    err = float((got.detach().double().cpu() - want).abs().max())
    room = REL * max(1.0, float(want.abs().max()))
    say(f"  {name}: max_abs={err:.3e} of {room:.3e}")
    assert err <= room, name


def test_training_step():
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_token_logprobs_hip

    tokens, targets = _tokens()
    weights = torch.randn(len(tokens), generator=torch.Generator().manual_seed(4))
    cpu = _model()
    ref_logits, ref_loss, ref_grads = _reference(cpu, tokens, targets, weights)
    p = {k: v.cuda().requires_grad_(True) for k, v in cpu.items()}
    _, cu = cu_of(LENGTHS)
    g = DECAY.cuda()
    logits = _forward(p, p["emb"][tokens.cuda()],
                      lambda q, k, v: varlen_linear_attention_hip(q, k, v, g, cu))
    out = varlen_token_logprobs_hip(logits, targets.cuda())
    loss = -(weights.cuda() * out.logprob).sum() - 0.01 * out.entropy.sum()
    loss.backward()
    _close("logits", logits, ref_logits)
    _close("loss", loss, ref_loss)
    for k in p:
        _close(f"d{k}", p[k].grad, ref_grads[k])


def test_prompts_then_decoding():
    """Prompts' states carried into single-token steps give the logits of the
    whole sequences, and each step's alternatives are the reference's."""
    from scree_amd.kernels.hip import (linear_attention_step_hip, varlen_linear_attention_hip,
                                       varlen_token_logprobs_hip)

    tokens, targets = _tokens()
    cpu = _model()
    ref_logits, _, _ = _reference(cpu, tokens, targets, torch.ones(len(tokens)))
    p = {k: v.cuda() for k, v in cpu.items()}
    g = DECAY.cuda()
    starts = [0, 71, 271]  # the sequences of 70, 200 and 33 tokens
    prompts = [60, 190, 23]
    rows = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, prompts)])
    _, cu = cu_of(prompts)
    kept = {}

    def prompt(q, k, v):
        o, kept["state"] = varlen_linear_attention_hip(q, k, v, g, cu, return_state=True)
        return o

    _close("prompt logits", _forward(p, p["emb"][tokens[rows].cuda()], prompt), ref_logits[rows])
    for i in range(10):
        at = torch.tensor([a + n + i for a, n in zip(starts, prompts)])
        logits = _forward(p, p["emb"][tokens[at].cuda()],
                          lambda q, k, v: linear_attention_step_hip(q, k, v, g, kept["state"]))
        _close(f"step {i} logits", logits, ref_logits[at])
        out = varlen_token_logprobs_hip(logits, targets[at].cuda(), top_k=5)
        ref = torch.log_softmax(ref_logits[at], dim=-1)
        _close(f"step {i} alternatives", out.top_logprob, ref.topk(5, dim=-1).values)
