"""GPU parity of linear attention: chunked forward and backward, single steps.

The oracle is the token-by-token recurrence in fp64 on the rounded inputs.
Every output is ``sum_j lam^{i-j} (x_i . y_j) z_j + lam^{i+e} x_i A``, and with
``abs`` the same sum over absolute values (the oracle again), ``u`` the unit
roundoff of the operands' type and ``e = 2^-24`` the bound is

    |error| <= (3.03 u + F e) abs + u |output| + small

(u: each score rounded once; each state's operand is rounded twice, as the
weighted row that enters it and as the operand of the product; 3 covers both
paths with one to spare.  fp32 operands are not rounded: u = 0 there.)  F counts the
fp32 roundings on a term's way: k products of a dot, the 64 rows of a chunk and one
factor per chunk it survives, and 64 for the weights (``lam^n`` is off by
``2 |n log lam| e``, of which terms with ``|n log lam| > 16`` keep less than
1e-7).  A final state is held to ``(F e + 2^-22) abs``: its operands come in
terms whose rest is below ``2^-22``.  fp16 rounds values below its normals to
multiples of ``2^-24``: ``small`` allows each rounded operand ``2^-25`` times
what it multiplies.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import scree_amd
from oracle.linear_attention import linear_attention_bwd, linear_attention_fwd
from parity import UNIT, cu_of, np64, randn, say

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EDGE = [1, 0, 2, 63, 64, 65, 130, 0, 17]


def check_close(name, got, want, bound, extra=0.0, unit=0.0):
    """``|got - want| <= bound + unit * extra``, bound elementwise."""
    err = np.abs(got - want)
    room = np.broadcast_to(bound + unit * extra, err.shape)
    worst = float((err - room).max()) if err.size else 0.0
    use = float((err / np.maximum(room, 1e-300)).max()) if err.size else 0.0
    say(f"  {name}: max_abs={float(err.max()) if err.size else 0:.3e} of its bound at most {use:.3f}")
    assert worst <= 0.0, f"{name}: exceeds tolerance by {worst:.3e}"


def _decays(hk, strongest=0.3):
    # the last head does not decay at all
    return torch.linspace(-strongest, 0.0, hk, dtype=torch.float32).cuda() if hk > 1 else (
        torch.tensor([-0.05]).cuda())


def _inputs(lengths, h, hk, dk, dv, dtype, seed, state, train, scale=1.0):
    n, b = sum(lengths), len(lengths)
    t = {"q": randn((n, h, dk), dtype, seed, scale=scale), "k": randn((n, hk, dk), dtype, seed + 1, scale=scale),
         "v": randn((n, hk, dv), dtype, seed + 2, scale=scale), "g": _decays(hk)}
    if state:
        t["s0"] = randn((b, hk, dk, dv), torch.float32, seed + 3)
    if train:
        t["do"] = randn((n, h, dv), dtype, seed + 4)
        if state:
            t["ds"] = randn((b, hk, dk, dv), torch.float32, seed + 5)
    return t


def _bounds(dtype, lengths, t, s, chunk=64):
    """Bounds for o, last, dq, dk, dv, dinit from the oracle over absolute values."""
    a = {k: np.abs(np64(x)) for k, x in t.items() if k != "g"}
    g = np64(t["g"])
    off, _ = cu_of(lengths)
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    longest = max(lengths) if lengths else 0
    group = t["q"].shape[1] // t["k"].shape[1]
    F = max(t["q"].shape[2], t["v"].shape[2]) + group * chunk + 4 * (longest // chunk + 1) + 64
    out = {}
    o, last = linear_attention_fwd(a["q"], a["k"], a["v"], g, off, s, a.get("s0"))
    out["o"], out["last"] = (3.03 * u + F * EPS) * o, (F * EPS + 2.0 ** -22) * last
    names = ["o"]
    if "do" in a:
        dq, dk, dv, d0 = linear_attention_bwd(a["do"], a["q"], a["k"], a["v"], g, off, s, a.get("s0"), a.get("ds"))
        for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
            out[name] = (3.03 * u + F * EPS) * x
        out["d0"] = (F * EPS + 2.0 ** -22) * d0
        names += ["dq", "dk", "dv"]
    if dtype == torch.float16:
        # a rounded score meets a z, a weighted z a y and an x, a state an x
        ones = {k: np.ones_like(x) for k, x in a.items()}
        zero = np.zeros_like(g)
        big = {k: np.maximum(x, 1.0) for k, x in a.items()}
        for name in names + ["last"] + (["d0"] if "do" in a else []):
            out[name] = out[name] + 2.0 ** -25
        o1, l1 = linear_attention_fwd(big["q"], big["k"], ones["v"], zero, off, 1.0)
        out["o"] = out["o"] + 2.0 ** -25 * (3 * o1 + linear_attention_fwd(
            ones["q"] / ones["q"].shape[2], ones["k"], big["v"], zero, off, 1.0)[0])
        out["last"] = out["last"] + 2.0 ** -25 * l1
        if "do" in a:
            for q_, k_, v_, d_ in ((big, big, big, ones), (big, big, ones, big), (big, ones, big, big), (ones, big, big, big)):
                r = linear_attention_bwd(d_["do"], q_["q"], k_["k"], v_["v"], zero, off, max(1.0, s))
                for name, x in zip(("dq", "dk", "dv", "d0"), r):
                    out[name] = out[name] + 2.0 ** -25 * x
    return out, u


def _check(lengths, h, hk, dk, dv, dtype, seed=0, state=True, train=True, t=None, scale=None):
    from scree_amd.kernels.hip import varlen_linear_attention_hip

    say(f"case: lengths={lengths if len(lengths) < 12 else len(lengths)} H={h} Hkv={hk} dk={dk} dv={dv} {dtype} "
        f"state={state} train={train}")
    off, cu = cu_of(lengths)
    t = t or _inputs(lengths, h, hk, dk, dv, dtype, seed, state, train)
    s = 1.0 / math.sqrt(dk) if scale is None else scale
    leaves = [t[x].detach().requires_grad_(train) for x in ("q", "k", "v", "s0") if x in t]
    q, k, v = leaves[:3]
    s0 = leaves[3] if state else None
    res = varlen_linear_attention_hip(q, k, v, t["g"], cu, scale=scale, initial_state=s0, return_state=state)
    o, last = res if state else (res, None)
    assert o.dtype == dtype and o.shape == (sum(lengths), h, dv)
    bound, u = _bounds(dtype, lengths, t, s)
    n64 = {x: np64(y) for x, y in t.items()}
    ro, rlast = linear_attention_fwd(n64["q"], n64["k"], n64["v"], n64["g"], off, s, n64.get("s0"))
    check_close("o", np64(o), ro, bound["o"], extra=np.abs(ro), unit=u)
    if state:
        check_close("last", np64(last), rlast, bound["last"] + EPS * np.abs(rlast))
    if not train:
        return o, last
    outs, gs = ((o, last), (t["do"], t["ds"])) if state else ((o,), (t["do"],))
    grads = torch.autograd.grad(outs, leaves, gs)
    want = linear_attention_bwd(n64["do"], n64["q"], n64["k"], n64["v"], n64["g"], off, s, n64.get("s0"), n64.get("ds"))
    for name, got, ref in zip(("dq", "dk", "dv", "d0"), grads, want):
        uu = u if name != "d0" else EPS
        check_close(name, np64(got), ref, bound[name], extra=np.abs(ref), unit=uu)
    return o, last


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", [(8, 8), (32, 32), (64, 64), (96, 40), (128, 128), (64, 128), (128, 32),
                                   (256, 256), (256, 24), (40, 256)])
def test_head_dims(dtype, dk, dv):
    _check(EDGE, 2, 2, dk, dv, dtype, seed=dk + dv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,hk", [(1, 1), (4, 1), (6, 3), (8, 2)])
@pytest.mark.parametrize("state", [False, True])
def test_grouped_heads(dtype, h, hk, state):
    _check([70, 3, 0, 129], h, hk, 32, 64, dtype, seed=h, state=state)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[1500], [700, 0, 1, 300, 256, 257, 1100], [127, 128, 129, 512, 513]])
def test_segmented_sequences(dtype, lengths):
    """Long sequences are walked in several segments (here of 128 tokens)."""
    from scree_amd.kernels.hip.linear_attention import workspace_bytes

    assert workspace_bytes(len(lengths), sum(lengths), 2, 1, 64, 64, False) > 0
    _check(lengths, 2, 1, 64, 64, dtype, seed=7)
    _check(lengths, 2, 2, 32, 96, dtype, seed=8, state=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_and_many_short_sequences(dtype):
    _check([1], 1, 1, 64, 64, dtype)
    rng = np.random.default_rng(1)
    _check([int(x) for x in rng.integers(0, 6, size=150)], 2, 1, 32, 32, dtype, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decays_and_none(dtype):
    t = _inputs([100, 300], 4, 4, 32, 32, dtype, 5, True, True)
    t["g"] = torch.tensor([-40.0, -float("inf"), 0.0, -1e-4]).cuda()
    _check([100, 300], 4, 4, 32, 32, dtype, t=t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_states_past_the_range_of_fp16(dtype):
    """Sums of k v^T of 1e6 and more under small queries: outputs of ordinary size."""
    for h, hk in ((2, 2), (4, 1)):
        t = _inputs([400, 900], h, hk, 64, 64, dtype, 5, True, True)
        t["k"], t["v"] = t["k"] * 20, (t["v"] + 2.0) * 30
        t["q"], t["do"] = t["q"] * 1e-3, t["do"] * 1e-3
        t["g"] = torch.zeros(hk).cuda()
        o, last = _check([400, 900], h, hk, 64, 64, dtype, t=t)
        assert last.abs().max() > 1e5 and torch.isfinite(o).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_views_and_unaligned_inputs(dtype):
    from scree_amd.kernels.hip import varlen_linear_attention_hip

    lengths = [90, 300]
    off, cu = cu_of(lengths)
    qkv = randn((390, 3, 4, 64), dtype, 3)
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    g = _decays(4)
    want = varlen_linear_attention_hip(q.contiguous(), k.contiguous(), v.contiguous(), g, cu)
    assert torch.equal(varlen_linear_attention_hip(q, k, v, g, cu), want)
    flat = randn((390 * 4 * 64 + 1,), dtype, 4)[1:].view(390, 4, 64)  # one element off 16 bytes
    copy = flat.clone()
    assert torch.equal(varlen_linear_attention_hip(flat, k, v, g, cu), varlen_linear_attention_hip(copy, k, v, g, cu))
    out = torch.zeros(390, 64, 4, dtype=dtype, device="cuda").transpose(1, 2)  # head_dim not contiguous
    assert varlen_linear_attention_hip(q, k, v, g, cu, out=out) is out and torch.equal(out, want)
    # gradients through views
    leaf = qkv.clone().requires_grad_(True)
    do = randn((390, 4, 64), dtype, 6)
    o = varlen_linear_attention_hip(leaf[:, 0], leaf[:, 1], leaf[:, 2], g, cu)
    got, = torch.autograd.grad(o, [leaf], [do.transpose(1, 2).contiguous().transpose(1, 2)])
    ls = [t.contiguous().requires_grad_(True) for t in (q, k, v)]
    ref = torch.autograd.grad(varlen_linear_attention_hip(*ls, g, cu), ls, [do])
    assert torch.equal(got, torch.stack(ref, dim=1))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_behind_the_last_sequence(dtype):
    """Left as they were in the output, zero in the gradients; never read."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_linear_attention_hip_backward

    lengths = [40, 300]
    _, cu = cu_of(lengths)
    t = _inputs([40, 300, 60], 4, 2, 64, 64, dtype, 5, False, True)
    for x in ("q", "k", "v", "do"):
        t[x][340:] = float("nan")
    out = torch.full_like(t["do"], 7.0)
    varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, out=out)
    assert (out[340:] == 7.0).all() and torch.isfinite(out[:340]).all()
    short = varlen_linear_attention_hip(t["q"][:340], t["k"][:340], t["v"][:340], t["g"], cu)
    assert torch.equal(out[:340], short)
    for grad in varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu)[:3]:
        assert (grad[340:] == 0).all() and torch.isfinite(grad).all()


def test_prompt_in_parts_and_single_steps():
    """A prompt in one call, in two with the state carried, and token by token."""
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    t = _inputs([9, 9, 9], 4, 2, 64, 96, torch.float32, 11, True, False)
    q, k, v = (t[x].view(3, 9, *t[x].shape[1:]) for x in ("q", "k", "v"))
    _, cu9 = cu_of([9, 9, 9])
    o, last = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu9, initial_state=t["s0"], return_state=True)
    _, cu4 = cu_of([4, 4, 4])
    _, cu5 = cu_of([5, 5, 5])
    part = lambda x, s: x[:, s].reshape(-1, *x.shape[2:])  # noqa: E731
    a, mid = varlen_linear_attention_hip(*[part(x, slice(0, 4)) for x in (q, k, v)], t["g"], cu4,
                                         initial_state=t["s0"], return_state=True)
    b, end = varlen_linear_attention_hip(*[part(x, slice(4, 9)) for x in (q, k, v)], t["g"], cu5,
                                         initial_state=mid, return_state=True)
    two = torch.cat([a.view(3, 4, 4, 96), b.view(3, 5, 4, 96)], dim=1).view(27, 4, 96)
    state = t["s0"].clone()
    steps = torch.stack([linear_attention_step_hip(q[:, i], k[:, i], v[:, i], t["g"], state) for i in range(9)], 1)
    bound, _ = _bounds(torch.float32, [9, 9, 9], t, 0.125)
    for name, got, ref in (("two calls", two, o), ("steps", steps.view(27, 4, 96), o)):
        check_close(name, np64(got), np64(ref), 2 * bound["o"] + 2 * EPS * np.abs(np64(ref)))
    for name, got in (("state of two calls", end), ("state of steps", state)):
        check_close(name, np64(got), np64(last), 2 * bound["last"] + 2 * EPS * np.abs(np64(last)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,dk,dv", [(1, 1, 1, 8, 8), (3, 4, 2, 64, 64), (2, 8, 1, 128, 40), (5, 2, 2, 256, 256),
                                          (1, 16, 16, 128, 128), (70, 6, 3, 96, 32)])
def test_step(dtype, b, h, hk, dk, dv):
    from scree_amd.kernels.hip import linear_attention_step_hip

    say(f"case: step b={b} H={h} Hkv={hk} dk={dk} dv={dv} {dtype}")
    t = _inputs([1] * b, h, hk, dk, dv, dtype, 2, True, False)
    n64 = {x: np64(y) for x, y in t.items()}
    off = np.arange(b + 1)
    s = 1.0 / math.sqrt(dk)
    ro, rs = linear_attention_fwd(n64["q"], n64["k"], n64["v"], n64["g"], off, s, n64["s0"])
    ab = {x: np.abs(y) for x, y in n64.items()}
    bo, bs = linear_attention_fwd(ab["q"], ab["k"], ab["v"], n64["g"], off, s, ab["s0"])
    # fp32 throughout: a state's two products and lam (2 |log lam| + 2 roundings), dk of a dot
    pool = torch.full((b, hk * dk * dv + 8), 5.0, device="cuda")
    rows = pool[:, 4:4 + hk * dk * dv].view(b, hk, dk, dv)
    rows.copy_(t["s0"])
    new = torch.empty_like(t["s0"])
    o = linear_attention_step_hip(t["q"], t["k"], t["v"], t["g"], rows, state_out=new)
    assert torch.equal(rows, t["s0"])
    check_close("state", np64(new), rs, 6 * EPS * bs)
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0
    check_close("o", np64(o), ro, (dk + 16) * EPS * bo + small, extra=np.abs(ro), unit=u)
    assert torch.equal(linear_attention_step_hip(t["q"], t["k"], t["v"], t["g"], rows), o)  # in place
    assert torch.equal(rows, new) and (pool[:, :4] == 5).all() and (pool[:, 4 + hk * dk * dv:] == 5).all()


def test_no_tokens():
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    x = torch.empty((0, 2, 64), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    _, cu = cu_of([0, 0])
    g = _decays(2)
    s0 = randn((2, 2, 64, 64), torch.float32, 1).requires_grad_(True)
    o, last = varlen_linear_attention_hip(x, x, x, g, cu, initial_state=s0, return_state=True)
    assert o.shape == (0, 2, 64) and torch.equal(last, s0)
    d0, dx = torch.autograd.grad([last], [s0, x], [s0.detach() * 2])
    assert torch.equal(d0, s0 * 2) and dx.shape == x.shape
    with torch.no_grad():
        assert linear_attention_step_hip(x, x, x, g, s0[:0]).shape == (0, 2, 64)


def test_refusals_on_the_device():
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    _, cu = cu_of([4, 6])
    t = _inputs([4, 6], 4, 2, 64, 32, torch.float16, 1, True, False)
    base = {"q": t["q"], "k": t["k"], "v": t["v"], "log_decay": t["g"], "cu_seqlens": cu}
    for bad in (dict(q=t["q"][:, :3]), dict(q=t["q"][:5]), dict(v=t["v"][..., :20]), dict(q=t["q"].float()),
                dict(log_decay=t["g"].double()), dict(log_decay=t["g"][:1]), dict(log_decay=t["g"].cpu()),
                dict(initial_state=t["s0"][:1]), dict(initial_state=t["s0"].half()), dict(out=t["q"]),
                dict(cu_seqlens=cu[:1]), dict(k=t["k"].double(), q=t["q"].double(), v=t["v"].double())):
        with pytest.raises(AssertionError):
            varlen_linear_attention_hip(**{**base, **bad})
    with pytest.raises(NotImplementedError, match="log_decay"):
        varlen_linear_attention_hip(**{**base, "log_decay": t["g"].clone().requires_grad_(True)})
    q, k, v = t["q"][:2], t["k"][:2], t["v"][:2]
    for state in (t["s0"].half(), t["s0"].transpose(2, 3), t["s0"][:1], t["s0"][:1].expand(2, -1, -1, -1),
                  t["s0"].clone().requires_grad_(True)):
        with pytest.raises(AssertionError):
            linear_attention_step_hip(q, k, v, t["g"], state)


def test_array_level_and_explicit_backward():
    from scree_amd.kernels import varlen_linear_attention
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_linear_attention_hip_backward

    lengths = [30, 0, 100]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 2, 64, 64, torch.bfloat16, 5, True, True)
    arrs = [scree_amd.Array(values=t[x], offsets=cu) for x in ("q", "k", "v")]
    o, last = varlen_linear_attention(*arrs, t["g"], initial_state=t["s0"], return_state=True)
    ro, rlast = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"], return_state=True)
    assert o.offsets is cu and torch.equal(o.values, ro) and torch.equal(last, rlast)
    leaves = [t[x].clone().requires_grad_(True) for x in ("q", "k", "v", "s0")]
    out = varlen_linear_attention_hip(*leaves[:3], t["g"], cu, initial_state=leaves[3], return_state=True)
    want = torch.autograd.grad(out, leaves, (t["do"], t["ds"]))
    got = varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu,
                                               initial_state=t["s0"], dstate=t["ds"])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    other = scree_amd.Array(values=t["k"], offsets=cu_of([31, 0, 99])[1])
    with pytest.raises(ValueError, match="offsets"):
        varlen_linear_attention(arrs[0], other, arrs[2], t["g"])


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 128)])  # below and past 64 KB of LDS
def test_graph_replays_match_eager_without_host_sync(dtype, dim):
    from scree_amd.kernels.hip import varlen_linear_attention_hip_backward, varlen_linear_attention_hip

    lengths = [700, 33]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 2, dim, dim, dtype, 9, True, True)

    def step():
        o, last = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"],
                                              return_state=True)
        return (o, last, *varlen_linear_attention_hip_backward(
            t["do"], t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"], dstate=t["ds"]))

    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    step()
    torch.cuda.set_sync_debug_mode("default")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        t["q"].copy_(randn(tuple(t["q"].shape), dtype, 90 + seed))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_past_2_31_elements(dtype):
    """Row strides up to the limit of 2^24 elements: places past 2^31."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_linear_attention_hip_backward

    lengths, stride = [3, 127], (1 << 24) - 8
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 2, 2, 64, 64, dtype, 5, False, True)
    far = torch.empty((130 * stride,), dtype=dtype, device="cuda")
    far_t = {}
    for i, x in enumerate(("q", "k", "v", "do")):
        far_t[x] = far.as_strided((130, 2, 64), (stride, 64, 1), 1024 * i)
        far_t[x].copy_(t[x])
    out = far.as_strided((130, 2, 64), (stride, 64, 1), 4096)
    varlen_linear_attention_hip(far_t["q"], far_t["k"], far_t["v"], t["g"], cu, out=out)
    assert torch.equal(out, varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu))
    got = varlen_linear_attention_hip_backward(far_t["do"], far_t["q"], far_t["k"], far_t["v"], t["g"], cu)
    want = varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a, b)


def test_offsets_that_do_not_ascend_stay_inside_the_tensors():
    """Clamped to [0, total]; what comes out is not specified."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_linear_attention_hip_backward

    for offsets in ([0, 300, 100, 400], [0, -7, 900, 400], [250, 0, 0, 400], [400, 400, 400, 0]):
        say(f"case: offsets {offsets}")
        cu = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        t = _inputs([400], 4, 2, 64, 64, torch.bfloat16, 5, False, True)
        s0 = randn((3, 2, 64, 64), torch.float32, 6)
        room = torch.full((600, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=s0, return_state=True,
                                    out=room[100:500])
        varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu, initial_state=s0, dstate=s0)
        torch.cuda.synchronize()
        assert (room[:100] == 7).all() and (room[500:] == 7).all()


def test_non_finite_values_stay_in_their_sequence_and_head():
    from scree_amd.kernels.hip import varlen_linear_attention_hip, varlen_linear_attention_hip_backward

    lengths = [200, 90, 300]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 2, 64, 64, torch.bfloat16, 5, False, True)
    t["v"][250, 1, 3], t["k"][260, 1, 5] = float("nan"), float("inf")
    o = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu)
    grads = varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu)[:3]
    hit = torch.zeros(590, dtype=torch.bool, device="cuda")
    hit[200:290] = True
    assert torch.isnan(o[250:290, 2:, 3]).all()
    for x in (o, *grads):
        half = x.shape[1] // 2
        assert torch.isfinite(x[~hit]).all() and torch.isfinite(x[:, :half]).all()


def test_backward_twice_and_broadcast_heads():
    """A retained graph gives the same gradients again; K/V heads expanded from
    one sum theirs."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip

    lengths = [500, 40]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 4, 64, 64, torch.float32, 5, False, True)
    one = [t[x][:, :1].clone().requires_grad_(True) for x in ("k", "v")]
    q = t["q"].clone().requires_grad_(True)
    g = torch.full((4,), -0.1, device="cuda")
    o = varlen_linear_attention_hip(q, *[x.expand(-1, 4, -1) for x in one], g, cu)
    first = torch.autograd.grad(o, [q, *one], t["do"], retain_graph=True)
    for a, b in zip(first, torch.autograd.grad(o, [q, *one], t["do"])):
        assert torch.equal(a, b)
    # against four query heads on one K/V head
    o1 = varlen_linear_attention_hip(q, *one, g[:1], cu)
    assert torch.equal(o, o1)
    want = torch.autograd.grad(o1, [q, *one], t["do"])
    bound, _ = _bounds(torch.float32, lengths, {**t, "k": t["k"][:, :1], "v": t["v"][:, :1], "g": g[:1]}, 0.125)
    for name, a, b in zip(("dq", "dk", "dv"), first, want):
        check_close(name, np64(a), np64(b), 2 * bound[name] + 8 * EPS * np.abs(np64(b)))


def test_on_another_stream():
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    lengths = [300, 40]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 2, 64, 64, torch.bfloat16, 5, True, True)
    want = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"], return_state=True)
    step = linear_attention_step_hip(t["q"][:2], t["k"][:2], t["v"][:2], t["g"], t["s0"].clone())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"], return_state=True)
        got_step = linear_attention_step_hip(t["q"][:2], t["k"][:2], t["v"][:2], t["g"], t["s0"].clone())
    side.synchronize()
    for a, b in zip((*got, got_step), (*want, step)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,rows,h,hk,d", [([300], 20000, 4, 2, 64), ([9000, 1, 0], 9001 + 40, 8, 1, 128),
                                                 ([0, 0], 5000, 2, 2, 32), ([5000], 9000, 32, 8, 64)])
def test_long_tails_become_zeros_in_the_gradients(dtype, lengths, rows, h, hk, d):
    """Fewer rows than a segment behind the last sequence, and many segments' worth."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip_backward

    n = sum(lengths)
    _, cu = cu_of(lengths)
    t = _inputs([rows], h, hk, d, d, dtype, 5, False, True)
    for x in ("q", "k", "v", "do"):
        t[x][n:] = float("nan")
    junk = torch.full((4 * rows, h, d), float("nan"), device="cuda")  # what the gradients' memory held
    del junk
    grads = varlen_linear_attention_hip_backward(t["do"], t["q"], t["k"], t["v"], t["g"], cu)[:3]
    for grad in grads:
        assert (grad[n:] == 0).all() and torch.isfinite(grad).all()


def test_an_infinite_state_column_stays_alone():
    """An infinity in one column of an fp16 walk's state leaves the others' values."""
    from scree_amd.kernels.hip import varlen_linear_attention_hip

    lengths = [150, 20]
    _, cu = cu_of(lengths)
    t = _inputs(lengths, 4, 2, 64, 64, torch.float16, 5, True, False)
    want, last = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=t["s0"], return_state=True)
    s0 = t["s0"].clone()
    s0[0, 1, 7, 5] = float("inf")
    o, got = varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, initial_state=s0, return_state=True)
    others = [c for c in range(64) if c != 5]
    assert torch.equal(o[..., others], want[..., others]) and torch.equal(got[..., others], last[..., others])
    assert not torch.isfinite(o[:150, 2:, 5]).any() and torch.equal(o[:, :2], want[:, :2])


def test_in_place_writes_are_seen_by_autograd():
    """A state or output that a recorded graph still needs is not changed unseen;
    a second derivative is refused."""
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    _, cu = cu_of([5, 3])
    t = _inputs([5, 3], 4, 2, 64, 32, torch.float32, 1, True, True)
    q = t["q"].clone().requires_grad_(True)
    o = varlen_linear_attention_hip(q, t["k"], t["v"], t["g"], cu, initial_state=t["s0"])
    with torch.no_grad():
        linear_attention_step_hip(t["q"][:2], t["k"][:2], t["v"][:2], t["g"], t["s0"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    w = torch.ones_like(t["do"], requires_grad=True)
    buf = torch.empty_like(t["do"])
    y = w * buf
    varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(AssertionError, match="expanded"):
        varlen_linear_attention_hip(t["q"], t["k"], t["v"], t["g"], cu, out=buf[:, :1].expand(-1, 4, -1))
    grad, = torch.autograd.grad(varlen_linear_attention_hip(q, t["k"], t["v"], t["g"], cu).sum(), [q], create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivative"):
        grad.sum().backward()
    with torch.inference_mode():
        s = t["s0"].clone()
        linear_attention_step_hip(t["q"][:2], t["k"][:2], t["v"][:2], t["g"], s)
        assert torch.equal(s, t["s0"]) is False
