"""GPU parity of the token log probabilities, forward and backward.

The oracle runs in fp64 on the rounded logits.  Bounds, in units of
``e = 2^-24``: a thread adds up to ``vocab / 256 + 8`` positive terms one after
the other and ten more levels join the threads, each with a rounding of the
sum (and, when the maximum rises, of the factor); exp of ``d = x - m`` is off
by ``(1.5 |d| + 2) e`` of itself, and terms with ``|d| > 30`` carry less than
``1e-8`` of a sum.  So ``s`` is off by ``E = (vocab / 256 + 80) e`` of itself,
``t`` by ``E`` of ``sum p |d|``, logprob by ``E + 2 e (|x_y - m| + ln s)``
and the entropy by ``E (1 + 2 sum p |d|) + 2 e (ln s + sum p |d|)``.  p_j in
the backward is off by ``(1.5 |d_j| + 6) e + E`` of itself; the gradient in a 16-bit
type adds its rounding, ``u`` of itself (and half the smallest subnormal).
exp flushes results below ``2^-126`` to zero, so p_j loses up to that much,
times its factor ``|g| + sum |gtop| + |gH| (|lp_j| + entropy)``.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import scree_amd
from oracle.logprobs import _log_softmax, token_logprobs, token_logprobs_bwd
from parity import UNIT, cu_of, np64, randn, say

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def _within(name, got, want, bound):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=name)
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf], err_msg=name)
    ok = np.isfinite(want)
    over = np.abs(got[ok] - want[ok]) - np.broadcast_to(bound, want.shape)[ok]
    say(f"  {name}: margin {-over.max() if over.size else 0:.3e}")
    assert not over.size or over.max() <= 0, f"{name}: exceeds its bound by {over.max():.3e}"


def _check(x, y, top_k, grads=None, backward=True):
    """Forward and backward of device logits ``x`` against the oracle."""
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    n, v = x.shape
    say(f"case: rows={n} vocab={v} top_k={top_k} {x.dtype} strides={x.stride()}")
    x64, yn = np64(x), y.cpu().numpy()
    leaf = x.detach().requires_grad_(backward)
    out = varlen_token_logprobs_hip(leaf, y, top_k)
    lp, ent, top, idx = token_logprobs(x64, yn, top_k)
    every = _log_softmax(x64)
    with np.errstate(all="ignore"):
        d = x64 - x64.max(axis=1, keepdims=True)
        p = np.exp(every)
        spd = np.where(p > 0, p * np.abs(d), 0.0).sum(axis=1)
    ls = np.log(v)
    E = (v / 256 + 80) * EPS
    _within("logprob", np64(out.logprob), lp, E + 2 * EPS * (np.abs(np.nan_to_num(lp)) + 2 * ls))
    _within("entropy", np64(out.entropy), ent, E * (1 + 2 * spd) + 2 * EPS * (ls + spd))
    assert out.logprob.dtype == out.entropy.dtype == torch.float32
    if top_k:
        bad = np.isnan(x64).any(axis=1)  # a row with NaN names no particular alternatives
        got_i = out.top_index.cpu().numpy()
        assert out.top_index.dtype == torch.int64 and (got_i >= 0).all() and (got_i < v).all()
        np.testing.assert_array_equal(got_i[~bad], idx[~bad])
        _within("top_logprob", np64(out.top_logprob)[~bad], top[~bad],
                E + 2 * EPS * (np.abs(np.nan_to_num(top[~bad])) + 2 * ls))
    else:
        assert out.top_logprob is None and out.top_index is None
    if not backward:
        return out
    if grads is None:
        grads = [randn((n,), torch.float32, 71), randn((n,), torch.float32, 72),
                 randn((n, top_k), torch.float32, 73) if top_k else None]
    outs = [o for o, g in zip(out[:3], grads) if g is not None]
    dx, = torch.autograd.grad(outs, [leaf], [g for g in grads if g is not None])
    assert dx.dtype == x.dtype and dx.shape == x.shape
    g64 = [None if g is None else np64(g) for g in grads]
    want = token_logprobs_bwd(x64, yn, *g64)
    size = np.abs(g64[0] if g64[0] is not None else 0)[..., None] if g64[0] is not None else 0.0
    if g64[2] is not None:
        size = size + np.abs(g64[2]).sum(axis=1)[:, None]
    gh = np.abs(g64[1])[:, None] if g64[1] is not None else 0.0
    with np.errstate(all="ignore"):
        lpa = np.where(p > 0, np.abs(every), 0.0)
        da = np.where(p > 0, np.abs(d), 0.0)
        bound = p * (size + gh * (lpa + ls)) * ((1.5 * da + 10) * EPS + E) + p * gh * (E * (1 + 2 * spd[:, None]) + 4 * EPS * ls)
        bound = bound + 4 * EPS * np.abs(want)  # the single columns' own sums
        bound = bound + 2.0 ** -126 * (size + gh * (lpa + ls))
    u = 0.0 if x.dtype == torch.float32 else UNIT[x.dtype]
    _within("dlogits", np64(dx), want, np.nan_to_num(bound) + u * np.abs(np.nan_to_num(want)) + TINY[x.dtype])
    return out


def _logits(n, v, dtype, seed, scale=3.0):
    x = randn((n, v), dtype, seed, scale=scale)
    y = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(seed)).cuda()
    return x, y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top_k", [(1, 1), (2, 0), (7, 7), (8, 3), (63, 20), (64, 64), (65, 1),
                                         (515, 64), (4097, 5), (20011, 20)])
def test_vocabularies(dtype, vocab, top_k):
    x, y = _logits(5, vocab, dtype, vocab)
    _check(x, y, top_k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 64, 1100])
def test_split_and_whole_rows(dtype, rows):
    """1 to 64 rows are split over workgroups and joined; 1,100 are not."""
    x, y = _logits(rows, 9001, dtype, rows)
    _check(x, y, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_int32_targets(dtype):
    wide = randn((9, 1040), dtype, 3, scale=3.0)
    y = torch.arange(9, dtype=torch.int32, device="cuda") * 100
    for cols in (slice(0, 1000), slice(1, 1002), slice(3, 1030)):  # rows at odd addresses
        view = wide[:, cols]
        assert view.stride(0) == 1040
        _check(view, y, 6)
    _check(wide[::2, 5:900], y[::2], 2)
    _check(wide.t()[:9, :9], y.clamp(max=8), 2)  # last axis not contiguous: copied


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [300, 33000])
def test_ties_take_the_lowest_index(dtype, vocab):
    x, y = _logits(4, vocab, dtype, 8)
    x[0] = 0.5                                # every logit equal
    x[1] = torch.randint(0, 3, (vocab,), generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    x[2, ::2], x[2, 1::2] = 0.0, -0.0         # signed zeros are equal
    x[3] = torch.arange(vocab, device="cuda").to(dtype)  # rising: every element beats the list
    _check(x, y, 40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 40000])
def test_masked_and_non_finite_logits(dtype, vocab):
    x, y = _logits(10, vocab, dtype, 21)
    keep = torch.rand((vocab,), generator=torch.Generator().manual_seed(2)).cuda() < 0.05
    x[0].masked_fill_(~keep, -float("inf"))                 # nine tenths ruled out
    x[1] = -float("inf")
    x[1, vocab // 2] = 1.0                                  # one logit left
    x[2].masked_fill_(~keep, torch.finfo(dtype).min)        # masked with the type's lowest value
    x[3] = torch.finfo(dtype).min                           # ... throughout: uniform
    x[4] = -float("inf")                                    # nothing left: NaN
    x[5, 17] = float("nan")
    x[6, vocab - 1] = float("inf")
    x[7, y[7]] = -float("inf")                              # the target itself ruled out
    x[8] = torch.finfo(dtype).max
    y[1] = vocab // 2
    out = _check(x, y, 10)
    assert torch.isnan(out.logprob[4:7]).all() and out.logprob[7] == -float("inf")
    assert out.logprob[1] == 0 and out.entropy[1] == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_target(dtype):
    x, y = _logits(6, 5000, dtype, 4)
    y[0], y[1], y[2] = -100, -1, 5000
    x[1] = -float("inf")  # a padding row with no logits left
    g = randn((6,), torch.float32, 5)
    # with the log probability's gradient alone, rows without a target get zeros
    _check(x, y, 3, grads=[g, None, None])
    _check(x[2:], y[2:], 3, grads=[None, g[2:], None])
    _check(x[2:], y[2:], 3, grads=[None, None, randn((4, 3), torch.float32, 6)])
    _check(x[3:], y[3:], 3, grads=[torch.zeros(3, device="cuda"), None, None])


def test_target_among_the_alternatives():
    x, _ = _logits(4, 600, torch.float32, 9)
    _check(x, x.argmax(dim=1), 5)


def test_no_rows():
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    x = torch.empty((0, 100), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = varlen_token_logprobs_hip(x, torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert out.logprob.shape == (0,) and out.top_index.shape == (0, 3)
    dx, = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), [x])
    assert dx.shape == x.shape


def test_array_level_and_explicit_backward():
    from scree_amd.kernels import varlen_token_logprobs
    from scree_amd.kernels.hip import varlen_token_logprobs_hip, varlen_token_logprobs_hip_backward

    off, cu = cu_of([3, 0, 5, 1])
    x, y = _logits(9, 777, torch.bfloat16, 14)
    arr = scree_amd.Array(values=x, offsets=cu)
    out = varlen_token_logprobs(arr, scree_amd.Array(values=y, offsets=cu), top_k=2)
    flat = varlen_token_logprobs_hip(x, y, 2)
    for a, b in zip(out, flat):
        assert a.offsets is cu and torch.equal(a.values, b)
    with pytest.raises(ValueError, match="offsets"):
        varlen_token_logprobs(arr, scree_amd.Array(values=y, offsets=cu_of([2, 1, 5, 1])[1]))
    g = [randn((9,), torch.float32, 1), randn((9,), torch.float32, 2), randn((9, 2), torch.float32, 3)]
    leaf = x.clone().requires_grad_(True)
    res = varlen_token_logprobs_hip(leaf, y, 2)
    want, = torch.autograd.grad(res[:3], [leaf], g)
    assert torch.equal(varlen_token_logprobs_hip_backward(x, y, *g, top_k=2), want)


def test_refusals_on_the_device():
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    x, y = _logits(4, 50, torch.float16, 1)
    for bad in (dict(targets=y[:3]), dict(targets=y.float()), dict(targets=y.cpu()), dict(top_k=51),
                dict(top_k=65), dict(top_k=-1), dict(logits=x[None]), dict(logits=x.double())):
        args = {"logits": x, "targets": y, "top_k": 0, **bad}
        with pytest.raises(AssertionError):
            varlen_token_logprobs_hip(**args)


def test_gradients_on_the_host_and_second_derivatives_are_refused():
    from scree_amd.kernels.hip import varlen_token_logprobs_hip, varlen_token_logprobs_hip_backward

    x, y = _logits(4, 50, torch.float32, 1)
    for name, shape in (("dlogprob", (4,)), ("dentropy", (4,)), ("dtop_logprob", (4, 2))):
        with pytest.raises(AssertionError, match="same device"):
            varlen_token_logprobs_hip_backward(x, y, top_k=2, **{name: torch.zeros(shape)})
    leaf = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(varlen_token_logprobs_hip(leaf, y).logprob.sum(), [leaf], create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivative"):
        grad.sum().backward()


def test_graph_replays_match_eager_without_host_sync():
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    x, y = _logits(20, 30000, torch.bfloat16, 2)
    g = [randn((20,), torch.float32, 1), randn((20,), torch.float32, 2), randn((20, 8), torch.float32, 3)]
    buf = x.clone().requires_grad_(True)

    def step():
        out = varlen_token_logprobs_hip(buf, y, 8)
        dx, = torch.autograd.grad(out[:3], [buf], g)
        return tuple(t.detach() for t in out) + (dx,)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda.set_sync_debug_mode("error")
        step()
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            buf.copy_(randn((20, 30000), torch.bfloat16, 90 + seed, scale=3.0))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


def test_rows_past_2_31_elements():
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    small, y = _logits(3, 5000, torch.bfloat16, 12)
    far = torch.empty((2 * ((1 << 30) + 3) + 5000,), dtype=torch.bfloat16, device="cuda")
    view = far.as_strided((3, 5000), ((1 << 30) + 3, 1))
    view.copy_(small)
    for a, b in zip(varlen_token_logprobs_hip(view, y, 7), varlen_token_logprobs_hip(small, y, 7)):
        assert torch.equal(a, b)
    g = randn((3,), torch.float32, 1)
    leaf, near = view.detach().requires_grad_(True), small.clone().requires_grad_(True)
    got, = torch.autograd.grad(varlen_token_logprobs_hip(leaf, y).logprob, [leaf], g)
    want, = torch.autograd.grad(varlen_token_logprobs_hip(near, y).logprob, [near], g)
    assert torch.equal(got, want)


def test_large_logits_take_streaming_loads():
    """Past 256 MB the loads change; 70,000 rows of 4,001 fp16 are 560 MB."""
    from scree_amd.kernels.hip import varlen_token_logprobs_hip

    x = torch.randn((70000, 4001), device="cuda", dtype=torch.float16)
    y = torch.randint(0, 4001, (70000,), device="cuda")
    leaf = x.requires_grad_(True)
    out = varlen_token_logprobs_hip(leaf, y, 3)
    g = torch.randn(70000, device="cuda")
    dx, = torch.autograd.grad(out.logprob, [leaf], g)
    rows = slice(40000, 40007)
    part = x.detach()[rows].clone().requires_grad_(True)
    want = varlen_token_logprobs_hip(part, y[rows], 3)
    # the same sums in another order (few rows are split): both within E of exact
    E = (4001 / 256 + 80) * EPS
    assert torch.equal(out.top_index[rows], want.top_index)
    assert (out.logprob[rows] - want.logprob).abs().max() <= 2 * (E + 2 * EPS * 30)
    dw, = torch.autograd.grad(want.logprob, [part], g[rows])
    # each is one rounding of values E apart: 2 u and 2 E of themselves, and a subnormal's step
    assert ((dx[rows].float() - dw.float()).abs() <= 2 * (2.0 ** -11 + E) * dw.float().abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype,trip", [(torch.bfloat16, 8192), (torch.float32, 4096)])
@pytest.mark.parametrize("top_k", [1, 20, 64])
def test_rows_of_one_trip_and_a_little_more(dtype, trip, top_k):
    """Alternatives are ranked at once in rows of up to a trip of the workgroup,
    kept in lists beyond; more than 64 candidates to a wave, and in the last columns."""
    for vocab in (trip - 1, trip, trip + 3, trip + 200):
        x, y = _logits(8, vocab, dtype, vocab + top_k)
        x[1] = 2.0                                   # all equal
        x[2] = -float("inf")
        x[2, vocab - 3:] = torch.arange(3, dtype=dtype, device="cuda")   # the last columns alone
        y[2] = vocab - 1
        x[3, : vocab // 2] = 9.0                     # thousands of largest ones
        x[4, ::64] = 9.0
        x[5] = torch.sort(x[5].float()).values.to(dtype)
        x[6] = torch.sort(x[6].float(), descending=True).values.to(dtype)
        x[7, vocab - 1] = 50.0
        _check(x, y, top_k)
        # whole rows to a workgroup give the same
        many = x.repeat(160, 1)
        from scree_amd.kernels.hip import varlen_token_logprobs_hip
        a, b = varlen_token_logprobs_hip(x, y, top_k), varlen_token_logprobs_hip(many, y.repeat(160), top_k)
        assert torch.equal(b.top_index, a.top_index.repeat(160, 1))
