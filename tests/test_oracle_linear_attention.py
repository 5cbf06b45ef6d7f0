"""The linear attention oracle: its forward against the sum it stands for, its
gradients against torch autograd and differences; host refusals (no GPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle.linear_attention import linear_attention_bwd, linear_attention_fwd
from scree_amd.kernels.hip import _ffi

OFF = np.array([0, 5, 5, 6, 13], dtype=np.int32)


def _case(h, hk, dk, dv, seed=0):
    rng = np.random.default_rng(seed)
    n, b = int(OFF[-1]), len(OFF) - 1
    r = lambda *s: rng.normal(size=s)  # noqa: E731
    return (r(n, h, dk), r(n, hk, dk), r(n, hk, dv), -np.abs(r(hk)) * 0.3, r(b, hk, dk, dv),
            r(n, h, dv), r(b, hk, dk, dv))


@pytest.mark.parametrize("h,hk,dk,dv", [(2, 2, 4, 4), (6, 2, 3, 5)])
def test_forward_is_the_decayed_sum(h, hk, dk, dv):
    q, k, v, g, s0, _, _ = _case(h, hk, dk, dv)
    o, last = linear_attention_fwd(q, k, v, g, OFF, 0.7, s0)
    for b in range(len(OFF) - 1):
        rows = range(OFF[b], OFF[b + 1])
        for i, t in enumerate(rows):
            for hq in range(h):
                j = hq // (h // hk)
                want = np.exp(g[j] * (i + 1)) * (q[t, hq] @ s0[b, j])
                want = want + sum(np.exp(g[j] * (t - s)) * (q[t, hq] @ k[s, j]) * v[s, j]
                                  for s in range(OFF[b], t + 1))
                np.testing.assert_allclose(o[t, hq], 0.7 * want, atol=1e-12)
    np.testing.assert_allclose(last[1], s0[1])  # the empty sequence passes its state on


def test_gradients_against_autograd():
    q, k, v, g, s0, do, ds = _case(4, 2, 3, 5, 1)
    got = linear_attention_bwd(do, q, k, v, g, OFF, 0.7, s0, ds)
    leaves = [torch.from_numpy(t).requires_grad_(True) for t in (q, k, v, s0)]
    tq, tk, tv, ts = leaves
    lam = torch.from_numpy(np.exp(g))[:, None, None]
    loss = 0.0
    for b in range(len(OFF) - 1):
        s = ts[b]
        for t in range(OFF[b], OFF[b + 1]):
            s = lam * s + tk[t][:, :, None] * tv[t][:, None, :]
            o = 0.7 * torch.matmul(tq[t].reshape(2, 2, 3), s).reshape(4, 5)
            loss = loss + (o * torch.from_numpy(do[t])).sum()
        loss = loss + (s * torch.from_numpy(ds[b])).sum()
    for a, b in zip(got, torch.autograd.grad(loss, leaves)):
        np.testing.assert_allclose(a, b.numpy(), atol=1e-11)


def test_gradients_against_differences():
    args = _case(2, 1, 3, 2, 2)
    q, k, v, g, s0, do, ds = args
    got = linear_attention_bwd(do, q, k, v, g, OFF, 0.7, s0, ds)

    def loss(q, k, v, s0):
        o, last = linear_attention_fwd(q, k, v, g, OFF, 0.7, s0)
        return (o * do).sum() + (last * ds).sum()

    leaves = [q, k, v, s0]
    for i, grad in enumerate(got):
        for at in np.ndindex(grad.shape):
            up = [t.copy() for t in leaves]
            dn = [t.copy() for t in leaves]
            up[i][at] += 1e-4
            dn[i][at] -= 1e-4
            # the loss is linear in every single element: differences are exact but for rounding
            assert abs((loss(*up) - loss(*dn)) / 2e-4 - grad[at]) < 1e-9


def test_launcher_refusals():
    import scree_amd
    from scree_amd.kernels import varlen_linear_attention
    from scree_amd.kernels.hip import linear_attention_step_hip, varlen_linear_attention_hip

    x = torch.zeros(4, 2, 32)
    g, cu = torch.zeros(2), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(AssertionError, match="ROCm"):
        varlen_linear_attention_hip(x, x, x, g, cu)
    with pytest.raises(AssertionError, match="ROCm"):
        linear_attention_step_hip(x, x, x, g, torch.zeros(4, 2, 32, 32))
    arr = scree_amd.pack([np.zeros((3, 2, 32), dtype=np.float32)])
    with pytest.raises(TypeError, match="ROCm"):
        varlen_linear_attention(arr, arr, arr, g)


def test_c_abi_refusals():
    lib = _ffi.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    p, null = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16), ctypes.c_void_p(0)
    odd = ctypes.c_void_p(p.value + 4)
    err = lambda: lib.scree_last_error().decode()  # noqa: E731
    st = _ffi.int64_array([4 * 64, 64] * 7)

    def fwd(q=p, g=p, o=p, s0=null, s1=null, cu=p, b=2, n=10, h=4, hk=4, dk=64, dv=64, strides=st,
            dtype=1, ws=null, nws=0):
        return lib.scree_linear_attn_fwd(q, p, p, g, o, s0, s1, cu, b, n, h, hk, dk, dv, strides, 1.0,
                                         dtype, ws, nws, null)

    assert fwd(n=0, q=null) == _ffi.SCREE_OK
    for bad, code, text in [
            (dict(q=null), _ffi.SCREE_ERR_INVALID, "q is null"),
            (dict(o=odd), _ffi.SCREE_ERR_INVALID, "aligned"),
            (dict(s1=odd), _ffi.SCREE_ERR_INVALID, "aligned"),
            (dict(g=null), _ffi.SCREE_ERR_INVALID, "log_decay"),
            (dict(cu=null), _ffi.SCREE_ERR_INVALID, "cu_seqlens"),
            (dict(b=0), _ffi.SCREE_ERR_UNSUPPORTED, "batch"),
            (dict(n=-1), _ffi.SCREE_ERR_INVALID, "total_tokens"),
            (dict(n=(1 << 30) + 1), _ffi.SCREE_ERR_INVALID, "total_tokens"),
            (dict(hk=3), _ffi.SCREE_ERR_INVALID, "kv_heads"),
            (dict(hk=0), _ffi.SCREE_ERR_INVALID, "kv_heads"),
            (dict(dk=60), _ffi.SCREE_ERR_UNSUPPORTED, "head_dim"),
            (dict(dv=264), _ffi.SCREE_ERR_UNSUPPORTED, "head_dim"),
            (dict(dtype=5), _ffi.SCREE_ERR_UNSUPPORTED, "dtype"),
            (dict(strides=_ffi.int64_array([4 * 64 + 4, 64] * 7)), _ffi.SCREE_ERR_INVALID, "strides"),
            (dict(strides=_ffi.int64_array([32, 64] * 7)), _ffi.SCREE_ERR_INVALID, "overlaps"),
            (dict(n=100000), _ffi.SCREE_ERR_WORKSPACE, "workspace"),
            (dict(n=100000, ws=p, nws=1 << 12), _ffi.SCREE_ERR_WORKSPACE, "workspace")]:
        assert fwd(**bad) == code and text in err(), (bad, err())
    need = lib.scree_linear_attn_workspace_bytes(2, 100000, 4, 4, 64, 64, 0)
    assert need > 0 and lib.scree_linear_attn_workspace_bytes(2, 100000, 4, 4, 64, 64, 1) == 2 * need
    assert lib.scree_linear_attn_workspace_bytes(2, 100, 4, 4, 64, 64, 1) == 0
    # a small batch of short sequences is walked whole
    assert lib.scree_linear_attn_workspace_bytes(16, 1980, 4, 4, 32, 32, 1) == 0

    def bwd(dv=p, fwd=null, n=10, scale=1.0, ws=null, nws=0):
        return lib.scree_linear_attn_bwd(p, p, p, p, p, p, p, dv, null, null, null, fwd, p, 2, n, 4, 4, 64, 64,
                                         st, scale, 1, ws, nws, null)

    assert bwd(dv=null) == _ffi.SCREE_ERR_INVALID and "dv is null" in err()
    assert bwd(fwd=odd) == _ffi.SCREE_ERR_INVALID and "aligned" in err()
    for scale in (0.0, float("nan"), float("inf"), 1e-40):
        assert bwd(scale=scale) == _ffi.SCREE_ERR_INVALID and "scale" in err()
    # the forward's states at hand, half the room is enough
    assert bwd(n=100000, ws=p, nws=2 * need - 1) == _ffi.SCREE_ERR_WORKSPACE
    assert bwd(n=100000, ws=p, nws=need - 1, fwd=p) == _ffi.SCREE_ERR_WORKSPACE
    rows = _ffi.int64_array([256, 64] * 4 + [4 * 64 * 64, 4 * 64 * 64 - 4])
    rc = lib.scree_linear_attn_step(p, p, p, p, p, p, p, 2, 4, 4, 64, 64, rows, 1.0, 1, null)
    assert rc == _ffi.SCREE_ERR_INVALID and "state row stride" in err()
    rc = lib.scree_linear_attn_step(p, p, p, p, p, null, p, 2, 4, 4, 64, 64, rows, 1.0, 1, null)
    assert rc == _ffi.SCREE_ERR_INVALID and "null" in err()
