"""The token log probability oracle against torch, and its gradient against
differences; the host checks of the launchers and of the C ABI (no GPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle.logprobs import token_logprobs, token_logprobs_bwd
from scree_amd.kernels.hip import _ffi


def _case(rows, vocab, seed):
    rng = np.random.default_rng(seed)
    return rng.normal(size=(rows, vocab)) * 3, rng.integers(0, vocab, rows)


@pytest.mark.parametrize("rows,vocab,top_k", [(1, 1, 1), (5, 7, 3), (4, 300, 20)])
def test_oracle_matches_torch(rows, vocab, top_k):
    x, y = _case(rows, vocab, rows + vocab)
    logprob, entropy, top, idx = token_logprobs(x, y, top_k)
    lp = torch.log_softmax(torch.from_numpy(x), dim=1)
    np.testing.assert_allclose(logprob, lp[torch.arange(rows), torch.from_numpy(y)], atol=1e-12)
    np.testing.assert_allclose(entropy, torch.distributions.Categorical(logits=torch.from_numpy(x)).entropy(),
                               atol=1e-12)
    want = torch.topk(lp, top_k, dim=1)
    np.testing.assert_allclose(top, want.values, atol=1e-12)
    np.testing.assert_array_equal(idx, want.indices)


def test_oracle_edges():
    x = np.array([[1.0, -np.inf, 1.0, 0.0], [-np.inf] * 4, [0.0, np.nan, 1.0, 2.0], [0.0, np.inf, 1.0, 2.0]])
    logprob, entropy, top, idx = token_logprobs(x, [1, -1, 0, 4], 3)
    assert logprob[0] == -np.inf and logprob[1] == 0 and np.isnan(logprob[2:]).all()
    assert np.isfinite(entropy[0]) and np.isnan(entropy[1:]).all()
    np.testing.assert_array_equal(idx[:2], [[0, 2, 3], [0, 1, 2]])  # ties: the lowest index first
    dx = token_logprobs_bwd(x, [1, -1, 0, 4], np.ones(4))
    assert np.isfinite(dx[0]).all() and (dx[1] == 0).all() and np.isnan(dx[2:]).all()


def test_oracle_gradient_against_differences():
    x, y = _case(3, 9, 5)
    y[1] = -1
    rng = np.random.default_rng(6)
    g, gh, gt = rng.normal(size=3), rng.normal(size=3), rng.normal(size=(3, 4))
    got = token_logprobs_bwd(x, y, g, gh, gt)

    def loss(z):
        lp, ent, top, _ = token_logprobs(z, y, 4)
        return (g * lp).sum() + (gh * ent).sum() + (gt * top).sum()

    h = 1e-5
    for i in range(3):
        for j in range(9):
            z = x.copy()
            z[i, j] += h
            up = loss(z)
            z[i, j] -= 2 * h
            # central differences: error h^2 / 6 times third derivatives of order |g|, and 1e-16 / h
            assert abs((up - loss(z)) / (2 * h) - got[i, j]) < 1e-8


def test_launcher_refusals():
    from scree_amd.kernels import varlen_token_logprobs
    from scree_amd.kernels.hip import varlen_token_logprobs_hip
    from scree_amd.kernels.hip import logprobs as L

    x, y = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(AssertionError, match="ROCm"):
        varlen_token_logprobs_hip(x, y)
    import scree_amd

    with pytest.raises(TypeError, match="ROCm"):
        varlen_token_logprobs(scree_amd.pack([np.zeros((3, 8), dtype=np.float32)]), y)
    # rows whose last axis is not contiguous, or that overlap, are copied
    strided = torch.zeros(3, 16)[:, ::2]
    assert L._rows_view(strided) is not strided and L._rows_view(strided).is_contiguous()
    padded = torch.zeros(3, 16)[:, :9]
    assert L._rows_view(padded) is padded
    shared = torch.zeros(1, 8).expand(3, 8)
    assert L._rows_view(shared).stride(0) == 8


def test_c_abi_refusals():
    lib = _ffi.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p, null = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16), ctypes.c_void_p(0)
    err = lambda: lib.scree_last_error().decode()  # noqa: E731

    def fwd(stride=100, tb=8, rows=4, vocab=100, k=0, logits=p, top=null, dtype=1, ws=p, nws=1 << 15):
        return lib.scree_token_logprobs(logits, stride, p, tb, rows, vocab, k, p, p, p, top, top, dtype,
                                        ws, nws, null)

    assert fwd(rows=0, logits=null) == _ffi.SCREE_OK
    assert fwd(logits=null) == _ffi.SCREE_ERR_INVALID and "null" in err()
    assert fwd(vocab=0) == _ffi.SCREE_ERR_INVALID and "vocab" in err()
    assert fwd(rows=(1 << 23) + 1) == _ffi.SCREE_ERR_INVALID and "range" in err()
    assert fwd(rows=-1) == _ffi.SCREE_ERR_INVALID
    assert fwd(stride=99) == _ffi.SCREE_ERR_INVALID and "overlaps" in err()
    assert fwd(k=65, top=p) == _ffi.SCREE_ERR_INVALID and "top_k" in err()
    assert fwd(k=101, top=p) == _ffi.SCREE_ERR_INVALID
    assert fwd(k=4) == _ffi.SCREE_ERR_INVALID and "top_logprob" in err()
    assert fwd(tb=2) == _ffi.SCREE_ERR_INVALID and "targets" in err()
    assert fwd(dtype=9) == _ffi.SCREE_ERR_UNSUPPORTED and "dtype" in err()
    # few rows of a large vocabulary are split: partial results need room
    need = lib.scree_token_logprobs_workspace_bytes(4, 100000, 20)
    assert need > 0 and lib.scree_token_logprobs_workspace_bytes(4096, 100000, 20) == 0
    assert fwd(vocab=100000, stride=100000, ws=null, nws=0) == _ffi.SCREE_ERR_WORKSPACE
    assert fwd(vocab=100000, stride=100000, k=20, top=p, nws=need - 1) == _ffi.SCREE_ERR_WORKSPACE
    rc = lib.scree_token_logprobs_bwd(p, 100, p, 8, 4, 100, 0, p, p, null, p, p, p, p, 100, 1, null)
    assert rc == _ffi.SCREE_ERR_INVALID and "top_index" in err()
    rc = lib.scree_token_logprobs_bwd(p, 100, p, 8, 4, 100, 0, p, p, null, p, p, null, p, 99, 1, null)
    assert rc == _ffi.SCREE_ERR_INVALID and "overlaps" in err()
