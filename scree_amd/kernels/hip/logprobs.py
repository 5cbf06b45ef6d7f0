"""Log probabilities of given tokens on the HIP kernels: the loss and scoring
end of a packed language-model step.

No counterpart in the reference.  For every row of packed ``logits`` and its
given token :func:`varlen_token_logprobs_hip` returns the token's log
probability, the entropy of the row's distribution and, on request, its most
likely tokens, from one pass over the logits.  The call is autograd-aware; the
backward (:func:`varlen_token_logprobs_hip_backward`) reads the logits again
and writes their gradient, no probabilities are kept.
"""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _ffi
from ._once import once

MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    """``logprob`` and ``entropy`` ``(total,)`` fp32; ``top_logprob`` fp32 and
    ``top_index`` int64 ``(total, top_k)``, None for ``top_k = 0``."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


@functools.lru_cache(maxsize=512)
def _check_shapes(xs, dtype, ys, ydtype, top_k):
    assert len(xs) == 2 and xs[1] >= 1, "logits must be (total_tokens, vocab)"
    assert dtype in (torch.float32, torch.float16, torch.bfloat16), f"unsupported dtype {dtype}"
    assert ys == xs[:1], "targets must have one token per row of logits"
    assert ydtype in (torch.int32, torch.int64), "targets must be int32 or int64"
    assert 0 <= top_k <= min(MAX_TOP_K, xs[1]), (
        f"top_k must be in [0, {MAX_TOP_K}] and at most the vocabulary")


def _check(logits, targets, top_k):
    dev = logits.get_device()
    assert dev >= 0, "varlen_token_logprobs on HIP requires ROCm device tensors"
    _check_shapes(logits.shape, logits.dtype, targets.shape, targets.dtype, top_k)
    assert dev == targets.get_device(), "targets must be on the same device as logits"


def _rows_view(x):
    """``x`` itself when its rows can be read in place, else a contiguous copy."""
    ok = x.shape[1] == 1 or x.stride(1) == 1
    return x if ok and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, vocab, top_k):
    return int(_ffi.lib().scree_token_logprobs_workspace_bytes(rows, vocab, top_k))


def logprobs_fwd(x, targets, top_k, want_stats):
    rows, vocab = x.shape
    logprob = x.new_empty(rows, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    stats = x.new_empty((rows, 2), dtype=torch.float32) if want_stats else None
    top_lp = top_i = None
    if top_k:
        top_lp = x.new_empty((rows, top_k), dtype=torch.float32)
        top_i = x.new_empty((rows, top_k), dtype=torch.int64)
    if rows:
        nbytes = _workspace_bytes(rows, vocab, top_k)
        ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _ffi.launch(_ffi.lib().scree_token_logprobs, x, x.data_ptr(), x.stride(0),
                    targets.data_ptr(), targets.element_size(), rows, vocab, top_k,
                    logprob.data_ptr(), entropy.data_ptr(), _ffi.ptr(stats), _ffi.ptr(top_lp),
                    _ffi.ptr(top_i), _ffi.dtype_code(x.dtype), _ffi.ptr(ws), nbytes)
    return logprob, entropy, stats, top_lp, top_i


def _grad_of(g, shape, x):
    if g is None:
        return None
    assert g.shape == shape, f"a gradient must have its output's shape {tuple(shape)}"
    assert g.get_device() == x.get_device(), "a gradient must be on the same device as logits"
    if g.dtype == torch.float32 and g.is_contiguous():
        return g
    return g.float().contiguous()


def logprobs_bwd(x, targets, stats, entropy, top_i, dlogprob, dentropy, dtop):
    rows, vocab = x.shape
    dx = torch.empty_like(x) if x.is_contiguous() else x.new_empty((rows, vocab))
    top_k = 0 if top_i is None else top_i.shape[1]
    grads = [_grad_of(dlogprob, (rows,), x), _grad_of(dentropy, (rows,), x),
             _grad_of(dtop, (rows, top_k), x)]
    if rows:
        _ffi.launch(_ffi.lib().scree_token_logprobs_bwd, x, x.data_ptr(), x.stride(0),
                    targets.data_ptr(), targets.element_size(), rows, vocab, top_k,
                    stats.data_ptr(), entropy.data_ptr(), _ffi.ptr(top_i),
                    *[_ffi.ptr(g) for g in grads], dx.data_ptr(), vocab,
                    _ffi.dtype_code(x.dtype))
    return dx


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k):
        x, y = _rows_view(logits), targets.contiguous()
        logprob, entropy, stats, top_lp, top_i = logprobs_fwd(x, y, top_k, True)
        ctx.save_for_backward(x, y, stats, entropy, top_i)
        ctx.set_materialize_grads(False)
        if top_k == 0:
            return logprob, entropy
        ctx.mark_non_differentiable(top_i)
        return logprob, entropy, top_lp, top_i

    @staticmethod
    def backward(ctx, dlogprob, dentropy, dtop=None, _=None):
        if dlogprob is None and dentropy is None and dtop is None:
            return None, None, None
        dx = logprobs_bwd(*ctx.saved_tensors, dlogprob, dentropy, dtop)
        return *once("token log probabilities", dx), None, None


def varlen_token_logprobs_hip(logits, targets, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of ``targets`` under packed ``logits`` ``(total, vocab)``.

    ``targets`` are int32 or int64 ``(total,)`` on the same device.  A negative
    target means the row has none: its log probability is 0 and sends no
    gradient back.  A target past the vocabulary gives NaN (the host never
    reads them).  ``top_k`` (0 to 64) asks for that many most likely tokens of
    each row, in falling order, the lowest index first among equal logits.
    Logits may be fp16, bf16 or fp32, their rows strided; the results are fp32.

    A logit of -inf has probability zero.  A row with nothing but -inf, or
    with a NaN or +inf, has NaN results, as ``torch.log_softmax``.
    """
    _check(logits, targets, top_k)
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _TokenLogprobsFn.apply(logits, targets, top_k)
        return TokenLogprobs(*out) if top_k else TokenLogprobs(*out, None, None)
    logprob, entropy, _, top_lp, top_i = logprobs_fwd(_rows_view(logits), targets.contiguous(),
                                                      top_k, False)
    return TokenLogprobs(logprob, entropy, top_lp, top_i)


def varlen_token_logprobs_hip_backward(logits, targets, dlogprob=None, dentropy=None,
                                       dtop_logprob=None, top_k: int = 0):
    """Gradient wrt ``logits`` of :func:`varlen_token_logprobs_hip` given the
    gradients of its outputs (None for zero), the forward run again for its
    statistics."""
    _check(logits, targets, top_k)
    x, y = _rows_view(logits.detach()), targets.contiguous()
    _, entropy, stats, _, top_i = logprobs_fwd(x, y, top_k, True)
    assert dtop_logprob is None or top_k, "dtop_logprob needs top_k"
    return logprobs_bwd(x, y, stats, entropy, top_i, dlogprob, dentropy, dtop_logprob)
