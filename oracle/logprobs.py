"""Oracle: log probabilities of given tokens, entropy, most likely tokens and
the gradient with respect to the logits, in fp64 (no counterpart in the
reference).  Rows with a NaN or +inf, or nothing but -inf, are NaN."""

from __future__ import annotations

import numpy as np


def _log_softmax(x):
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(all="ignore"):
        m = x.max(axis=1, keepdims=True)
        d = x - m
        return d - np.log(np.exp(d).sum(axis=1, keepdims=True))


def _p_log_p(lp):
    with np.errstate(all="ignore"):
        return np.where(lp == -np.inf, 0.0, np.exp(lp) * lp)


def token_logprobs(x, targets, top_k=0):
    """``(logprob, entropy, top_logprob, top_index)``; a negative target has
    log probability 0, one past the vocabulary NaN."""
    lp = _log_softmax(x)
    n, v = lp.shape
    y = np.asarray(targets)
    ok = (y >= 0) & (y < v)
    logprob = np.where(ok, lp[np.arange(n), np.where(ok, y, 0)], np.where(y < 0, 0.0, np.nan))
    entropy = -_p_log_p(lp).sum(axis=1)
    # a stable sort of the negated logits: the lowest index first among equals
    top = np.argsort(-np.asarray(x, dtype=np.float64), axis=1, kind="stable")[:, :top_k]
    return logprob, entropy, np.take_along_axis(lp, top, axis=1), top


def token_logprobs_bwd(x, targets, dlogprob=None, dentropy=None, dtop=None):
    """Gradient of sum(dlogprob logprob + dentropy entropy + dtop top_logprob)."""
    lp = _log_softmax(x)
    n, v = lp.shape
    y = np.asarray(targets)
    dx = np.zeros_like(lp)
    rows = np.arange(n)
    with np.errstate(all="ignore"):
        p = np.exp(lp)
        for i in rows:
            g = 0.0 if dlogprob is None or y[i] < 0 else float(dlogprob[i])
            gh = 0.0 if dentropy is None else float(dentropy[i])
            gt = np.zeros(0) if dtop is None else np.asarray(dtop[i], dtype=np.float64)
            if g == 0.0 and gh == 0.0 and not np.any(gt != 0.0):
                continue
            if y[i] >= v:
                dx[i] = np.nan
                continue
            each = _p_log_p(lp[i])
            dx[i] = -p[i] * (g + gt.sum()) - gh * (each - p[i] * each.sum())
            if y[i] >= 0:
                dx[i, y[i]] += g
            top = np.argsort(-np.asarray(x[i], dtype=np.float64), kind="stable")[:len(gt)]
            dx[i, top] += gt
    return dx
