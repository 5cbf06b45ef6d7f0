"""Oracle: varlen linear attention with a decay per head, token by token in
fp64 (no counterpart in the reference).

``S_t = lam S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t`` per sequence and
K/V head, ``lam = exp(log_decay)``; query head ``h`` reads K/V head
``h // group``.  The backward runs the recurrence of ``R_t = dL/dS_t``.
"""

from __future__ import annotations

import numpy as np


def linear_attention_fwd(q, k, v, log_decay, offsets, scale, initial_state=None):
    """``(o, final_state)``."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    n, h, dk = q.shape
    hk, dv = v.shape[1:]
    lam = np.exp(np.asarray(log_decay, dtype=np.float64))[:, None, None]
    batch = len(offsets) - 1
    out = np.zeros((n, h, dv))
    last = np.zeros((batch, hk, dk, dv))
    if initial_state is not None:
        last[:] = initial_state
    for b in range(batch):
        s = last[b]
        for t in range(int(offsets[b]), int(offsets[b + 1])):
            s = lam * s + k[t][:, :, None] * v[t][:, None, :]
            out[t] = scale * np.matmul(q[t].reshape(hk, -1, dk), s).reshape(h, dv)
        last[b] = s
    return out, last


def linear_attention_bwd(do, q, k, v, log_decay, offsets, scale, initial_state=None, dstate=None):
    """``(dq, dk, dv, dinitial_state)``."""
    do, q, k, v = (np.asarray(t, dtype=np.float64) for t in (do, q, k, v))
    n, h, dk_ = q.shape
    hk, dv_ = v.shape[1:]
    g = h // hk
    lam = np.exp(np.asarray(log_decay, dtype=np.float64))[:, None, None]
    batch = len(offsets) - 1
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    dinit = np.zeros((batch, hk, dk_, dv_))
    for b in range(batch):
        rows = range(int(offsets[b]), int(offsets[b + 1]))
        s = np.zeros((hk, dk_, dv_)) if initial_state is None else np.array(initial_state[b], dtype=np.float64)
        for t in rows:
            s = lam * s + k[t][:, :, None] * v[t][:, None, :]
            dq[t] = scale * np.matmul(do[t].reshape(hk, g, dv_), s.transpose(0, 2, 1)).reshape(h, dk_)
        # the gradient of the state that a token receives; the last token's is dstate
        a = np.zeros((hk, dk_, dv_)) if dstate is None else np.array(dstate[b], dtype=np.float64)
        for t in reversed(rows):
            r = a + scale * np.matmul(q[t].reshape(hk, g, dk_).transpose(0, 2, 1), do[t].reshape(hk, g, dv_))
            dk[t] = np.matmul(r, v[t][:, :, None])[:, :, 0]
            dv[t] = np.matmul(k[t][:, None, :], r)[:, 0]
            a = lam * r
        dinit[b] = a
    return dq, dk, dv, dinit
