"""Varlen linear attention with a decay per head on the HIP kernels.

No counterpart in the reference.  Where :func:`varlen_attention_hip` keeps
every key and value, this mixer keeps one ``(k_dim, v_dim)`` state per
sequence and K/V head:

    S_t = exp(log_decay) S_{t-1} + k_t v_t^T,    o_t = scale * q_t S_t

* :func:`varlen_linear_attention_hip` walks packed sequences in chunks
  (training and prompts); autograd-aware, the explicit backward is
  :func:`varlen_linear_attention_hip_backward`;
* :func:`linear_attention_step_hip` takes one token of every sequence of a
  batch (decoding), updating the states in place.

States are fp32 ``(batch, kv_heads, k_dim, v_dim)``; a prompt's final state is
the decoding steps' first.  ``log_decay`` is a constant of each K/V head: a
call with one that requires grad is refused.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _ffi
from .attention import _cu, _kernel_view

MAX_DIM = 256


def _check(q, k, v, log_decay):
    assert q.is_cuda, "linear attention on HIP requires ROCm device tensors"
    assert q.dim() == k.dim() == v.dim() == 3, "q, k, v must be (tokens, heads, head_dim)"
    assert k.shape[:2] == v.shape[:2], "k and v must share tokens and heads"
    assert q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2], (
        "q and k must share tokens and head_dim")
    assert k.shape[1] >= 1 and q.shape[1] >= 1 and q.shape[1] % k.shape[1] == 0, (
        "k/v heads must divide q heads (grouped-query attention)")
    for d in (q.shape[2], v.shape[2]):
        assert 8 <= d <= MAX_DIM and d % 8 == 0, "head dims must be multiples of 8 up to 256"
    assert q.dtype in (torch.float16, torch.bfloat16, torch.float32), f"unsupported dtype {q.dtype}"
    assert q.dtype == k.dtype == v.dtype, "q, k, v must share a dtype"
    assert q.device == k.device == v.device, "q, k, v must be on the same device"
    assert log_decay.shape == k.shape[1:2] and log_decay.dtype == torch.float32, (
        "log_decay must be float32, one per K/V head")
    assert log_decay.device == q.device, "log_decay must be on q's device"
    if torch.is_grad_enabled() and log_decay.requires_grad:
        raise NotImplementedError("log_decay is a constant of the head: it has no gradient here")


def _check_state(s, name, batch, k, v):
    assert s.shape == (batch, k.shape[1], k.shape[2], v.shape[2]), (
        f"{name} must be (batch, kv_heads, k_dim, v_dim)")
    assert s.dtype == torch.float32, f"{name} must be float32"
    assert s.device == k.device, f"{name} must be on q's device"


def _view(t):
    """``t`` itself when the library can read it in place, else an aligned copy."""
    t = _kernel_view(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _state(s):
    if s is None:
        return None
    s = s.contiguous()
    return s if s.data_ptr() % 16 == 0 else s.clone()


@functools.lru_cache(maxsize=256)
def workspace_bytes(batch, total, heads, kv_heads, k_dim, v_dim, backward):
    """Bytes of fp32 states between the segments that long sequences are walked in."""
    return int(_ffi.lib().scree_linear_attn_workspace_bytes(batch, total, heads, kv_heads, k_dim,
                                                            v_dim, int(backward)))


def _workspace(cu, q, k, v, backward):
    n = workspace_bytes(cu.numel() - 1, q.shape[0], q.shape[1], k.shape[1], q.shape[2], v.shape[2],
                        backward)
    return (torch.empty(n, dtype=torch.uint8, device=q.device) if n else None), n


def _strides(ts):
    return _ffi.int64_array(sum((t.stride()[:2] for t in ts), ()))


def linear_fwd(q, k, v, log_decay, cu, scale, init, want_state, out):
    """``(final states or None, workspace or None)``; the backward of the same
    call can take the workspace's states."""
    batch = cu.numel() - 1
    last = None
    if want_state:
        last = torch.empty((batch, k.shape[1], k.shape[2], v.shape[2]), dtype=torch.float32,
                           device=q.device)
    ws, nws = _workspace(cu, q, k, v, False)
    _ffi.launch(_ffi.lib().scree_linear_attn_fwd, q, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                log_decay.data_ptr(), out.data_ptr(), _ffi.ptr(init), _ffi.ptr(last), cu.data_ptr(),
                batch, q.shape[0], q.shape[1], k.shape[1], q.shape[2], v.shape[2],
                _strides((q, k, v, out)), scale, _ffi.dtype_code(q.dtype), _ffi.ptr(ws), nws)
    return last, ws


def linear_bwd(do, q, k, v, log_decay, cu, scale, init, dlast, want_dinit, fwd_ws=None):
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    batch = cu.numel() - 1
    dinit = None
    if want_dinit:
        dinit = torch.empty((batch, k.shape[1], k.shape[2], v.shape[2]), dtype=torch.float32,
                            device=q.device)
    ws, nws = _workspace(cu, q, k, v, fwd_ws is None)
    _ffi.launch(_ffi.lib().scree_linear_attn_bwd, q, do.data_ptr(), q.data_ptr(), k.data_ptr(),
                v.data_ptr(), log_decay.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                _ffi.ptr(init), _ffi.ptr(dlast), _ffi.ptr(dinit), _ffi.ptr(fwd_ws), cu.data_ptr(), batch,
                q.shape[0], q.shape[1], k.shape[1], q.shape[2], v.shape[2],
                _strides((do, q, k, v, dq, dk, dv)), scale, _ffi.dtype_code(q.dtype), _ffi.ptr(ws), nws)
    return dq, dk, dv, dinit


class _LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, cu, scale, init, want_state):
        qk, kk, vk, s0 = _view(q), _view(k), _view(v), _state(init)
        out = torch.empty((*q.shape[:2], v.shape[2]), dtype=q.dtype, device=q.device)
        # the workspace's states between segments serve the backward too
        last, ws = linear_fwd(qk, kk, vk, log_decay, cu, scale, s0, want_state, out)
        ctx.save_for_backward(qk, kk, vk, log_decay, cu, s0, ws)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if want_state else out

    @staticmethod
    def backward(ctx, do, dlast=None):
        q, k, v, log_decay, cu, s0, ws = ctx.saved_tensors
        if do is None and dlast is None:
            return (None,) * 8
        if do is None:
            do = torch.zeros((*q.shape[:2], v.shape[2]), dtype=q.dtype, device=q.device)
        dq, dk, dv, dinit = linear_bwd(_view(do), q, k, v, log_decay, cu, ctx.scale, s0,
                                       _state(dlast), ctx.needs_input_grad[6], ws)
        return dq, dk, dv, None, None, None, dinit, None


def _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state):
    _check(q, k, v, log_decay)
    cu = _cu(cu_seqlens, q.device)
    assert cu.dim() == 1 and cu.numel() >= 2, "cu_seqlens must have batch + 1 entries"
    if initial_state is not None:
        _check_state(initial_state, "initial_state", cu.numel() - 1, k, v)
    return cu, 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)


def varlen_linear_attention_hip(q, k, v, log_decay, cu_seqlens, scale=None, initial_state=None,
                                return_state: bool = False, out=None):
    """Causal linear attention of packed sequences with a decay per K/V head.

    ``q`` ``(total_tokens, heads, k_dim)``, ``k`` ``(total_tokens, kv_heads,
    k_dim)`` and ``v`` ``(total_tokens, kv_heads, v_dim)`` share a dtype (fp16,
    bf16 or fp32); ``kv_heads`` divides ``heads`` and the dims are multiples of
    8 up to 256.  ``log_decay`` is fp32 ``(kv_heads,)``, ``log(lam)`` of each
    head (0 for no decay).  ``cu_seqlens`` int32 ``(batch + 1,)`` offsets; an
    empty sequence passes its state on.  ``scale`` defaults to
    ``1 / sqrt(k_dim)``.  ``initial_state`` fp32 ``(batch, kv_heads, k_dim,
    v_dim)`` continues earlier tokens; ``return_state`` also returns the
    states after the last tokens.  ``out`` is an optional preallocated output
    (not when a gradient is recorded); rows past the last sequence are left as
    they were.

    Returns ``out`` ``(total_tokens, heads, v_dim)`` or ``(out, state)``.
    """
    cu, scale = _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state)
    tracked = [t for t in (q, k, v, initial_state) if t is not None and t.requires_grad]
    if torch.is_grad_enabled() and tracked:
        assert out is None, "out= is not supported when an input requires grad"
        return _LinearAttentionFn.apply(q, k, v, log_decay.contiguous(), cu, scale, initial_state,
                                        bool(return_state))
    shape = (*q.shape[:2], v.shape[2])
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    else:
        assert out.shape == shape and out.dtype == q.dtype and out.device == q.device, (
            "out must be (total_tokens, heads, v_dim) like q")
    ok = _view(out)
    last, _ = linear_fwd(_view(q), _view(k), _view(v), log_decay.contiguous(), cu, scale,
                         _state(initial_state), return_state, ok)
    if ok is not out:
        out.copy_(ok)
    return (out, last) if return_state else out


def varlen_linear_attention_hip_backward(do, q, k, v, log_decay, cu_seqlens, scale=None,
                                         initial_state=None, dstate=None):
    """``(dq, dk, dv, dinitial_state)`` of :func:`varlen_linear_attention_hip`.

    ``dstate`` is the gradient of the returned states (None for zero);
    ``dinitial_state`` is None without an ``initial_state``.  Gradient rows
    past the last sequence are zero.
    """
    cu, scale = _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state)
    assert do.shape == (*q.shape[:2], v.shape[2]) and do.dtype == q.dtype and do.device == q.device, (
        "do must be (total_tokens, heads, v_dim) like q")
    if dstate is not None:
        _check_state(dstate, "dstate", cu.numel() - 1, k, v)
    return linear_bwd(_view(do), _view(q), _view(k), _view(v), log_decay.contiguous(), cu, scale,
                      _state(initial_state), _state(dstate), initial_state is not None)


def _step_rows(s, name):
    assert s.stride()[1:] == (s.shape[2] * s.shape[3], s.shape[3], 1) and s.stride(0) % 4 == 0 and (
        s.shape[0] <= 1 or s.stride(0) >= s[0].numel()) and s.data_ptr() % 16 == 0, (
        f"{name} must hold each row's state contiguously, 16-byte aligned")


def linear_attention_step_hip(q, k, v, log_decay, state, scale=None, state_out=None, out=None):
    """One decoding step: a token for each of ``batch`` sequences.

    ``q`` ``(batch, heads, k_dim)``, ``k`` ``(batch, kv_heads, k_dim)``, ``v``
    ``(batch, kv_heads, v_dim)``; ``state`` fp32 ``(batch, kv_heads, k_dim,
    v_dim)``, rows of a larger pool of states allowed, becomes
    ``exp(log_decay) state + k v^T`` in place, or in ``state_out`` when given
    (which must not overlap ``state``).  Returns ``scale * q state``
    ``(batch, heads, v_dim)``; one step of what
    :func:`varlen_linear_attention_hip` computes.  No gradient is recorded.
    """
    _check(q, k, v, log_decay)
    assert not (torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state))), (
        "a decoding step records no gradient; use varlen_linear_attention_hip")
    b = q.shape[0]
    _check_state(state, "state", b, k, v)
    _step_rows(state, "state")
    if state_out is None:
        state_out = state
    else:
        _check_state(state_out, "state_out", b, k, v)
        _step_rows(state_out, "state_out")
    shape = (*q.shape[:2], v.shape[2])
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
    else:
        assert out.shape == shape and out.dtype == q.dtype and out.device == q.device, (
            "out must be (batch, heads, v_dim) like q")
    if b == 0:
        return out
    qk, kk, vk, ok = _view(q), _view(k), _view(v), _view(out)
    strides = _ffi.int64_array(qk.stride()[:2] + kk.stride()[:2] + vk.stride()[:2] + ok.stride()[:2]
                               + (state.stride(0), state_out.stride(0)))
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    _ffi.launch(_ffi.lib().scree_linear_attn_step, qk, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(),
                log_decay.contiguous().data_ptr(), ok.data_ptr(), state.data_ptr(),
                state_out.data_ptr(), b, q.shape[1], k.shape[1], q.shape[2], v.shape[2], strides,
                scale, _ffi.dtype_code(q.dtype))
    if ok is not out:
        out.copy_(ok)
    return out
