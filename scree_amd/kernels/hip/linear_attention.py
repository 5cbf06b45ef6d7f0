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
from torch.autograd.graph import increment_version

from . import _ffi
from ._once import once
from .attention import _MAX_STRIDE, _cu

MAX_DIM = 256


@functools.lru_cache(maxsize=256)
def _shape_plan(qs, ks, vs, dtype):
    """Checks that depend on shapes and dtype alone; ``(dtype code, default scale)``."""
    assert len(qs) == len(ks) == len(vs) == 3, "q, k, v must be (tokens, heads, head_dim)"
    assert ks[:2] == vs[:2], "k and v must share tokens and heads"
    assert qs[0] == ks[0] and qs[2] == ks[2], "q and k must share tokens and head_dim"
    assert ks[1] >= 1 and qs[1] >= 1 and qs[1] % ks[1] == 0, (
        "k/v heads must divide q heads (grouped-query attention)")
    for d in (qs[2], vs[2]):
        assert 8 <= d <= MAX_DIM and d % 8 == 0, "head dims must be multiples of 8 up to 256"
    assert dtype in (torch.float16, torch.bfloat16, torch.float32), f"unsupported dtype {dtype}"
    return _ffi.dtype_code(dtype), 1.0 / math.sqrt(qs[2])


def _check(q, k, v, log_decay):
    dev = q.get_device()
    assert dev >= 0, "linear attention on HIP requires ROCm device tensors"
    plan = _shape_plan(q.shape, k.shape, v.shape, q.dtype)
    assert q.dtype == k.dtype == v.dtype, "q, k, v must share a dtype"
    assert dev == k.get_device() == v.get_device(), "q, k, v must be on the same device"
    assert log_decay.shape == k.shape[1:2] and log_decay.dtype == torch.float32, (
        "log_decay must be float32, one per K/V head")
    assert log_decay.get_device() == dev, "log_decay must be on q's device"
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("log_decay is a constant of the head: it has no gradient here")
    return plan


def _check_state(s, name, batch, k, v):
    assert s.shape == (batch, *k.shape[1:], v.shape[2]), (
        f"{name} must be (batch, kv_heads, k_dim, v_dim)")
    assert s.dtype == torch.float32, f"{name} must be float32"
    assert s.get_device() == k.get_device(), f"{name} must be on q's device"


def _row_head(t):
    """Row and head strides; those of an axis of one are the contiguous ones."""
    n, h, d = t.shape
    s0, s1, _ = t.stride()
    if h == 1:
        s1 = d
    return (h * d if n <= 1 else s0), s1


def _view(t):
    """``t`` itself when the library can read it in place, else an aligned copy."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        s0, s1 = _row_head(t)
        if (t.stride(2) == 1 and s0 % 8 == 0 and s1 % 8 == 0 and 0 <= s1 < _MAX_STRIDE
                and t.shape[2] <= s0 < _MAX_STRIDE):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _out(out, shape, q, what):
    """``(out, where the library writes it)``, ``out`` checked or a new tensor."""
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=q.device)
        return out, out
    assert out.shape == shape and out.dtype == q.dtype and out.device == q.device, (
        f"out must be ({what}, heads, v_dim) like q")
    assert out.is_contiguous() or 0 not in out.stride(), "out must not be an expanded tensor"
    # autograd sees the write, as that of any in-place operation
    increment_version(out)
    return out, _view(out)


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


def _strides(ts, extra=()):
    return _ffi.int64_array(sum([_row_head(t) for t in ts], ()) + extra)


def _like(t):
    """A fresh contiguous tensor of ``t``'s shape."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _new_state(cu, k, v):
    return torch.empty((cu.numel() - 1, *k.shape[1:], v.shape[2]), dtype=torch.float32,
                       device=k.device)


def _sizes(q, k, v, cu):
    n, h, dk = q.shape
    return cu.numel() - 1, n, h, k.shape[1], dk, v.shape[2]


def linear_fwd(q, k, v, log_decay, cu, scale, init, want_state, out):
    """``(final states or None, workspace or None)``; the backward of the same
    call can take the workspace's states."""
    last = _new_state(cu, k, v) if want_state else None
    sizes = _sizes(q, k, v, cu)
    nws = workspace_bytes(*sizes, False)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
    _ffi.launch(_ffi.lib().scree_linear_attn_fwd, q, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                log_decay.data_ptr(), out.data_ptr(), _ffi.ptr(init), _ffi.ptr(last), cu.data_ptr(),
                *sizes, _strides((q, k, v, out)), scale, _ffi.dtype_code(q.dtype), _ffi.ptr(ws), nws)
    return last, ws


# The backward runs on autograd's own thread, where Python costs several times
# what it does here: what the forward knows of the call (sizes, the strides of
# a contiguous gradient) is laid out by it.
def _bwd_plan(q, k, v, cu):
    n, h, _ = q.shape
    dv = v.shape[2]
    rows = [_row_head(t) for t in (q, k, v)]
    fresh = [(t.shape[1] * t.shape[2], t.shape[2]) for t in (q, k, v)]
    return (_sizes(q, k, v, cu),
            _ffi.int64_array(sum([(h * dv, dv), *rows, *fresh], ())),
            _ffi.dtype_code(q.dtype))


def linear_bwd(do, q, k, v, log_decay, cu, scale, init, dlast, want_dinit, fwd_ws=None, plan=None):
    dq, dk, dv = _like(q), _like(k), _like(v)
    dinit = _new_state(cu, k, v) if want_dinit else None
    sizes, strides, code = _bwd_plan(q, k, v, cu) if plan is None else plan
    if not do.is_contiguous():
        strides = _strides((do, q, k, v, dq, dk, dv))
    nws = workspace_bytes(*sizes, fwd_ws is None)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
    _ffi.launch(_ffi.lib().scree_linear_attn_bwd, q, do.data_ptr(), q.data_ptr(), k.data_ptr(),
                v.data_ptr(), log_decay.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                _ffi.ptr(init), _ffi.ptr(dlast), _ffi.ptr(dinit), _ffi.ptr(fwd_ws), cu.data_ptr(),
                *sizes, strides, scale, code, _ffi.ptr(ws), nws)
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
        ctx.plan = _bwd_plan(qk, kk, vk, cu)
        ctx.set_materialize_grads(False)
        return (out, last) if want_state else out

    @staticmethod
    def backward(ctx, do, dlast=None):
        q, k, v, log_decay, cu, s0, ws = ctx.saved_tensors
        if do is None and dlast is None:
            return (None,) * 8
        if do is None:
            do = torch.zeros((*q.shape[:2], v.shape[2]), dtype=q.dtype, device=q.device)
        grads = linear_bwd(_view(do), q, k, v, log_decay, cu, ctx.scale, s0, _state(dlast),
                           ctx.needs_input_grad[6], ws, ctx.plan)
        dq, dk, dv, dinit = once("varlen linear attention", *grads)
        return dq, dk, dv, None, None, None, dinit, None


def _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state):
    _, default_scale = _check(q, k, v, log_decay)
    cu = _cu(cu_seqlens, q.device)
    assert cu.dim() == 1 and cu.numel() >= 2, "cu_seqlens must have batch + 1 entries"
    if initial_state is not None:
        _check_state(initial_state, "initial_state", cu.numel() - 1, k, v)
    return cu, default_scale if scale is None else float(scale)


def varlen_linear_attention_hip(q, k, v, log_decay, cu_seqlens, scale=None, initial_state=None,
                                return_state: bool = False, out=None):
    """Causal linear attention of packed sequences with a decay per K/V head.

    ``q`` ``(total_tokens, heads, k_dim)``, ``k`` ``(total_tokens, kv_heads,
    k_dim)`` and ``v`` ``(total_tokens, kv_heads, v_dim)`` share a dtype (fp16,
    bf16 or fp32); ``kv_heads`` divides ``heads`` and the dims are multiples of
    8 up to 256.  ``log_decay`` is fp32 ``(kv_heads,)``, ``log(lam)`` of each
    head: 0 for no decay, -inf for none of the past; growth (above 0) can pass
    the range of the 16-bit products' operands.  ``cu_seqlens`` int32 ``(batch + 1,)`` offsets; an
    empty sequence passes its state on.  ``scale`` defaults to
    ``1 / sqrt(k_dim)``.  ``initial_state`` fp32 ``(batch, kv_heads, k_dim,
    v_dim)`` continues earlier tokens; ``return_state`` also returns the
    states after the last tokens.  ``out`` is an optional preallocated output
    (not when a gradient is recorded) that overlaps no input; rows past the last
    sequence are left as they were.  A gradient needs a finite ``1 / scale``; it
    has no derivative of its own.

    In fp16 a score ``scale * q.k`` past 65504 overflows.  A NaN or infinity in a
    token's k or v may reach earlier outputs of its own sequence and head, at
    most 63 rows before it.

    Returns ``out`` ``(total_tokens, heads, v_dim)`` or ``(out, state)``.
    """
    cu, scale = _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state)
    tracked = [t for t in (q, k, v, initial_state) if t is not None and t.requires_grad]
    if torch.is_grad_enabled() and tracked:
        assert out is None, "out= is not supported when an input requires grad"
        return _LinearAttentionFn.apply(q, k, v, log_decay.contiguous(), cu, scale, initial_state,
                                        bool(return_state))
    out, ok = _out(out, (*q.shape[:2], v.shape[2]), q, "total_tokens")
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


def _step_state(s, name, batch, k, v):
    _check_state(s, name, batch, k, v)
    _, hk, dk, dv = s.shape
    s0, s1, s2, s3 = s.stride()
    if batch <= 1:
        s0 = hk * dk * dv
    assert (s1 == dk * dv or hk == 1) and s2 == dv and s3 == 1 and s0 % 4 == 0 and (
        s0 >= hk * dk * dv) and s.data_ptr() % 16 == 0, (
        f"{name} must hold each row's state contiguously, 16-byte aligned")
    return s0


def linear_attention_step_hip(q, k, v, log_decay, state, scale=None, state_out=None, out=None):
    """One decoding step: a token for each of ``batch`` sequences.

    ``q`` ``(batch, heads, k_dim)``, ``k`` ``(batch, kv_heads, k_dim)``, ``v``
    ``(batch, kv_heads, v_dim)``; ``state`` fp32 ``(batch, kv_heads, k_dim,
    v_dim)``, rows of a larger pool of states allowed, becomes
    ``exp(log_decay) state + k v^T`` in place, or in ``state_out`` when given
    (which must not overlap ``state``, nor ``out`` any input).  Returns ``scale * q state``
    ``(batch, heads, v_dim)``; one step of what
    :func:`varlen_linear_attention_hip` computes.  No gradient is recorded.
    """
    code, default_scale = _check(q, k, v, log_decay)
    assert not ((q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)
                and torch.is_grad_enabled()), (
        "a decoding step records no gradient; use varlen_linear_attention_hip")
    b, h, dk = q.shape
    hk, dv = v.shape[1:]
    rows = _step_state(state, "state", b, k, v)
    if state_out is None:
        state_out, rows_out = state, rows
    else:
        rows_out = _step_state(state_out, "state_out", b, k, v)
    out, ok = _out(out, (b, h, dv), q, "batch")
    if b == 0:
        return out
    increment_version(state_out)
    qk, kk, vk = _view(q), _view(k), _view(v)
    _ffi.launch(_ffi.lib().scree_linear_attn_step, qk, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(),
                log_decay.contiguous().data_ptr(), ok.data_ptr(), state.data_ptr(),
                state_out.data_ptr(), b, h, hk, dk, dv, _strides((qk, kk, vk, ok), (rows, rows_out)),
                default_scale if scale is None else float(scale), code)
    if ok is not out:
        out.copy_(ok)
    return out
