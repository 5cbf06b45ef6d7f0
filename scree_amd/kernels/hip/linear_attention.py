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


class _Plan:
    """What a call's shapes, strides and dtypes decide; a loop asks for the same
    one every step.  The arrays of strides are only read."""

    __slots__ = ("code", "scale", "out_shape", "sizes", "in_place", "rows", "strides",
                 "bwd_strides")

    def __init__(self, qs, ks, vs, dtype, qst, kst, vst):
        self.code = _ffi.dtype_code(dtype)
        self.scale = 1.0 / math.sqrt(qs[2])
        self.out_shape = (qs[0], qs[1], vs[2])
        self.sizes = (qs[0], qs[1], ks[1], qs[2], vs[2])  # total, heads, kv_heads, k_dim, v_dim
        # q, k and v are read where they lie (if they are aligned)
        self.in_place = all(_readable(*x) for x in ((qs, qst), (ks, kst), (vs, vst)))
        rows = _row_head(qs, qst) + _row_head(ks, kst) + _row_head(vs, vst)
        o = (qs[1] * vs[2], vs[2])
        fresh = tuple(x for t in (qs, ks, vs) for x in (t[1] * t[2], t[2]))
        self.rows = rows + o
        self.strides = _ffi.int64_array(self.rows)
        self.bwd_strides = _ffi.int64_array(o + rows + fresh)


@functools.lru_cache(maxsize=512)
def _plan(qs, ks, vs, gs, dtype, kdtype, vdtype, gdtype, qst, kst, vst):
    assert len(qs) == len(ks) == len(vs) == 3, "q, k, v must be (tokens, heads, head_dim)"
    assert ks[:2] == vs[:2], "k and v must share tokens and heads"
    assert qs[0] == ks[0] and qs[2] == ks[2], "q and k must share tokens and head_dim"
    assert ks[1] >= 1 and qs[1] >= 1 and qs[1] % ks[1] == 0, (
        "k/v heads must divide q heads (grouped-query attention)")
    for d in (qs[2], vs[2]):
        assert 8 <= d <= MAX_DIM and d % 8 == 0, "head dims must be multiples of 8 up to 256"
    assert dtype in (torch.float16, torch.bfloat16, torch.float32), f"unsupported dtype {dtype}"
    assert dtype == kdtype == vdtype, "q, k, v must share a dtype"
    assert gs == ks[1:2] and gdtype == torch.float32, "log_decay must be float32, one per K/V head"
    return _Plan(qs, ks, vs, dtype, qst, kst, vst)


def _check(q, k, v, log_decay):
    dev = q.get_device()
    assert dev >= 0, "linear attention on HIP requires ROCm device tensors"
    plan = _plan(q.shape, k.shape, v.shape, log_decay.shape, q.dtype, k.dtype, v.dtype,
                 log_decay.dtype, q.stride(), k.stride(), v.stride())
    assert dev == k.get_device() == v.get_device(), "q, k, v must be on the same device"
    assert dev == log_decay.get_device(), "log_decay must be on q's device"
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("log_decay is a constant of the head: it has no gradient here")
    return plan


def _check_state(s, name, batch, k, v):
    assert s.shape == (batch, *k.shape[1:], v.shape[2]), (
        f"{name} must be (batch, kv_heads, k_dim, v_dim)")
    assert s.dtype == torch.float32, f"{name} must be float32"
    assert s.get_device() == k.get_device(), f"{name} must be on q's device"


def _row_head(shape, stride):
    """Row and head strides; those of an axis of one are the contiguous ones."""
    n, h, d = shape
    s0, s1, _ = stride
    if h == 1:
        s1 = d
    return (h * d if n <= 1 else s0), s1


def _readable(shape, stride):
    """Whether the library can read these rows in place."""
    n, h, d = shape
    s0, s1 = _row_head(shape, stride)
    if n == 0 or (stride[2] == 1 and s1 == d and s0 == h * d):
        return True
    return (stride[2] == 1 and s0 % 8 == 0 and s1 % 8 == 0 and 0 <= s1 < _MAX_STRIDE
            and d <= s0 < _MAX_STRIDE)


def _view(t):
    """``t`` itself when the library can read it in place, else an aligned copy."""
    if t.data_ptr() % 16 == 0 and _readable(t.shape, t.stride()):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _read(plan, q, k, v):
    """q, k and v for the library, and whether the plan's strides are theirs."""
    if plan.in_place and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        return q, k, v, True
    return _view(q), _view(k), _view(v), False


def _out(out, shape, q, what):
    """``(out, where the library writes it)``, ``out`` checked or a new tensor."""
    if out is None:
        out = q.new_empty(shape)
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
    return _ffi.int64_array(sum([_row_head(t.shape, t.stride()) for t in ts], ()) + extra)


def _like(t):
    """A fresh contiguous tensor of ``t``'s shape."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return t.new_empty(t.shape)


def _new_state(cu, plan, q):
    _, _, hk, dk, dv = plan.sizes
    return torch.empty((cu.numel() - 1, hk, dk, dv), dtype=torch.float32, device=q.device)


def linear_fwd(plan, planned, q, k, v, log_decay, cu, scale, init, want_state, out):
    """``(final states or None, workspace or None)``; the backward of the same
    call can take the workspace's states."""
    last = _new_state(cu, plan, q) if want_state else None
    sizes = (cu.numel() - 1, *plan.sizes)
    nws = workspace_bytes(*sizes, False)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
    strides = plan.strides if planned and out.is_contiguous() else _strides((q, k, v, out))
    _ffi.launch(_ffi.lib().scree_linear_attn_fwd, q, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                log_decay.data_ptr(), out.data_ptr(), _ffi.ptr(init), _ffi.ptr(last), cu.data_ptr(),
                *sizes, strides, scale, plan.code, _ffi.ptr(ws), nws)
    return last, ws


def linear_bwd(plan, planned, do, q, k, v, log_decay, cu, scale, init, dlast, want_dinit,
               fwd_ws=None):
    dq, dk, dv = _like(q), _like(k), _like(v)
    dinit = _new_state(cu, plan, q) if want_dinit else None
    sizes = (cu.numel() - 1, *plan.sizes)
    strides = (plan.bwd_strides if planned and do.is_contiguous()
               else _strides((do, q, k, v, dq, dk, dv)))
    nws = workspace_bytes(*sizes, fwd_ws is None)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
    _ffi.launch(_ffi.lib().scree_linear_attn_bwd, q, do.data_ptr(), q.data_ptr(), k.data_ptr(),
                v.data_ptr(), log_decay.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                _ffi.ptr(init), _ffi.ptr(dlast), _ffi.ptr(dinit), _ffi.ptr(fwd_ws), cu.data_ptr(),
                *sizes, strides, scale, plan.code, _ffi.ptr(ws), nws)
    return dq, dk, dv, dinit


class _LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, cu, scale, init, want_state, plan):
        qk, kk, vk, planned = _read(plan, q, k, v)
        s0 = _state(init)
        out = q.new_empty(plan.out_shape)
        # the workspace's states between segments serve the backward too
        last, ws = linear_fwd(plan, planned, qk, kk, vk, log_decay, cu, scale, s0, want_state, out)
        ctx.save_for_backward(qk, kk, vk, log_decay, cu, s0, ws)
        ctx.call = plan, planned, scale
        ctx.set_materialize_grads(False)
        return (out, last) if want_state else out

    @staticmethod
    def backward(ctx, do, dlast=None):
        q, k, v, log_decay, cu, s0, ws = ctx.saved_tensors
        if do is None and dlast is None:
            return (None,) * 9
        plan, planned, scale = ctx.call
        if do is None:
            do = q.new_zeros(plan.out_shape)
        grads = linear_bwd(plan, planned, _view(do), q, k, v, log_decay, cu, scale, s0, _state(dlast),
                           ctx.needs_input_grad[6], ws)
        dq, dk, dv, dinit = once("varlen linear attention", *grads)
        return dq, dk, dv, None, None, None, dinit, None, None


def _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state):
    plan = _check(q, k, v, log_decay)
    cu = _cu(cu_seqlens, q.device)
    assert cu.dim() == 1 and cu.numel() >= 2, "cu_seqlens must have batch + 1 entries"
    if initial_state is not None:
        _check_state(initial_state, "initial_state", cu.numel() - 1, k, v)
    return plan, cu, plan.scale if scale is None else float(scale)


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
    plan, cu, scale = _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (
            initial_state is not None and initial_state.requires_grad)):
        assert out is None, "out= is not supported when an input requires grad"
        return _LinearAttentionFn.apply(q, k, v, log_decay.contiguous(), cu, scale, initial_state,
                                        bool(return_state), plan)
    out, ok = _out(out, plan.out_shape, q, "total_tokens")
    qk, kk, vk, planned = _read(plan, q, k, v)
    last, _ = linear_fwd(plan, planned, qk, kk, vk, log_decay.contiguous(), cu, scale,
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
    plan, cu, scale = _prepare(q, k, v, log_decay, cu_seqlens, scale, initial_state)
    assert do.shape == plan.out_shape and do.dtype == q.dtype and do.device == q.device, (
        "do must be (total_tokens, heads, v_dim) like q")
    if dstate is not None:
        _check_state(dstate, "dstate", cu.numel() - 1, k, v)
    qk, kk, vk, planned = _read(plan, q, k, v)
    return linear_bwd(plan, planned, _view(do), qk, kk, vk, log_decay.contiguous(), cu, scale,
                      _state(initial_state), _state(dstate), initial_state is not None)


@functools.lru_cache(maxsize=512)
def _state_row(name, shape, stride, dtype, batch, hk, dk, dv):
    """The row stride of a decoding state of this layout."""
    assert shape == (batch, hk, dk, dv), f"{name} must be (batch, kv_heads, k_dim, v_dim)"
    assert dtype == torch.float32, f"{name} must be float32"
    s0, s1, s2, s3 = stride
    if batch <= 1:
        s0 = hk * dk * dv
    assert (s1 == dk * dv or hk == 1) and s2 == dv and s3 == 1 and s0 % 4 == 0 and (
        s0 >= hk * dk * dv), f"{name} must hold each row's state contiguously"
    return s0


def _step_state(s, name, q, sizes):
    assert s.get_device() == q.get_device(), f"{name} must be on q's device"
    row = _state_row(name, s.shape, s.stride(), s.dtype, sizes[0], *sizes[2:])
    assert s.data_ptr() % 16 == 0, f"{name} must be 16-byte aligned"
    return row


@functools.lru_cache(maxsize=512)
def _step_strides(rows, *state_rows):
    return _ffi.int64_array(rows + state_rows)


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
    plan = _check(q, k, v, log_decay)
    assert not ((q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)
                and torch.is_grad_enabled()), (
        "a decoding step records no gradient; use varlen_linear_attention_hip")
    rows = rows_out = _step_state(state, "state", q, plan.sizes)
    if state_out is None:
        state_out = state
    else:
        rows_out = _step_state(state_out, "state_out", q, plan.sizes)
    out, ok = _out(out, plan.out_shape, q, "batch")
    if plan.sizes[0] == 0:
        return out
    increment_version(state_out)
    qk, kk, vk, planned = _read(plan, q, k, v)
    if planned and ok.is_contiguous():
        strides = _step_strides(plan.rows, rows, rows_out)
    else:
        strides = _strides((qk, kk, vk, ok), (rows, rows_out))
    _ffi.launch(_ffi.lib().scree_linear_attn_step, qk, qk.data_ptr(), kk.data_ptr(), vk.data_ptr(),
                log_decay.contiguous().data_ptr(), ok.data_ptr(), state.data_ptr(),
                state_out.data_ptr(), *plan.sizes, strides,
                plan.scale if scale is None else float(scale), plan.code)
    if ok is not out:
        out.copy_(ok)
    return out
