"""Leaky attention: linear attention with a decay for each head, the leaky
integrator with a matrix for a state (csrc/leaky_attn.cu).

    S_t = b S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t,   b = exp(log_decay[h])

    o        = leaky_attention(q, k, v, log_decay)                       # training
    o, state = leaky_attention(q, k, v, log_decay, state=state, lengths=lengths, return_state=True)   # prompts
    o        = leaky_attention_step(q, k, v, log_decay, state, slots)    # one token, the state in place

q [B, T, H, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv] in fp32 or bf16 (the step
takes fp16 too), H a multiple of Hk (each key/value head serves H / Hk query
heads), widths up to 128, log_decay [H] fp32 and at most 0 (-inf: no memory),
states [B, H, Dk, Dv] fp32.  Any strides.  Sequences run on the tensor cores where
rows of Dk and of Dv elements are whole multiples of 16 bytes (widths of 8 in bf16, 4 in
fp32); other widths run on the fp32 pipe, some 15 times slower in bf16 and 4 in fp32
(zero columns added to q, k and v change nothing but the default scale).  An operand or
gradient whose last dimension is not dense, whose address or distances are not multiples
of 16 bytes or, in bf16, whose distance is 0 (expand) is copied first.  B H < 2^16.
fp16 is refused for sequences: a sum over many tokens leaves its range before
it leaves bf16's.  States and sums are fp32.  In bf16 the outputs of calls of up to 128
tokens, or up to 8192 tokens of heads in all (B T H), are rounded once; in larger
ones the decayed scores and the state are rounded to bf16 before they meet v and q
too (relative error 2.4e-3 in place of 1.7e-3; fp32 inputs: 3e-7).  The decay is a
constant: it gets no gradient.  The reference has no such operator.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPES, addr, check, need_cuda, on_device, raw_stream, refuse_tangents

MAX_WIDTH = 128


def _last_dense(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _rows(t, tc):
    """t with a dense last dimension; with tc (widths that the tensor-core kernels take) in the
    16-byte layout that they read: an operand that is not would send the whole call to the fp32 pipe."""
    t = _last_dense(t)
    e = t.element_size()
    if not tc or (t.data_ptr() % 16 == 0 and all(
            n < 2 or (s * e % 16 == 0 and (e == 4 or s > 0)) for n, s in zip(t.shape[:3], t.stride()[:3]))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _tc_widths(q, v):
    return q.shape[-1] * q.element_size() % 16 == 0 and v.shape[-1] * v.element_size() % 16 == 0


def _pack(q, k, v, log_decay, state, lengths, scale):
    B, T, H, Dk = q.shape
    Hk, Dv = v.shape[2:]
    return _lib.LEAKY_ATTN.pack(addr(q), addr(k), addr(v), addr(log_decay), addr(state), addr(lengths), B, T, H, Hk,
                                Dk, Dv, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], scale, DTYPES[q.dtype])


def _forward(q, k, v, log_decay, state, lengths, scale, return_state):
    B, T, H, Dk = q.shape
    Dv = v.shape[3]
    o = q.new_empty((B, T, H, Dv))
    out = q.new_empty((B, H, Dk, Dv), dtype=torch.float32) if return_state else None
    lib = _lib.load()
    args = _pack(q, k, v, log_decay, state, lengths, scale)
    with on_device(q):
        _lib.poll_device_sometimes("leaky_attention")
        nb = lib.lifb_leaky_attn_workspace_bytes(args, 0)
        ws = q.new_empty(nb, dtype=torch.uint8) if nb else None
        check(lib.lifb_leaky_attn_fwd(args, addr(o), addr(out), addr(ws), nb, raw_stream(q)), "leaky_attention")
    return o, out


class LeakyAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale, return_state):
        o, out = _forward(q, k, v, log_decay, state, lengths, scale, return_state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, out

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dout):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        if do is None and dout is None:
            return (None,) * 8
        dev = q.device
        if do is None:
            do = torch.zeros(*q.shape[:3], v.shape[3], dtype=q.dtype, device=dev)
        do = _rows(do, _tc_widths(q, v))
        dout = None if dout is None else dout.contiguous()
        dq, dk, dv = q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(v.shape)
        ds = torch.empty_like(state) if state is not None and ctx.needs_input_grad[4] else None
        lib = _lib.load()
        args = _pack(q, k, v, log_decay, state, lengths, ctx.scale)
        with on_device(q):
            nb = lib.lifb_leaky_attn_workspace_bytes(args, 1)
            ws = q.new_empty(nb, dtype=torch.uint8) if nb else None
            check(lib.lifb_leaky_attn_bwd(args, addr(do), (_lib.c_i64 * 3)(*do.stride()[:3]), addr(dout), addr(dq),
                                          addr(dk), addr(dv), addr(ds), addr(ws), nb, raw_stream(q)),
                  "leaky_attention")
            _lib.poll_device_sometimes("leaky_attention")
        return dq, dk, dv, None, ds, None, None, None


_SEQ_TYPES = (torch.float32, torch.bfloat16)
_STEP_TYPES = tuple(DTYPES)


def _check(what, q, k, v, log_decay, lead, types):
    qs, ks, vs = q.shape, k.shape, v.shape
    if not len(qs) == len(ks) == len(vs) == lead + 2:
        raise ValueError(f"{what}: q, k and v must have {lead + 2} dimensions")
    H, Dk = qs[lead:]
    Hk, Dv = vs[lead:]
    if ks[:lead] != qs[:lead] or vs[:lead] != qs[:lead] or ks[lead] != Hk or ks[lead + 1] != Dk:
        raise ValueError(f"{what}: q {tuple(qs)}, k {tuple(ks)} and v {tuple(vs)} do not fit")
    if H % Hk if Hk else H:
        raise ValueError(f"{what}: {H} heads cannot share {Hk} key/value heads")
    if Dk > MAX_WIDTH or Dv > MAX_WIDTH:
        raise ValueError(f"{what}: head widths {Dk} and {Dv}; at most {MAX_WIDTH}")
    dt = q.dtype
    if dt not in types or k.dtype != dt or v.dtype != dt:
        raise TypeError(f"{what}: q, k and v must share one of {', '.join(str(t) for t in types)}, got {q.dtype}, "
                        f"{k.dtype}, {v.dtype}")
    if log_decay.dim() != 1 or log_decay.shape[0] != H or log_decay.dtype != torch.float32:
        raise ValueError(f"{what}: log_decay must be [{H}] fp32, got {tuple(log_decay.shape)} {log_decay.dtype}")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: the decay is a constant and gets no gradient: pass log_decay.detach()")
    return H, Hk, Dk, Dv


def leaky_attention(q, k, v, log_decay, state=None, lengths=None, scale=None, return_state=False):
    """o [B, T, H, Dv], or (o, final state) with return_state.

    state [B, H, Dk, Dv] fp32: the state before the first token (None: zeros).
    lengths [B] int32: tokens at and past a sequence's length are not read, give
    zeros and leave the state alone.  scale: Dk ** -0.5 by default.  Gradients for
    q, k, v and state."""
    out = _lib.fast().attention(q, k, v, log_decay, state, lengths, scale, return_state)
    if out is not None:
        return out
    what = "leaky_attention"
    H, _, Dk, Dv = _check(what, q, k, v, log_decay, 2, _SEQ_TYPES)
    need_cuda(what, "q k v log_decay state lengths", q, k, v, log_decay, state, lengths)
    refuse_tangents(what, q, k, v, log_decay, state)
    B = q.shape[0]
    if state is not None:
        if state.shape != (B, H, Dk, Dv) or state.dtype != torch.float32:
            raise ValueError(f"{what}: state must be [{B}, {H}, {Dk}, {Dv}] fp32, got {tuple(state.shape)} "
                             f"{state.dtype}")
        state = state.contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.dtype != torch.int32:
            raise ValueError(f"{what}: lengths must be [{B}] int32, got {tuple(lengths.shape)} {lengths.dtype}")
        lengths = lengths.contiguous()
    scale = float(Dk) ** -0.5 if scale is None and Dk > 0 else float(scale or 0.0)
    tc = _tc_widths(q, v)
    args = (_rows(q, tc), _rows(k, tc), _rows(v, tc), log_decay.contiguous(), state, lengths, scale, bool(return_state))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        o, out = LeakyAttention.apply(*args)
    else:
        o, out = _forward(*args)
    return (o, out) if return_state else o


def _overlap(n, s0, h, s1, mat):
    """Whether two of n x h matrices of `mat` elements, at distances s0 and s1, share memory."""
    if n > 1 and s0 < mat:
        return True
    for j in range(1, h):
        i = min(n - 1, j * s1 // s0) if n > 1 else 0  # the nearest ones below and above
        if abs(j * s1 - i * s0) < mat or abs(j * s1 - min(i + 1, n - 1) * s0) < mat:
            return True
    return False


def leaky_attention_step(q, k, v, log_decay, state, slots=None, scale=None):
    """One token of each sequence: o [B, H, Dv]; `state` is updated in place.

    q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; state [n_slots, H, Dk, Dv] fp32, each
    head's matrix contiguous; slots [B] int32: the place of each sequence's state
    (None: its own index), at most one sequence to a slot; a place outside the
    cache (-1, say) is empty: zeros out, nothing changed.  Not differentiable."""
    o = _lib.fast().attention_step(q, k, v, log_decay, state, slots, scale)
    if o is not None:
        return o
    what = "leaky_attention_step"
    H, Hk, Dk, Dv = _check(what, q, k, v, log_decay, 1, _STEP_TYPES)
    need_cuda(what, "q k v log_decay state slots", q, k, v, log_decay, state, slots)
    refuse_tangents(what, q, k, v, log_decay, state)
    B = q.shape[0]
    if state.dim() != 4 or state.shape[1:] != (H, Dk, Dv) or state.dtype != torch.float32:
        raise ValueError(f"{what}: state must be [slots, {H}, {Dk}, {Dv}] fp32, got {tuple(state.shape)} {state.dtype}")
    st = state.stride()
    if Dk * Dv > 1 and ((Dv > 1 and st[3] != 1) or (Dk > 1 and st[2] != Dv)):
        raise ValueError(f"{what}: each head's state must be contiguous")
    if Dk * Dv and state.shape[0] and _overlap(state.shape[0], st[0], H, st[1], Dk * Dv):
        raise ValueError(f"{what}: slots or heads of the state share memory")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError(f"{what}: {B} sequences but {state.shape[0]} states")
    elif slots.shape != (B,) or slots.dtype != torch.int32:
        raise ValueError(f"{what}: slots must be [{B}] int32, got {tuple(slots.shape)} {slots.dtype}")
    else:
        slots = slots.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError(f"{what} is not differentiable: use leaky_attention, or torch.no_grad()")
    q, k, v, log_decay = _last_dense(q), _last_dense(k), _last_dense(v), log_decay.contiguous()
    scale = float(Dk) ** -0.5 if scale is None and Dk > 0 else float(scale or 0.0)
    o = q.new_empty((B, H, Dv))
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    args = _lib.LEAKY_ATTN_STEP.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), addr(slots), B, H,
                                     Hk, Dk, Dv, state.shape[0], q0, q1, k0, k1, v0, v1, st[0], st[1], scale,
                                     DTYPES[q.dtype])
    with on_device(q):
        _lib.poll_device_sometimes(what)
        torch.autograd.graph.increment_version(state)  # who has saved it hears of the change
        check(_lib.load().lifb_leaky_attn_step(args, addr(o), addr(state), raw_stream(q)), what)
    return o
