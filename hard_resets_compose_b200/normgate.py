"""The norms around a block, its gate and its scaled residual, fused
(csrc/normgate.cu):

    y  = rmsnorm(h) * post_weight
    x' = x + residual_scale * act(gate) * y       # the residual stream
    n  = rmsnorm(x') * pre_weight                 # the next block's input

    x, n = norm_gate_residual(x, h, gate, post_weight, pre_weight, ...)
    n    = rms_norm(x, pre_weight)                # before the first block

with rmsnorm(z) = z / sqrt(mean(z^2) + eps).  Rows are fp32, bf16 or fp16, all
arithmetic is fp32, and x' enters its norm unrounded.  The backward reads each
tensor once; the weights' gradients add the rows in a fixed order.  The
reference has no such operator.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPES, addr, check, need_cuda, on_device, raw_stream, refuse_tangents

ACTS = {"silu": 0, "sigmoid": 1, "none": 2}
MAX_WIDTH = 8192


def _rows(t, D):
    """t as [R, D] rows with a row stride, without a copy where it has one."""
    if t.dim() != 2:
        t = t.reshape(-1, D)
    if t.is_contiguous():
        return t
    s0, s1 = t.stride()
    if s1 != 1 and D > 1 or s0 < D and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _pack(x, h, gate, post, pre, rstd, scale, eps, act):
    R, D = x.shape
    w = post if post is not None else pre
    return _lib.NORM_GATE.pack(x.data_ptr(), addr(h), addr(gate), addr(post), addr(pre), addr(rstd), R, D,
                               x.stride(0), 0 if h is None else h.stride(0), 0 if gate is None else gate.stride(0),
                               0 if gate is None else gate.shape[1], scale, eps, act, DTYPES[x.dtype],
                               DTYPES[w.dtype])


def _forward(x, h, gate, post, pre, scale, eps, act, keep):
    """x' and n in x's shape, and (keep) what the backward needs: the operands as
    rows and each row's two factors."""
    shape, D = x.shape, x.shape[-1]
    xo = None if h is None else x.new_empty(shape)
    n = None if pre is None else x.new_empty(shape)
    x = _rows(x, D)
    h = None if h is None else _rows(h, D)
    gate = None if gate is None else _rows(gate, gate.shape[-1])
    rstd = x.new_empty((2, x.shape[0]), dtype=torch.float32) if keep else None
    with on_device(x):
        _lib.poll_device_sometimes("norm_gate_residual")
        check(_lib.load().lifb_norm_gate_fwd(_pack(x, h, gate, post, pre, rstd, scale, eps, act), addr(xo), addr(n),
                                             raw_stream(x)), "norm_gate_residual")
    return xo, n, (x, h, gate, rstd)


class NormGateResidual(torch.autograd.Function):
    """x [..., D], h [..., D] or None, gate [..., D], [..., 1] or None."""

    @staticmethod
    def forward(ctx, x, h, gate, post, pre, scale, eps, act):
        xo, n, (x2, h2, g2, rstd) = _forward(x, h, gate, post, pre, scale, eps, act, True)
        ctx.save_for_backward(x2, h2, g2, post, pre, rstd)
        ctx.cfg = (scale, eps, act)
        ctx.shapes = (x.shape, None if gate is None else gate.shape)
        ctx.set_materialize_grads(False)
        return xo, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dxo, dn):
        if dxo is None and dn is None:
            return (None,) * 8
        x, h, gate, post, pre, rstd = ctx.saved_tensors
        R, D = x.shape
        shape, gate_shape = ctx.shapes
        dxo = None if dxo is None else _rows(dxo, D)
        dn = None if dn is None else _rows(dn, D)
        need = ctx.needs_input_grad
        dx = x.new_empty(shape) if need[0] else None
        dh = x.new_empty(shape) if need[1] else None
        dgate = x.new_empty(gate_shape) if need[2] else None
        dpost = torch.empty_like(post) if need[3] else None
        dpre = torch.empty_like(pre) if need[4] else None
        lib = _lib.load()
        with on_device(x):
            nb = lib.lifb_norm_gate_bwd_workspace_bytes(R, D, DTYPES[x.dtype]) if need[3] or need[4] else 0
            ws = x.new_empty(nb, dtype=torch.uint8)
            check(lib.lifb_norm_gate_bwd(_pack(x, h, gate, post, pre, rstd, *ctx.cfg), addr(dxo),
                                         D if dxo is None else dxo.stride(0), addr(dn),
                                         D if dn is None else dn.stride(0), addr(dx), addr(dh), addr(dgate),
                                         addr(dpost), addr(dpre), ws.data_ptr(), nb, raw_stream(x)),
                  "norm_gate_residual")
            _lib.poll_device_sometimes("norm_gate_residual")
        return dx, dh, dgate, dpost, dpre, None, None, None


def _run(what, x, h, gate, post, pre, scale, eps, act):
    shape, dt = x.shape, x.dtype
    D = shape[-1] if shape else 0
    if dt not in DTYPES:
        raise TypeError(f"{what}: x must be fp32, bf16 or fp16, got {dt}")
    need_cuda(what, "x h gate post_weight pre_weight", x, h, gate, post, pre)
    refuse_tangents(what, x, h, gate, post, pre)
    for name, t in (("h", h), ("gate", gate)):
        if t is not None:
            if t.dtype != dt:
                raise TypeError(f"{what}: {name} must be {dt} like x, got {t.dtype}")
            if t.shape != shape and not (name == "gate" and t.shape == shape[:-1] + (1,)):
                raise ValueError(f"{what}: {name} {tuple(t.shape)} does not fit x {tuple(shape)}")
    wd = None
    for name, w in (("post_weight", post), ("pre_weight", pre)):
        if w is not None:
            if w.dim() != 1 or w.shape[0] != D:
                raise ValueError(f"{what}: {name} must be [{D}], got {tuple(w.shape)}")
            if w.dtype not in (torch.float32, dt) or wd not in (None, w.dtype):
                raise TypeError(f"{what}: the weights must both be fp32 or both {dt}")
            wd = w.dtype
    if D > MAX_WIDTH:
        raise ValueError(f"{what}: rows of {D} elements; at most {MAX_WIDTH}")
    post = None if post is None else post.contiguous()
    pre = None if pre is None else pre.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, h, gate, post, pre)):
        return NormGateResidual.apply(x, h, gate, post, pre, float(scale), float(eps), act)
    return _forward(x, h, gate, post, pre, float(scale), float(eps), act, False)[:2]


def norm_gate_residual(x, h, gate, post_weight, pre_weight=None, residual_scale=1.0, act="silu", eps=1e-6):
    """x' = x + residual_scale * act(gate) * rmsnorm(h) * post_weight, and n =
    rmsnorm(x') * pre_weight: returns (x', n), or x' alone without pre_weight.

    x, h [..., D]; gate [..., D], [..., 1] or None (no gate); the weights [D],
    fp32 or of x's type; act "silu", "sigmoid" or "none" (the gate itself)."""
    if act not in ACTS:
        raise ValueError(f"norm_gate_residual: unknown act {act!r}")
    if h is None or post_weight is None:
        raise ValueError("norm_gate_residual: needs the block's output h and its post_weight (rms_norm has neither)")
    out = _lib.fast().norm_gate(x, h, gate, post_weight, pre_weight, residual_scale, eps, ACTS[act])
    if out is not None:
        return out
    xo, n = _run("norm_gate_residual", x, h, gate, post_weight, pre_weight, residual_scale, eps, ACTS[act])
    return xo if pre_weight is None else (xo, n)


def rms_norm(x, weight, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension."""
    if weight is None:
        raise ValueError("rms_norm: needs a weight")
    n = _lib.fast().norm_gate(x, None, None, None, weight, 1.0, eps, 2)
    if n is not None:
        return n
    return _run("rms_norm", x, None, None, None, weight, 1.0, eps, 2)[1]
