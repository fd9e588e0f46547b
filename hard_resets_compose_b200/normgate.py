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
from ._lib import DTYPES, addr, check, need_cuda, on_device, raw_stream

ACTS = {"silu": 0, "sigmoid": 1, "none": 2}
MAX_WIDTH = 8192


def _rows(t, D):
    """t as [R, D] rows with a row stride, without a copy where it has one."""
    if t.dim() != 2:
        t = t.reshape(-1, D)
    if t.shape[0] > 1 and t.stride(0) < D or D > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _pack(x, h, gate, post, pre, rstd, scale, eps, act):
    R, D = x.shape
    cols = 0 if gate is None else gate.shape[1]
    w = post if post is not None else pre
    return _lib.NORM_GATE.pack(addr(x), addr(h), addr(gate), addr(post), addr(pre), addr(rstd), R, D, x.stride(0),
                               0 if h is None else h.stride(0), 0 if gate is None else gate.stride(0), cols, scale,
                               eps, act, DTYPES[x.dtype], DTYPES[w.dtype])


def _forward(x, h, gate, post, pre, scale, eps, act, keep):
    R, D = x.shape
    xo = None if h is None else torch.empty(R, D, dtype=x.dtype, device=x.device)
    n = None if pre is None else torch.empty(R, D, dtype=x.dtype, device=x.device)
    rstd = torch.empty(2, R, device=x.device) if keep else None
    with on_device(x):
        check(_lib.load().lifb_norm_gate_fwd(_pack(x, h, gate, post, pre, rstd, scale, eps, act), addr(xo), addr(n),
                                             raw_stream(x)), "norm_gate_residual")
    return xo, n, rstd


class NormGateResidual(torch.autograd.Function):
    """Over rows: x [R, D], h [R, D] or None, gate [R, D], [R, 1] or None."""

    @staticmethod
    def forward(ctx, x, h, gate, post, pre, scale, eps, act):
        xo, n, rstd = _forward(x, h, gate, post, pre, scale, eps, act, True)
        ctx.save_for_backward(x, h, gate, post, pre, rstd)
        ctx.cfg = (scale, eps, act)
        ctx.set_materialize_grads(False)
        return xo, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dxo, dn):
        x, h, gate, post, pre, rstd = ctx.saved_tensors
        R, D = x.shape
        dev = x.device
        if dxo is None and dn is None:
            return (None,) * 8
        dxo = None if dxo is None else _rows(dxo, D)
        dn = None if dn is None else _rows(dn, D)
        need = ctx.needs_input_grad

        def out(i, t):
            return torch.empty(t.shape, dtype=t.dtype, device=dev) if t is not None and need[i] else None

        dx, dh, dgate, dpost, dpre = out(0, x), out(1, h), out(2, gate), out(3, post), out(4, pre)
        lib = _lib.load()
        with on_device(x):
            nb = lib.lifb_norm_gate_bwd_workspace_bytes(R, D, DTYPES[x.dtype])
            ws = torch.empty(nb, dtype=torch.uint8, device=dev)
            check(lib.lifb_norm_gate_bwd(_pack(x, h, gate, post, pre, rstd, *ctx.cfg), addr(dxo),
                                         D if dxo is None else dxo.stride(0), addr(dn),
                                         D if dn is None else dn.stride(0), addr(dx), addr(dh), addr(dgate),
                                         addr(dpost), addr(dpre), addr(ws), nb, raw_stream(x)), "norm_gate_residual")
        return dx, dh, dgate, dpost, dpre, None, None, None


def _run(what, x, h, gate, post, pre, scale, eps, act):
    D = x.shape[-1] if x.dim() else 0
    if x.dtype not in DTYPES:
        raise TypeError(f"{what}: x must be fp32, bf16 or fp16, got {x.dtype}")
    need_cuda(what, x=x, h=h, gate=gate, post_weight=post, pre_weight=pre)
    for name, t in (("h", h), ("gate", gate)):
        if t is not None:
            if t.dtype != x.dtype:
                raise TypeError(f"{what}: {name} must be {x.dtype} like x, got {t.dtype}")
            if t.shape != x.shape and not (name == "gate" and t.shape == x.shape[:-1] + (1,)):
                raise ValueError(f"{what}: {name} {tuple(t.shape)} does not fit x {tuple(x.shape)}")
    wd = None
    for name, w in (("post_weight", post), ("pre_weight", pre)):
        if w is not None:
            if w.shape != (D,):
                raise ValueError(f"{what}: {name} must be [{D}], got {tuple(w.shape)}")
            if w.dtype not in (torch.float32, x.dtype) or wd not in (None, w.dtype):
                raise TypeError(f"{what}: the weights must both be fp32 or both {x.dtype}")
            wd = w.dtype
    if D > MAX_WIDTH:
        raise ValueError(f"{what}: rows of {D} elements; at most {MAX_WIDTH}")
    shape = x.shape
    x = _rows(x, D)
    h = None if h is None else _rows(h, D)
    gate = None if gate is None else _rows(gate, gate.shape[-1])
    post = None if post is None else post.contiguous()
    pre = None if pre is None else pre.contiguous()
    args = (x, h, gate, post, pre, float(scale), float(eps), act)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, h, gate, post, pre)):
        xo, n = NormGateResidual.apply(*args)
    else:
        xo, n, _ = _forward(*args, False)
    return (None if xo is None else xo.view(shape)), (None if n is None else n.view(shape))


def norm_gate_residual(x, h, gate, post_weight, pre_weight=None, residual_scale=1.0, act="silu", eps=1e-6):
    """x' = x + residual_scale * act(gate) * rmsnorm(h) * post_weight, and n =
    rmsnorm(x') * pre_weight: returns (x', n), or x' alone without pre_weight.

    x, h [..., D]; gate [..., D], [..., 1] or None (no gate); the weights [D],
    fp32 or of x's type; act "silu", "sigmoid" or "none" (the gate itself)."""
    if act not in ACTS:
        raise ValueError(f"norm_gate_residual: unknown act {act!r}")
    if h is None or post_weight is None:
        raise ValueError("norm_gate_residual: needs the block's output h and its post_weight (rms_norm has neither)")
    xo, n = _run("norm_gate_residual", x, h, gate, post_weight, pre_weight, residual_scale, eps, ACTS[act])
    return xo if pre_weight is None else (xo, n)


def rms_norm(x, weight, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension."""
    if weight is None:
        raise ValueError("rms_norm: needs a weight")
    return _run("rms_norm", x, None, None, None, weight, 1.0, eps, 2)[1]
