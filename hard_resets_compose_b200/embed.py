"""Embedding with scaling, and its gradient by sorted tokens (csrc/embed.cu).

    y = embedding(tokens, weight, scale)      # y[i] = scale * weight[tokens[i]]

Negative tokens are padding: zeros out, no gradient.  A token past the table
gives zeros too and is reported as a device error (code 102): raised by one of the
next calls of this package's sequence operators (each polls, at most every 20 ms),
or by `_lib.check_device`.  The weight's gradient adds the rows of
each token in fp32, in an order that the tokens alone fix, and is rounded
once: the same bits on every call.  The reference has no such operator.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPES, addr, check, need_cuda, on_device, raw_stream, refuse_tangents


def _forward(tokens, weight, scale):
    V, D = weight.shape
    y = weight.new_empty(tokens.shape + (D,))
    with on_device(weight):
        _lib.poll_device_sometimes("embedding")
        check(_lib.load().lifb_embed_fwd(tokens.data_ptr(), tokens.element_size(), weight.data_ptr(), y.data_ptr(),
                                         tokens.numel(), V, D, max(weight.stride(0), D), scale, DTYPES[weight.dtype],
                                         raw_stream(weight)), "embedding")
    return y


class Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale):
        ctx.save_for_backward(tokens)
        ctx.cfg = (weight.shape, weight.dtype, scale)
        return _forward(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        tokens, = ctx.saved_tensors
        (V, D), dtype, scale = ctx.cfg
        n = tokens.numel()
        if dy.dim() != 2:
            dy = dy.reshape(n, D)
        s0, s1 = dy.stride()
        if s1 != 1 or s0 < D:
            dy = dy.contiguous()
            s0 = D
        dw = dy.new_empty((V, D))
        lib = _lib.load()
        with on_device(dy):
            nb = lib.lifb_embed_bwd_workspace_bytes(n, V, D)
            ws = dy.new_empty(nb, dtype=torch.uint8)
            check(lib.lifb_embed_bwd(addr(tokens), tokens.element_size(), addr(dy), addr(dw), n, V, D,
                                     max(s0, D), scale, DTYPES[dtype], ws.data_ptr(), nb, raw_stream(dy)),
                  "embedding")
            _lib.poll_device_sometimes("embedding")
        return None, dw, None


def embedding(tokens, weight, scale=1.0):
    """scale * weight[tokens]: tokens of any shape (int32 or int64, negative:
    padding), weight [V, D] (fp32, bf16 or fp16); returns [*tokens.shape, D]."""
    y = _lib.fast().embedding(tokens, weight, scale)
    if y is not None:
        return y
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be [V, D], got {tuple(weight.shape)}")
    if weight.dtype not in DTYPES:
        raise TypeError(f"embedding: weight must be fp32, bf16 or fp16, got {weight.dtype}")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"embedding: tokens must be int32 or int64, got {tokens.dtype}")
    need_cuda("embedding", "tokens weight", tokens, weight)
    refuse_tangents("embedding", weight)
    tokens = tokens.contiguous()
    if not weight.is_contiguous() and (weight.stride(1) != 1 or weight.stride(0) < weight.shape[1]):
        weight = weight.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return Embedding.apply(tokens, weight, float(scale))
    return _forward(tokens, weight, float(scale))
