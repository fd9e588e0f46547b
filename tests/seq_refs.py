"""Plain 64-bit forms of the sequence-model operators, for their tests."""
import torch

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}  # half an ulp, relative


def attention(q, k, v, log_decay, state=None, lengths=None, scale=None, do=None, dstate=None):
    """The recurrence token by token in fp64.  Returns (o, state) and, with do
    (and the final state's gradient dstate), (dq, dk, dv, dstate0) too."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, H, Dk = q.shape
    Hk, Dv = v.shape[2:]
    g = H // Hk
    scale = Dk ** -0.5 if scale is None else scale
    k, v = k.repeat_interleave(g, 2), v.repeat_interleave(g, 2)
    b = log_decay.double().exp()[None, :, None, None]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=q.device) if state is None else state.double().clone()
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.clamp(0, T)
    live = [(t < n)[:, None, None, None] for t in range(T)]
    o, dq = torch.zeros(B, T, H, Dv, dtype=torch.float64, device=q.device), torch.zeros_like(q)
    do = None if do is None else do.double()
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    for t in range(T):
        S = torch.where(live[t], b * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o[:, t] = torch.where(live[t][..., 0], scale * (q[:, t, :, :, None] * S).sum(2), zero)
        if do is not None:
            dq[:, t] = torch.where(live[t][..., 0], scale * (S * do[:, t, :, None, :]).sum(3), zero)
    if do is None:
        return o, S
    G = torch.zeros_like(S) if dstate is None else dstate.double().clone()
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(range(T)):
        F = G + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = torch.where(live[t][..., 0], (F * v[:, t, :, None, :]).sum(3), zero)
        dv[:, t] = torch.where(live[t][..., 0], (F * k[:, t, :, :, None]).sum(2), zero)
        G = torch.where(live[t], b * F, G)
    dk, dv = (x.reshape(B, T, Hk, g, -1).sum(3) for x in (dk, dv))
    return o, S, dq, dk, dv, G


def norm_gate(x, h, gate, post, pre, scale, act, eps):
    """(x', n) in fp64, differentiable."""
    if h is not None:
        y = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * post
        if gate is not None:
            y = y * {"silu": lambda g: g * torch.sigmoid(g), "sigmoid": torch.sigmoid, "none": lambda g: g}[act](gate)
        x = x + scale * y
    n = None if pre is None else x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * pre
    return x, n


def rel(a, b):
    nb = b.double().norm().item()
    return (a.double() - b.double()).norm().item() / (nb if nb else 1.0)
