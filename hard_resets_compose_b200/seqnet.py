"""A token sequence model around the hard-reset LIF layer: embedding, blocks of
leaky attention and spiking neurons between fused norms, and a readout.

Each block has two halves on one residual stream x (n is its norm):

    h = W_o leaky_attention(W_q n, W_k n, W_v n);        x, n = norm_gate_residual(x, h, W_g n, ...)
    h = W_2 lif(W_1 n);                                  x, n = norm_gate_residual(x, h, W_s n, ...)

The same weights run a training batch (`forward`, differentiable), prompts that
leave a state (`prompt`), and one token of each running sequence (`step`), with a
cache of states that sequences have slots in (`new_cache`).

    net = SeqNet(vocab=700, width=256, heads=4, layers=2).cuda()
    loss = torch.nn.functional.cross_entropy(net(tokens).flatten(0, 1), targets.flatten())
    cache = net.new_cache(slots=64)
    logits = net.prompt(tokens, cache, slots, lengths)     # [B, V]: after each prompt's last token
    logits = net.step(next_tokens, cache, slots)           # [B, V]

Attention, norms and embedding run in the weights' type (fp32 or bf16); the LIF
layer's input, potential and spikes are fp32, as everywhere in this package.  Under
autocast to bf16 the linear layers, attention and readout run in bf16 around an fp32 stream.
The reference has no such model.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import lifscan as L
from .embed import embedding
from .leakyattn import leaky_attention, leaky_attention_step
from .normgate import norm_gate_residual, rms_norm


class _Places:
    """Where B sequences' states lie in a cache of n slots: slots [B] int32, outside [0, n) an
    empty place, as for leaky_attention_step.  An empty place is given the slot of a
    live one and writes what that one writes, so that the cache changes by the live ones
    alone (by none if there is none) without the host knowing which they are."""

    def __init__(self, slots, n):
        self.live = (slots >= 0) & (slots < n)
        self.any = self.live.any()
        rows = torch.arange(len(slots), device=slots.device)
        self.source = torch.where(self.live, rows, self.live.long().argmax()) if len(slots) else rows
        self.at = torch.where(self.any, slots.long()[self.source], 0)

    def get(self, cache):
        """The live sequences' rows (an empty place's row is some live one's)."""
        return cache[self.at]

    def put(self, cache, rows, old=None):
        """Writes the live sequences' rows; old: what get gave."""
        cache[self.at] = torch.where(self.any, rows[self.source], self.get(cache) if old is None else old)


class SeqBlock(nn.Module):
    """Leaky attention and a LIF layer, each followed by its norms, gate and residual."""

    def __init__(self, width, heads, kv_heads, beta):
        super().__init__()
        if width % heads or heads % kv_heads:
            raise ValueError(f"{heads} heads of {kv_heads} key/value heads do not fit a width of {width}")
        self.heads, self.kv_heads, self.dim, self.beta = heads, kv_heads, width // heads, beta
        kv = kv_heads * self.dim
        self.splits = (width, kv, kv, width)
        self.qkvg = nn.Linear(width, sum(self.splits), bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.lif_in = nn.Linear(width, 2 * width, bias=False)  # current and gate
        self.lif_out = nn.Linear(width, width, bias=False)
        self.post_attn, self.pre_lif, self.post_lif = (nn.Parameter(torch.ones(width)) for _ in range(3))
        # memories from a few tokens to thousands
        memory = torch.linspace(2.0, 10.0, heads, dtype=torch.float32)
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-memory)))

    def _apply(self, fn, recurse=True):
        """Moves of the module; the decay stays fp32 (1 - 2^-10 is 1 in bf16), bit for bit."""
        decay = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != decay.dtype:
            self.log_decay = decay.to(self.log_decay.device)
        return self

    def attention_in(self, n):
        q, k, v, g = self.qkvg(n).split(self.splits, -1)
        heads = lambda t, h: t.unflatten(-1, (h, self.dim))  # noqa: E731
        return heads(q, self.heads), heads(k, self.kv_heads), heads(v, self.kv_heads), g

    def lif_input(self, n):
        i, g = self.lif_in(n).split(n.shape[-1], -1)
        return i.float(), g


class SeqNet(nn.Module):
    def __init__(self, vocab, width=256, heads=4, layers=2, kv_heads=None, beta=0.95, theta=1.0):
        super().__init__()
        self.width, self.theta = width, theta
        self.embed = nn.Parameter(torch.randn(vocab, width) * width ** -0.5)
        self.blocks = nn.ModuleList(SeqBlock(width, heads, kv_heads or heads, beta) for _ in range(layers))
        # the norm before each block and before the readout
        self.pre = nn.ParameterList(nn.Parameter(torch.ones(width)) for _ in range(layers + 1))
        self.residual_scale = (2 * layers) ** -0.5

    def _embed(self, tokens):
        x = embedding(tokens, self.embed, scale=self.width ** 0.5)
        return x, rms_norm(x, self.pre[0])

    def _logits(self, n):
        return n @ self.embed.t()

    def _block(self, i, x, n, attend, spike):
        """Block i; attend(block, q, k, v) and spike(block, current) keep its states."""
        b, s = self.blocks[i], self.residual_scale
        stream = lambda *ts: [t.to(x.dtype) for t in ts]  # noqa: E731 (autocast's linear layers give bf16)
        q, k, v, g = b.attention_in(n)
        h, g = stream(b.out(attend(b, q, k, v).flatten(-2)), g)
        x, n = norm_gate_residual(x, h, g, b.post_attn, b.pre_lif, residual_scale=s)
        current, g = b.lif_input(n)
        h, g = stream(b.lif_out(spike(b, current).to(n.dtype)), g)
        return norm_gate_residual(x, h, g, b.post_lif, self.pre[i + 1], residual_scale=s, act="sigmoid")

    def _spikes(self, b, current):
        """[B, T, D] currents to spikes, from rest."""
        B, T, D = current.shape
        if current.numel() == 0:
            return current
        i = current.transpose(0, 1).reshape(T, B * D)
        s = L.lif_tuned(i, i.new_zeros(B * D), beta=b.beta, theta=self.theta)
        return s.view(T, B, D).transpose(0, 1)

    def forward(self, tokens, lengths=None):
        """Logits [B, T, V] of tokens [B, T]; lengths [B] int32: padded sequences."""
        x, n = self._embed(tokens)
        for i in range(len(self.blocks)):
            x, n = self._block(i, x, n, lambda b, q, k, v: leaky_attention(q, k, v, b.log_decay, lengths=lengths),
                               self._spikes)
        return self._logits(n)

    def new_cache(self, slots):
        """States of `slots` sequences at rest: for each block the attention's and
        the LIF layer's potentials."""
        zeros = lambda *shape: torch.zeros(slots, *shape, device=self.embed.device, dtype=torch.float32)  # noqa: E731
        return [(zeros(b.heads, b.dim, b.dim), zeros(self.width)) for b in self.blocks]

    @torch.no_grad()
    def prompt(self, tokens, cache, slots, lengths):
        """Runs prompts [B, T] from rest into the slots [B] int32, at most one to a slot (outside
        the cache: the prompt's states are not kept), lengths [B] int32, taken into 0..T;
        logits [B, V] after each one's last token (an empty prompt's are the readout's of zeros)."""
        B, T = tokens.shape
        places = _Places(slots, cache[0][0].shape[0]) if cache else None
        if T == 0:  # no token: all at rest
            for pair in cache:
                for states in pair:
                    places.put(states, states.new_zeros(B, *states.shape[1:]))
            return self.embed.new_zeros(B, self.embed.shape[0])
        x, n = self._embed(tokens)
        last = lengths.long().clamp(max=T).sub(1).clamp(min=0)  # as the attention takes them
        rows = torch.arange(B, device=tokens.device)
        empty = (lengths <= 0)[:, None]

        for i, (states, potentials) in enumerate(cache):
            def attend(b, q, k, v):
                o, s = leaky_attention(q, k, v, b.log_decay, lengths=lengths, return_state=True)
                places.put(states, s)
                return o

            def spike(b, current):
                i = current.transpose(0, 1).reshape(T, B * self.width).contiguous()
                u, s = L.serial_forward(i, b.beta, self.theta, 0.0, i.new_zeros(i.shape[1]))
                places.put(potentials, torch.where(empty, 0.0, u.view(T, B, self.width)[last, rows]))
                return s.view(T, B, self.width).transpose(0, 1)

            x, n = self._block(i, x, n, attend, spike)
        return self._logits(torch.where(empty, torch.zeros_like(n[:, 0]), n[rows, last]))

    @torch.no_grad()
    def step(self, tokens, cache, slots):
        """One token [B] of each sequence (slots [B] int32, at most one sequence to a slot);
        logits [B, V].  The cache is updated in place.  A slot outside the cache (-1, say)
        is an empty place: its logits are zeros and nothing changes."""
        x, n = self._embed(tokens)
        B = tokens.shape[0]
        places = _Places(slots, cache[0][0].shape[0]) if cache else None

        for i, (states, potentials) in enumerate(cache):
            def attend(b, q, k, v):
                return leaky_attention_step(q, k, v, b.log_decay, states, slots=slots)

            def spike(b, current):
                u0 = places.get(potentials)
                u, s = L.serial_forward(current.reshape(1, -1).contiguous(), b.beta, self.theta, 0.0, u0.reshape(-1))
                places.put(potentials, u.view(B, self.width), u0)
                return s.view(B, self.width)

            x, n = self._block(i, x, n, attend, spike)
        return self._logits(torch.where(places.live[:, None], n, 0.0) if places else n)
