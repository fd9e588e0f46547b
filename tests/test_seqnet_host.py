"""The sequence model's own bookkeeping (the decay's type, places of the cache, lengths)
on the CPU, its operators replaced by plain forms."""
import pytest
import torch

from hard_resets_compose_b200 import seqnet


def _rms(z, w, eps=1e-6):
    return z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + eps) * w


def _embedding(tokens, weight, scale=1.0):
    return torch.where((tokens >= 0)[..., None], weight[tokens.clamp(min=0)] * scale, 0.0)


def _norm(x, h, gate, post, pre=None, residual_scale=1.0, act="silu", eps=1e-6):
    a = torch.sigmoid(gate) * (gate if act == "silu" else 1.0)
    x = x + residual_scale * a * _rms(h, post)
    return x, _rms(x, pre)


def _step(q, k, v, log_decay, state, slots=None, scale=None):
    B, H, Dk = q.shape
    k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    o = q.new_zeros(B, H, v.shape[2])
    for i in range(B):
        s = i if slots is None else int(slots[i])
        if 0 <= s < state.shape[0]:
            state[s] = log_decay.exp()[:, None, None] * state[s] + k[i, :, :, None] * v[i, :, None, :]
            o[i] = Dk ** -0.5 * (q[i, :, :, None] * state[s]).sum(1)
    return o


def _attention(q, k, v, log_decay, state=None, lengths=None, scale=None, return_state=False):
    B, T, H, Dk = q.shape
    st = torch.zeros(B, H, Dk, v.shape[3])
    o = q.new_zeros(B, T, H, v.shape[3])
    for t in range(T):
        places = torch.arange(B) if lengths is None else torch.where(t < lengths, torch.arange(B), -1)
        o[:, t] = _step(q[:, t], k[:, t], v[:, t], log_decay, st, places)
    return (o, st) if return_state else o


def _serial(i, beta, theta, v_reset, u0):
    u, us, ss = u0, [], []
    for row in i:
        pot = beta * u + row
        s = (pot >= theta).to(row.dtype)
        u = torch.where(s > 0, torch.full_like(pot, v_reset), pot)
        us.append(u)
        ss.append(s)
    return (torch.stack(us), torch.stack(ss)) if us else (i, i)


@pytest.fixture
def net(monkeypatch):
    for name, f in (("embedding", _embedding), ("rms_norm", _rms), ("norm_gate_residual", _norm),
                    ("leaky_attention", _attention), ("leaky_attention_step", _step)):
        monkeypatch.setattr(seqnet, name, f)
    monkeypatch.setattr(seqnet.L, "serial_forward", _serial)
    torch.manual_seed(5)
    return seqnet.SeqNet(vocab=30, width=16, heads=2, layers=2)


def filled(net, slots, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [tuple(torch.randn(t.shape, generator=g) for t in pair) for pair in net.new_cache(slots)]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("kind", ("bfloat16", "to", "half", "double"))
def test_the_decay_keeps_its_bits(kind):
    n = seqnet.SeqNet(vocab=5, width=32, heads=4, layers=2)
    before = [b.log_decay.clone() for b in n.blocks]
    n = n.to(torch.bfloat16) if kind == "to" else getattr(n, kind)()
    assert n.blocks[0].out.weight.dtype != torch.float32
    for b, d in zip(n.blocks, before):
        assert b.log_decay.dtype == torch.float32 and torch.equal(b.log_decay, d)
        assert dict(b.named_buffers())["log_decay"] is b.log_decay


def test_a_step_with_empty_places(net):
    """Places outside the cache: nothing changes in it, the live ones get what they get alone."""
    n = 4
    slots, tokens = i32(2, -1, 3, n, -7), torch.tensor([1, 2, 3, 4, 5])
    live = torch.tensor([True, False, True, False, False])
    alone = filled(net, n)
    want = net.step(tokens[live], alone, slots[live])
    cache = filled(net, n)
    got = net.step(tokens, cache, slots)
    assert torch.equal(got[live], want) and not got[~live].any()
    for (s, p), (ws, wp) in zip(cache, alone):
        assert torch.equal(s, ws) and torch.equal(p, wp)


def test_a_step_of_empty_places_only(net):
    cache, before = filled(net, 3), filled(net, 3)
    assert not net.step(torch.tensor([1, 2]), cache, i32(-1, 3)).any()
    for a, b in zip(cache, before):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_prompt_with_empty_places(net):
    """A prompt without a place gets its logits; its states are kept nowhere."""
    n, lengths = 4, i32(5, 3, 0, 4)
    slots = i32(-1, 3, 0, n)
    tokens = torch.randint(0, 30, (4, 5), generator=torch.Generator().manual_seed(2))
    whole = net.new_cache(4)
    want = net.prompt(tokens, whole, i32(0, 1, 2, 3), lengths)
    cache, before = filled(net, n), filled(net, n)
    assert torch.equal(net.prompt(tokens, cache, slots, lengths), want)
    for pair, was, ref in zip(cache, before, whole):
        for t, w, r in zip(pair, was, ref):
            assert torch.equal(t[3], r[1]) and torch.equal(t[0], r[2]) and torch.equal(t[1:3], w[1:3])


def test_lengths_outside_the_batch(net):
    """Lengths past T count as T, below zero as zero, as the attention takes them."""
    tokens = torch.randint(0, 30, (3, 4), generator=torch.Generator().manual_seed(2))
    a, b = net.new_cache(3), net.new_cache(3)
    want = net.prompt(tokens, a, i32(0, 1, 2), i32(4, 0, 2))
    assert torch.equal(net.prompt(tokens, b, i32(0, 1, 2), i32(9, -3, 2)), want)
    assert all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


def test_prompts_without_tokens(net):
    cache = filled(net, 2)
    got = net.prompt(torch.zeros(2, 0, dtype=torch.long), cache, i32(0, 1), i32(0, 0))
    assert got.shape == (2, 30) and not got.any()
    assert not any(t.any() for pair in cache for t in pair)


def test_a_model_built_in_bf16(net):
    """Under another default type: the weights have it, the decay and the cache stay fp32."""
    torch.set_default_dtype(torch.bfloat16)
    try:
        n = seqnet.SeqNet(vocab=30, width=16, heads=2, layers=2)
        cache = n.new_cache(2)
    finally:
        torch.set_default_dtype(torch.float32)
    assert n.embed.dtype == torch.bfloat16
    for a, b in zip(n.blocks, net.blocks):
        assert torch.equal(a.log_decay, b.log_decay)
    assert all(t.dtype == torch.float32 for pair in cache for t in pair)
