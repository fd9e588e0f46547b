"""The sequence model (hard_resets_compose_b200.seqnet): training, prompts and
single tokens agree, its gradients match a plain form of the same network, and
it learns."""
import pytest
import torch

from tests.seq_refs import rel

pytestmark = pytest.mark.gpu


def net(dtype=torch.float32, **kw):
    from hard_resets_compose_b200.seqnet import SeqNet
    torch.manual_seed(3)
    n = SeqNet(vocab=50, width=64, heads=4, layers=2, **kw).cuda().to(dtype)
    for b in n.blocks:  # buffers keep fp32
        b.log_decay = b.log_decay.float()
    return n


def plain(n, tokens):
    """The same network in plain torch operations (fp64), spikes with lif_tuned's surrogate gradient."""
    class Spike(torch.autograd.Function):
        @staticmethod
        def forward(ctx, v):
            ctx.save_for_backward(v)
            return (v >= 1.0).to(v.dtype)

        @staticmethod
        def backward(ctx, g):
            v, = ctx.saved_tensors
            s = torch.sigmoid(4.0 * (v - 1.0))
            return g * 4.0 * s * (1 - s)

    rms = lambda z, w: z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    P = {k: v.detach().double().requires_grad_() for k, v in n.named_parameters()}
    B, T = tokens.shape
    x = P["embed"][tokens] * n.width ** 0.5
    z = rms(x, P["pre.0"])
    for i, b in enumerate(n.blocks):
        p = lambda k: P[f"blocks.{i}.{k}"]  # noqa: E731
        q, k, v, g = (z @ p("qkvg.weight").t()).split(b.splits, -1)
        q, k, v = q.view(B, T, b.heads, -1), k.view(B, T, b.kv_heads, -1), v.view(B, T, b.kv_heads, -1)
        k, v = (t.repeat_interleave(b.heads // b.kv_heads, 2) for t in (k, v))
        t = torch.arange(T, device=x.device)
        d = (t[:, None] - t[None]).double()
        m = torch.where(d >= 0, torch.exp(b.log_decay.double()[:, None, None] * d.clamp(min=0)), 0.0)
        sc = torch.einsum("bihd,bjhd->bhij", q, k) * m * b.dim ** -0.5
        o = torch.einsum("bhij,bjhd->bihd", sc, v).reshape(B, T, -1)
        x = x + n.residual_scale * torch.nn.functional.silu(g) * rms(o @ p("out.weight").t(), p("post_attn"))
        z = rms(x, p("pre_lif"))
        cur, g = (z @ p("lif_in.weight").t()).split(n.width, -1)
        u, spikes = torch.zeros(B, n.width, dtype=torch.float64, device=x.device), []
        for s in range(T):
            pot = b.beta * u + cur[:, s]
            spk = Spike.apply(pot)
            u = torch.where(spk.detach() > 0, 0.0, pot)
            spikes.append(spk)
        h = torch.stack(spikes, 1) @ p("lif_out.weight").t()
        x = x + n.residual_scale * torch.sigmoid(g) * rms(h, p("post_lif"))
        z = rms(x, P[f"pre.{i + 1}"])
    return z @ P["embed"].t(), P


@pytest.mark.parametrize("kv_heads", (4, 2))
def test_gradients_match_a_plain_network(cuda, kv_heads):
    """fp32 against fp64.  Some 20 operations deep, each within about 1e-6 of its
    own definition (their tests), the logits agree to 1e-4 and the gradients, which pass
    through the surrogate's slope twice, to 1e-3, as long as no spike falls the other way
    (one that did would move them by far more)."""
    m = net(kv_heads=kv_heads)
    tok = torch.randint(0, 50, (3, 40), device="cuda")
    out = m(tok)
    want, P = plain(m, tok)
    w = torch.randn_like(out)
    got = torch.autograd.grad(out, list(m.parameters()), w)
    ref = torch.autograd.grad(want, list(P.values()), w.double())
    assert rel(out, want) < 1e-4
    for (name, _), a, b in zip(m.named_parameters(), got, ref):
        assert rel(a, b) < 1e-3, name


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_prompt_and_steps_continue_the_batch(cuda, dtype):
    m = net(dtype, kv_heads=2)
    tok = torch.randint(0, 50, (4, 30), device="cuda")
    lengths = torch.tensor([20, 7, 0, 1], dtype=torch.int32, device="cuda")
    slots = torch.tensor([5, 0, 3, 1], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        full = m(tok)
    cache = m.new_cache(7)
    first = m.prompt(tok, cache, slots, lengths)
    rows = torch.arange(4, device="cuda")
    live = lengths > 0
    tol = 1e-4 if dtype == torch.float32 else 0.1
    assert rel(first[live], full[rows, (lengths.long() - 1).clamp(min=0)][live]) < tol
    at = lengths.long()
    for _ in range(8):
        got = m.step(tok[rows, at], cache, slots)
        assert rel(got, full[rows, at]) < tol
        at = at + 1


def test_lengths_hide_what_lies_past_them(cuda):
    m = net()
    tok = torch.randint(0, 50, (2, 33), device="cuda")
    n = torch.tensor([33, 12], dtype=torch.int32, device="cuda")
    other = tok.clone()
    other[1, 12:] = -1  # padding
    with torch.no_grad():
        a, b = m(tok, n), m(other, n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1, :12], b[1, :12])


def test_it_learns(cuda):
    """Copying the token before the last one: the loss falls to a third in 60 steps."""
    m = net()
    opt = torch.optim.AdamW(m.parameters(), lr=3e-3)
    first = last = None
    g = torch.Generator(device="cuda").manual_seed(0)
    for i in range(60):
        tok = torch.randint(0, 8, (16, 48), device="cuda", generator=g)
        loss = torch.nn.functional.cross_entropy(m(tok)[:, 1:].flatten(0, 1), tok[:, :-1].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        first = first if first is not None else loss.item()
        last = loss.item()
    assert last < first / 3, (first, last)
