"""bf16 leaky attention over few rows and several chunks: outputs rounded once."""
import pytest
import torch

from tests.seq_refs import U, attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,Hk", ((1, 129, 1, 1), (1, 200, 2, 1), (3, 256, 1, 1), (2, 383, 4, 2), (1, 1000, 3, 3),
                                      (1, 2000, 4, 1)))
@pytest.mark.parametrize("Dk,Dv", ((64, 64), (128, 32), (40, 72), (128, 128), (16, 16)))
def test_few_rows_bf16_are_rounded_once(cuda, B, T, H, Hk, Dk, Dv):
    """Up to 8192 tokens of heads: scores and states have two bf16 pieces (2^-16 together), powers of the decay
    at most 2^-17 (128 products of 2^-24), starting states of time segments 2^-18, the rest is fp32; 2^-15 of
    the sum of the terms' sizes covers them.  What is left is the output's own rounding (half an ulp, 2^-8)."""
    from hard_resets_compose_b200.leakyattn import leaky_attention
    g = torch.Generator(device=cuda).manual_seed(T * 1000 + H * 100 + Dk)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q, k = rand(B, T, H, Dk).bfloat16(), rand(B, T, Hk, Dk).bfloat16()
    v, do = rand(B, T, Hk, Dv).bfloat16(), rand(B, T, H, Dv).bfloat16()
    s0, ds = rand(B, H, Dk, Dv), rand(B, H, Dk, Dv)
    ld = torch.log1p(-torch.exp2(-torch.linspace(1, 10, H, device=cuda)))
    lengths = torch.tensor([T, (T + 1) // 2, 0][:B], dtype=torch.int32, device=cuda)
    p = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
    o, s = leaky_attention(p[0], p[1], p[2], ld, p[3], lengths, return_state=True)
    got = (o, *torch.autograd.grad((o, s), p[:3], (do, ds)))
    exact = attention(q, k, v, ld, s0, lengths, do=do, dstate=ds)
    sizes = attention(q.abs(), k.abs(), v.abs(), ld, s0.abs(), lengths, do=do.abs(), dstate=ds.abs())
    for name, a, e, z in zip(("o", "dq", "dk", "dv"), got, (exact[0], *exact[2:5]), (sizes[0], *sizes[2:5])):
        over = (a.double() - e).abs() - (U[torch.bfloat16] * e.abs() + 2.0 ** -15 * z)
        assert (over <= 0).all(), (name, over.max().item())
