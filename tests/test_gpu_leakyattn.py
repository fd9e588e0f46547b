"""Leaky attention (csrc/leaky_attn.cu, csrc/leaky_attn_tc.cu) against the
recurrence in 64 bits.

Bounds, elementwise, against the same recurrence on the operands' absolute
values, A (o is a sum of products q k v of A's size at most):
fp32: a product passes through at most Dk + Dv + 32 additions within a chunk,
one addition and one multiplication a chunk after it, and two powers of the
decay whose exponent n l2 carries 2 roundings (at most 24 * 2^-23 each where
the power is not negligible): (Dk + Dv + T / 16 + 200) 2^-24 A.
bf16: the scores of a chunk and the carried state enter their products rounded
to bf16 (u A, u = 2^-8 half an ulp), once each, and the output is rounded
(u A); a state is not rounded (its weights are split so that 24 bits of each
key stay): 2 u A + the fp32 bound for outputs, the fp32 bound for states (the tensor cores drop
bits of aligned sums: twice it)."""
import pytest
import torch

from tests.seq_refs import U, attention

pytestmark = pytest.mark.gpu


def make(B, T, H, Hk, Dk, Dv, dtype, state, ragged, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + B + 3 * T + 5 * H + 7 * Dk + 11 * Dv)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, v = rnd(B, T, H, Dk).to(dtype), (rnd(B, T, Hk, Dk) * Dk ** -0.5).to(dtype), (rnd(B, T, Hk, Dv) + 0.1).to(dtype)
    ld = torch.log1p(-torch.exp2(-torch.linspace(0.5, 13, H, device="cuda")))
    ld[-1] = 0.0
    if H > 2:
        ld[1] = -float("inf")
    st = rnd(B, H, Dk, Dv) if state else None
    ln = None
    if ragged:
        ln = torch.randint(0, T + 1, (B,), device="cuda", generator=g).int()
        ln[0] = T
        if B > 1:
            ln[-1] = 0
    return q, k, v, ld, st, ln, rnd(B, T, H, Dv).to(dtype), rnd(B, H, Dk, Dv)


def within(got, ref, mag, f32, factor, name):
    u = 2 * U[got.dtype] if got.dtype == torch.bfloat16 else 0.0
    err = (got.double() - ref).abs()
    bound = (u + factor * f32) * mag + 1e-30
    assert (err <= bound).all(), f"{name}: {(err / bound).max().item():.3g} times its bound"


def check(B, T, H, Hk, Dk, Dv, dtype, state, ragged, dstate=False, views=False):
    from hard_resets_compose_b200.leakyattn import leaky_attention
    q, k, v, ld, st, ln, do, ds = make(B, T, H, Hk, Dk, Dv, dtype, state, ragged)
    ds = ds if dstate else None
    if views:  # time before batch, heads before time, a slice of a wider tensor
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.randn(B, T, Hk, Dv + 16, device="cuda").to(dtype)
        wide[..., 8:8 + Dv] = v
        v = wide[..., 8:8 + Dv]
        do = do.transpose(0, 1).contiguous().transpose(0, 1)
    if ragged:  # what lies past a sequence's end is not read
        past = torch.arange(T, device="cuda")[None] >= ln[:, None]
        for t in (q, k, v, do):
            t[past] = float("nan")
    qa, ka, va = (t.detach().requires_grad_() for t in (q, k, v))
    sa = None if st is None else st.clone().requires_grad_()
    o, out = leaky_attention(qa, ka, va, ld, state=sa, lengths=ln, return_state=True)
    wrt = [qa, ka, va] + ([sa] if state else [])
    gr = torch.autograd.grad([o] + ([out] if dstate else []), wrt, [do] + ([ds] if dstate else []))
    if ragged:
        q, k, v, do = (torch.nan_to_num(t, nan=0.0) for t in (q, k, v, do))
    ref = attention(q, k, v, ld, st, ln, do=do, dstate=ds)
    ab = lambda t: None if t is None else t.abs()  # noqa: E731
    mag = attention(q.abs(), k.abs(), v.abs(), ld, ab(st), ln, do=do.abs(), dstate=ab(ds))
    f32 = (Dk + Dv + T / 16 + 200) * 2.0 ** -24 * (H // Hk)
    tc = 2 if dtype == torch.bfloat16 else 1
    for name, got, r, m in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, out) + gr, ref, mag):
        assert got.shape == r.shape
        within(got, r, m, f32, tc, name)
    with torch.no_grad():
        o2 = leaky_attention(q, k, v, ld, state=st, lengths=ln)
    assert o2.shape == o.shape
    return o


SIZES = ((1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 3, 5), (1, 31, 3, 3, 16, 16), (3, 33, 2, 2, 64, 64), (2, 128, 4, 2, 64, 64),
         (2, 129, 3, 1, 40, 48), (1, 257, 4, 4, 128, 128), (2, 300, 2, 1, 128, 64), (1, 500, 3, 3, 64, 128),
         (4, 100, 6, 2, 72, 112), (1, 1100, 2, 2, 32, 32), (2, 383, 3, 3, 17, 100), (1, 2000, 1, 1, 96, 80))


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("size", SIZES)
def test_forward_backward(cuda, dtype, size):
    check(*size, dtype, state=False, ragged=False)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("size", SIZES[1:])
def test_states_and_lengths(cuda, dtype, size):
    check(*size, dtype, state=True, ragged=True, dstate=True)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("size", ((2, 140, 4, 2, 64, 64), (2, 70, 3, 3, 24, 20), (1, 300, 4, 4, 128, 128)))
def test_other_orders(cuda, dtype, size):
    check(*size, dtype, state=True, ragged=False, views=True)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_many_chains(cuda, dtype):
    """More chains than blocks the GPU holds: no time segments."""
    check(40, 150, 8, 8, 64, 64, dtype, state=False, ragged=True)


def test_a_prompt_in_parts_and_in_steps(cuda):
    """A prompt at once, in two parts, and token by token: one recurrence."""
    from hard_resets_compose_b200.leakyattn import leaky_attention, leaky_attention_step
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, ld, st, _, _, _ = make(3, 200, 4, 2, 64, 48, dtype, True, False)
        with torch.no_grad():
            o, s = leaky_attention(q, k, v, ld, state=st, return_state=True)
            o1, s1 = leaky_attention(q[:, :77], k[:, :77], v[:, :77], ld, state=st, return_state=True)
            o2, s2 = leaky_attention(q[:, 77:], k[:, 77:], v[:, 77:], ld, state=s1, return_state=True)
            cache = st.clone()
            o3 = torch.stack([leaky_attention_step(q[:, t], k[:, t], v[:, t], ld, cache) for t in range(200)], 1)
        ro, rs = attention(q, k, v, ld, st)
        mo, ms = attention(q.abs(), k.abs(), v.abs(), ld, st.abs())
        f32 = (64 + 48 + 200 + 200) * 2.0 ** -24
        for got in (o, torch.cat([o1, o2], 1), o3):
            within(got, ro, mo, f32, 2, "o")
        for got in (s, s2, cache):
            within(got, rs, ms, f32, 2, "state")


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", ((1, 1, 1, 1, 1), (1, 4, 4, 64, 64), (5, 6, 2, 33, 30), (3, 2, 1, 128, 128),
                                          (7, 3, 3, 16, 100), (2, 8, 4, 100, 20)))
def test_step(cuda, dtype, B, H, Hk, Dk, Dv):
    from hard_resets_compose_b200.leakyattn import leaky_attention_step
    q, k, v, ld, _, _, _, _ = make(B, 1, H, Hk, Dk, Dv, torch.float32, False, False)
    q, k, v = (t[:, 0].to(dtype) for t in (q, k, v))
    n = B + 3
    state = torch.randn(n, H, Dk, Dv, device="cuda")
    slots = torch.randperm(n, device="cuda")[:B].int()
    if B > 2:
        slots[1], slots[2] = -1, n + 5  # empty places
    cache = state.clone()
    o = leaky_attention_step(q, k, v, ld, cache, slots)
    live = ((slots >= 0) & (slots < n)).cpu()
    at = slots.long().clamp(0, n - 1)
    ro, rs = attention(q[:, None], k[:, None], v[:, None], ld, state[at])
    mo, ms = attention(q.abs()[:, None], k.abs()[:, None], v.abs()[:, None], ld, state[at].abs())
    f32 = (Dk + 16) * 2.0 ** -24
    u = 0.0 if dtype == torch.float32 else U[dtype]
    for i in range(B):
        if live[i]:
            assert ((o[i].double() - ro[i, 0]).abs() <= (u + f32) * mo[i, 0] + (2.0 ** -24 if dtype == torch.float16 else 0)).all()
            assert ((cache[slots[i]].double() - rs[i]).abs() <= 4 * 2.0 ** -24 * ms[i]).all()
        else:
            assert not o[i].any()
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at[live.cuda()]] = False
    assert torch.equal(cache[rest], state[rest])
    # a cache with other strides, operands that are slices
    wide = torch.zeros(n, H + 1, Dk, Dv, device="cuda")
    wide[:, 1:] = state
    qkv = torch.cat([q.reshape(B, -1), k.reshape(B, -1), v.reshape(B, -1)], 1)
    qs = qkv[:, :H * Dk].view(B, H, Dk)
    ks = qkv[:, H * Dk:H * Dk + Hk * Dk].view(B, Hk, Dk)
    vs = qkv[:, H * Dk + Hk * Dk:].view(B, Hk, Dv)
    o2 = leaky_attention_step(qs, ks, vs, ld, wide[:, 1:], slots)
    assert torch.allclose(o2.float(), o.float(), rtol=2 * u + 1e-5, atol=1e-5)
    assert torch.allclose(wide[:, 1:], cache, rtol=1e-6, atol=1e-6)


def test_step_offsets_past_32_bits(cuda):
    """A cache of more than 2^31 elements: its last slots."""
    from hard_resets_compose_b200.leakyattn import leaky_attention_step
    n, H, D = 131073 + 40, 1, 128  # 2^31 elements and more, 8.6 GB
    state = torch.empty(n, H, D, D, device="cuda")
    state[-2:] = 1.0
    q, k, v, ld, _, _, _, _ = make(2, 1, H, H, D, D, torch.float32, False, False)
    ref, rs = attention(q, k, v, ld, torch.ones(2, H, D, D, device="cuda"))
    o = leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state, torch.tensor([n - 1, n - 2], device="cuda").int())
    assert torch.allclose(o.double(), ref[:, 0], rtol=1e-5, atol=1e-4)
    assert torch.allclose(state[-1].double(), rs[0], rtol=1e-6, atol=1e-6)
    del state
    torch.cuda.empty_cache()


def test_differences(cuda):
    """o is linear in q, in k, in v and in the state, so a central difference of
    any step is the derivative up to rounding."""
    from hard_resets_compose_b200.leakyattn import leaky_attention
    q, k, v, ld, st, _, do, _ = make(2, 90, 4, 2, 32, 24, torch.float32, True, False)
    f = lambda *t: leaky_attention(*t[:3], ld, state=t[3])  # noqa: E731
    ts = [q, k, v, st]
    leaves = [t.clone().requires_grad_() for t in ts]
    gr = torch.autograd.grad(f(*leaves), leaves, do)
    with torch.no_grad():
        for i, g in enumerate(gr):
            d = torch.randn_like(ts[i])
            up, dn, mg = list(ts), list(ts), [t.abs() for t in ts]
            up[i], dn[i], mg[i] = ts[i] + d, ts[i] - d, ts[i].abs() + d.abs()
            diff = ((f(*up) - f(*dn)).double() / 2 * do.double()).sum()
            mag = (f(*mg).double() * do.abs().double()).sum()
            assert abs(diff - (g.double() * d.double()).sum()) <= 400 * 2.0 ** -24 * mag


def test_runs_repeat_and_streams(cuda):
    from hard_resets_compose_b200.leakyattn import leaky_attention
    q, k, v, ld, st, ln, do, _ = make(2, 400, 4, 2, 64, 64, torch.bfloat16, True, True)
    runs = []
    side = torch.cuda.Stream()
    for i in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if i == 2 else torch.cuda.current_stream()):
            leaves = [t.clone().requires_grad_() for t in (q, k, v, st)]
            o = leaky_attention(*leaves[:3], ld, state=leaves[3], lengths=ln)
            runs.append((o.detach(),) + torch.autograd.grad(o, leaves, do))
        torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_non_finite_stays_in_its_head_and_after_its_token(cuda):
    from hard_resets_compose_b200.leakyattn import leaky_attention
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, ld, _, _, _, _ = make(2, 300, 2, 2, 64, 64, dtype, False, False)
        ld = torch.tensor([-0.1, -0.02], device="cuda")
        v[1, 150, 0, 3] = float("inf")
        o = leaky_attention(q, k, v, ld)
        assert torch.isfinite(o[0]).all() and torch.isfinite(o[1, :, 1]).all()
        assert torch.isfinite(o[1, :128, 0]).all()
        assert not torch.isfinite(o[1, 150:, 0, 3]).any()


def test_empty(cuda):
    from hard_resets_compose_b200.leakyattn import leaky_attention, leaky_attention_step
    q, k, v, ld, st, _, _, ds = make(2, 4, 2, 1, 8, 8, torch.float32, True, False)
    leaves = [t[:, :0].clone().requires_grad_() for t in (q, k, v)] + [st.clone().requires_grad_()]
    o, s = leaky_attention(*leaves[:3], ld, state=leaves[3], return_state=True)
    assert o.shape == (2, 0, 2, 8) and torch.equal(s, st)
    assert torch.equal(torch.autograd.grad(s, leaves[3], ds)[0], ds)
    o, s = leaky_attention(q[:0], k[:0], v[:0], ld, return_state=True)
    assert o.shape == (0, 4, 2, 8)
    none = leaky_attention(q, k, v, ld, lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert not none.any()
    assert leaky_attention_step(q[:0, 0], k[:0, 0], v[:0, 0], ld, st).shape == (0, 2, 8)


def test_refusals(cuda):
    from hard_resets_compose_b200.leakyattn import leaky_attention, leaky_attention_step
    q, k, v, ld, st, _, _, _ = make(2, 4, 2, 1, 8, 8, torch.float32, True, False)
    big = torch.zeros(1, 2, 1, 129, device="cuda")
    one = torch.zeros(1, device="cuda")
    for bad in (lambda: leaky_attention(q[0], k, v, ld), lambda: leaky_attention(q, k[:, :3], v, ld),
                lambda: leaky_attention(q, k[..., :4], v, ld), lambda: leaky_attention(q, k, v, ld[:1]),
                lambda: leaky_attention(q, k, v, ld.double()), lambda: leaky_attention(q, k, v, ld, state=st[:1]),
                lambda: leaky_attention(q, k, v, ld, state=st.half()),
                lambda: leaky_attention(q, k, v, ld, lengths=torch.zeros(2, device="cuda")),
                lambda: leaky_attention(big, big, big[..., :8], one),
                lambda: leaky_attention(q, k, v, ld.clone().requires_grad_()),
                lambda: leaky_attention(q, q.repeat(1, 1, 2, 1)[:, :, :3], v.repeat(1, 1, 3, 1), ld),
                lambda: leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st[:1]),
                lambda: leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st.transpose(2, 3)),
                lambda: leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st, torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: leaky_attention(q.half(), k.half(), v.half(), ld), lambda: leaky_attention(q, k.bfloat16(), v, ld)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        leaky_attention(q.cpu(), k.cpu(), v.cpu(), ld.cpu())
    with pytest.raises(RuntimeError):
        leaky_attention_step(q[:, 0].clone().requires_grad_(), k[:, 0], v[:, 0], ld, st)


@pytest.mark.parametrize("T", [1, 3, 11, 64, 127, 128])
@pytest.mark.parametrize("H,Hk,Dk,Dv", [(1, 1, 64, 64), (4, 1, 128, 32), (2, 2, 128, 128), (2, 1, 40, 72)])
def test_few_tokens_bf16_are_rounded_once(cuda, T, H, Hk, Dk, Dv):
    """One chunk or less: intermediate values have two bf16 pieces (2^-8 each, 2^-16 together), powers of the
    decay at most 2^-17 (128 products of 2^-24), the rest is fp32; 2^-15 of the sum of the terms' sizes covers
    them.  What is left is the output's own rounding (half an ulp, 2^-8)."""
    from hard_resets_compose_b200.leakyattn import leaky_attention
    g = torch.Generator(device=cuda).manual_seed(T * 1000 + H * 100 + Dk)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    q, k = rand(2, T, H, Dk).bfloat16(), rand(2, T, Hk, Dk).bfloat16()
    v, do = rand(2, T, Hk, Dv).bfloat16(), rand(2, T, H, Dv).bfloat16()
    s0, ds = rand(2, H, Dk, Dv), rand(2, H, Dk, Dv)
    ld = -torch.rand(H, generator=g, device=cuda)
    lengths = torch.tensor([T, (T + 1) // 2], dtype=torch.int32, device=cuda)
    p = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
    o, s = leaky_attention(p[0], p[1], p[2], ld, p[3], lengths, return_state=True)
    got = (o, *torch.autograd.grad((o, s), p[:3], (do, ds)))
    exact = attention(q, k, v, ld, s0, lengths, do=do, dstate=ds)
    sizes = attention(q.abs(), k.abs(), v.abs(), ld, s0.abs(), lengths, do=do.abs(), dstate=ds.abs())
    for name, a, e, z in zip(("o", "dq", "dk", "dv"), got, (exact[0], *exact[2:5]), (sizes[0], *sizes[2:5])):
        over = (a.double() - e).abs() - (U[torch.bfloat16] * e.abs() + 2.0 ** -15 * z)
        assert (over <= 0).all(), (name, over.max().item())
