"""What the sequence-model operators owe autograd and their callers, on both host paths (the C++
binding and the Python functions)."""
import time

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from hard_resets_compose_b200 import _lib, embed, leakyattn, normgate

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _LeaveAll:
    """A binding that takes no call."""
    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture(params=("binding", "python"))
def host(request, monkeypatch, cuda):
    if request.param == "python":
        monkeypatch.setattr(_lib, "fast", lambda: _LeaveAll())
    return request.param


def rand(*shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def test_a_cache_stepped_on_is_a_changed_tensor(host):
    """dq reads the state before the first token: a step on it in between is refused."""
    B, T, H, D = 2, 5, 3, 16
    q, k, v = (rand(B, T, H, D, seed=i) for i in range(3))
    ld, cache = -torch.ones(H, device=DEV), rand(B, H, D, D, seed=4)
    q.requires_grad_()
    o = leakyattn.leaky_attention(q, k, v, ld, state=cache)
    version = cache._version
    with torch.no_grad():
        leakyattn.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, cache)
    assert cache._version > version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_a_view_of_the_cache_counts_too(host):
    H, D = 2, 8
    big = rand(4, H + 1, D, D, seed=1)
    q = rand(3, H, D, seed=2)
    version = big._version
    leakyattn.leaky_attention_step(q, q, q, -torch.ones(H, device=DEV), big[:, 1:])
    assert big._version > version


def test_a_cache_made_in_inference_mode(host):
    """It has no version; the step takes it inside the mode and outside."""
    H, D = 2, 8
    q, ld = rand(3, H, D, seed=2), -torch.ones(H, device=DEV)
    with torch.inference_mode():
        cache = rand(3, H, D, D, seed=1)
        leakyattn.leaky_attention_step(q, q, q, ld, cache)
    want = rand(3, H, D, D, seed=1)
    for _ in range(2):
        leakyattn.leaky_attention_step(q, q, q, ld, want)
    leakyattn.leaky_attention_step(q, q, q, ld, cache)
    assert torch.equal(cache, want)


CALLS = {
    "embedding": lambda d: embed.embedding(torch.arange(4, device=DEV), d(4, 8)),
    "norm_x": lambda d: normgate.norm_gate_residual(d(4, 8), rand(4, 8, seed=2), None, rand(8, seed=3), rand(8, seed=4)),
    "norm_h": lambda d: normgate.norm_gate_residual(rand(4, 8, seed=2), d(4, 8), None, rand(8, seed=3)),
    "norm_gate": lambda d: normgate.norm_gate_residual(rand(4, 8, seed=2), rand(4, 8, seed=5), d(4, 1), rand(8, seed=3)),
    "norm_post": lambda d: normgate.norm_gate_residual(rand(4, 8, seed=2), rand(4, 8, seed=5), None, d(8)),
    "rms_norm": lambda d: normgate.rms_norm(rand(4, 8, seed=2), d(8)),
    "attention_q": lambda d: leakyattn.leaky_attention(d(2, 4, 2, 8), *(rand(2, 4, 2, 8, seed=i) for i in (1, 2)),
                                                       -torch.ones(2, device=DEV)),
    "attention_decay": lambda d: leakyattn.leaky_attention(*(rand(2, 4, 2, 8, seed=i) for i in (1, 2, 3)), d(2)),
    "attention_state": lambda d: leakyattn.leaky_attention(*(rand(2, 4, 2, 8, seed=i) for i in (1, 2, 3)),
                                                           -torch.ones(2, device=DEV), state=d(2, 2, 8, 8)),
    "step_v": lambda d: leakyattn.leaky_attention_step(rand(2, 2, 8, seed=1), rand(2, 2, 8, seed=2), d(2, 2, 8),
                                                       -torch.ones(2, device=DEV), rand(2, 2, 8, 8, seed=3)),
    "step_state": lambda d: leakyattn.leaky_attention_step(*(rand(2, 2, 8, seed=i) for i in (1, 2, 3)),
                                                           -torch.ones(2, device=DEV), d(2, 2, 8, 8)),
}


@pytest.mark.parametrize("grad", (True, False))
@pytest.mark.parametrize("call", sorted(CALLS))
def test_tangents_are_refused(host, call, grad):
    """No operator has a forward-mode derivative: a dual tensor is refused, not stripped."""
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        def dual(*shape):
            return fwAD.make_dual(-rand(*shape, seed=7).abs(), rand(*shape, seed=8))
        with pytest.raises(RuntimeError, match="forward-mode"):
            CALLS[call](dual)
        CALLS[call](lambda *shape: -rand(*shape, seed=7).abs())  # without a tangent it runs


def test_overlapping_caches_are_refused(host):
    """Slots or heads that share memory would be written by two sequences at once."""
    H, D = 2, 8
    q, ld = rand(3, H, D, seed=2), -torch.ones(2, device=DEV)
    for state in (rand(1, H, D, D, seed=1).expand(3, H, D, D), rand(3, 1, D, D, seed=1).expand(3, H, D, D),
                  torch.zeros(4 * H * D * D, device=DEV).as_strided((3, H, D, D), (D * D, D * D, D, 1))):
        with pytest.raises((ValueError, RuntimeError), match="share memory"):
            leakyattn.leaky_attention_step(q, q, q, ld, state)


def test_caches_in_other_orders(host):
    """Heads before slots, and slots between the heads of others: nothing overlaps."""
    n, H, D = 3, 2, 8
    q, ld, x = rand(n, H, D, seed=2), -torch.ones(2, device=DEV), rand(n, H, D, D, seed=1)
    want = x.clone()
    o = leakyattn.leaky_attention_step(q, q, q, ld, want)
    for strides in ((D * D, n * D * D), (2 * D * D, 7 * D * D)):
        cache = torch.zeros(20 * D * D, device=DEV).as_strided((n, H, D, D), (*strides, D, 1))
        cache.copy_(x)
        assert torch.equal(leakyattn.leaky_attention_step(q, q, q, ld, cache), o) and torch.equal(cache, want)


def test_bf16_models_run_as_they_come(host):
    """SeqNet(...).bfloat16() without a word to its buffers."""
    from hard_resets_compose_b200.seqnet import SeqNet
    torch.manual_seed(3)
    net = SeqNet(vocab=50, width=64, heads=4, layers=2).cuda().bfloat16()
    tok = torch.randint(0, 50, (3, 20), device=DEV)
    net(tok).float().sum().backward()
    cache, slots = net.new_cache(4), torch.tensor([1, 0, 3], dtype=torch.int32, device=DEV)
    n = torch.tensor([20, 3, 7], dtype=torch.int32, device=DEV)
    assert torch.isfinite(net.prompt(tok, cache, slots, n)).all()
    assert torch.isfinite(net.step(tok[:, 0], cache, slots)).all()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_the_model_leaves_empty_places_alone(host, dtype):
    """Prompts and steps of a batch with an empty place: the bits of the same batch with a place for
    it, and nothing else in the cache changes."""
    from hard_resets_compose_b200.seqnet import SeqNet
    torch.manual_seed(3)
    net = SeqNet(vocab=50, width=64, heads=4, layers=2, kv_heads=2).cuda().to(dtype)
    tok = torch.randint(0, 50, (3, 20), device=DEV)
    n = torch.tensor([20, 3, 7], dtype=torch.int32, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731

    def filled():
        torch.manual_seed(4)
        return [tuple(torch.randn_like(t) for t in pair) for pair in net.new_cache(5)]
    start, all_there, one_empty = filled(), filled(), filled()
    for slots, empty in ((i32(2, 0, 4), i32(2, -1, 4)), (i32(0, 3, 1), i32(5, 3, 1))):
        live = empty.clamp(0, 4) == empty
        for out, got in ((net.prompt(tok, all_there, slots, n), net.prompt(tok, one_empty, empty, n)),
                         (net.step(tok[:, 0], all_there, slots), net.step(tok[:, 0], one_empty, empty))):
            assert torch.equal(out[live], got[live])
    for a, b, was in zip(all_there, one_empty, start):
        for x, y, w in zip(a, b, was):
            assert torch.equal(x[1:], y[1:]) and torch.equal(y[0], w[0])
    before = [tuple(t.clone() for t in pair) for pair in one_empty]
    assert not net.step(tok[:, 0], one_empty, i32(-1, 5, 99)).any()
    assert all(torch.equal(x, y) for p, q in zip(before, one_empty) for x, y in zip(p, q))


def test_device_errors_reach_inference(host):
    """A token past the table, in a program that never runs a backward."""
    x, w = rand(4, 8, seed=1), rand(8, seed=2)
    q, ld, state = rand(2, 2, 8, seed=3), -torch.ones(2, device=DEV), rand(2, 2, 8, 8, seed=4)
    table, good = rand(10, 8, seed=5), torch.tensor([1], device=DEV)
    calls = (lambda: embed.embedding(good, table), lambda: normgate.rms_norm(x, w),
             lambda: leakyattn.leaky_attention_step(q, q, q, ld, state),
             lambda: leakyattn.leaky_attention(q[None], q[None], q[None], ld))
    _lib.check_device("before")
    for call in calls:
        embed.embedding(torch.tensor([99], device=DEV), table)
        torch.cuda.synchronize()
        try:
            with pytest.raises(_lib.LifbError) as e:
                for _ in range(5):
                    call()
                    torch.cuda.synchronize()
                    time.sleep(0.03)
            assert e.value.device_code == 102
        finally:
            with pytest.raises(_lib.LifbError):
                _lib.check_device("after", reset=True)
        _lib.check_device("cleared")


def test_a_step_that_reports_an_error_has_not_run(host):
    table = rand(10, 8, seed=5)
    q, ld, state = rand(2, 2, 8, seed=3), -torch.ones(2, device=DEV), rand(2, 2, 8, 8, seed=4)
    _lib.check_device("before")
    embed.embedding(torch.tensor([99], device=DEV), table)
    torch.cuda.synchronize()
    raised = False
    try:
        for _ in range(5):
            was = state.clone()
            try:
                leakyattn.leaky_attention_step(q, q, q, ld, state)
            except _lib.LifbError:
                raised = True
                assert torch.equal(state, was)
                break
            assert not torch.equal(state, was)
            time.sleep(0.03)
    finally:
        with pytest.raises(_lib.LifbError):
            _lib.check_device("after", reset=True)
    assert raised


def _layouts(B, T, H, D, dtype, seed):
    """The same values dense, and in layouts that a tensor map refuses."""
    x = rand(B, T, H, D, seed=seed, dtype=dtype)
    wide = torch.zeros(B, T, H, D + 1, device=DEV, dtype=dtype)
    wide[..., :D] = x
    off = torch.zeros(x.numel() + 1, device=DEV, dtype=dtype)[1:].view_as(x)
    off.copy_(x)
    return x, {"row": wide[..., :D], "address": off}


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("which", ("q", "k", "v", "do"))
@pytest.mark.parametrize("layout", ("row", "address"))
def test_layouts_do_not_choose_the_kernel(host, dtype, which, layout):
    """Operands off the 16-byte grid: the bits of the same call with dense operands."""
    B, T, H, D = 2, 200, 2, 64
    ld = -torch.tensor([0.1, 0.01], device=DEV)
    t = {n: _layouts(B, T, H, D, dtype, i) for i, n in enumerate(("q", "k", "v", "do"))}

    def run(odd):
        a = {n: (x[1][layout] if odd and n == which else x[0]) for n, x in t.items()}
        p = [a[n].detach().requires_grad_() for n in ("q", "k", "v")]
        o, s = leakyattn.leaky_attention(*p, ld, return_state=True)
        return (o, s, *torch.autograd.grad(o, p, a["do"]))
    for x, y in zip(run(True), run(False)):
        assert x.shape == y.shape and torch.equal(x, y)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_expanded_heads_and_gradients(host, dtype):
    """One key/value head expanded to all, and the gradient of a sum over time."""
    B, T, H, D = 2, 200, 4, 64
    q, k, v = rand(B, T, H, D, seed=1, dtype=dtype), rand(B, T, 1, D, seed=2, dtype=dtype), rand(B, T, 1, D, seed=3, dtype=dtype)
    ld, g = -torch.linspace(0.01, 0.2, H, device=DEV), rand(B, H, D, seed=4, dtype=dtype)

    def run(dense):
        fit = (lambda x: x.contiguous()) if dense else (lambda x: x)
        p = [x.detach().requires_grad_() for x in (q, fit(k.expand(B, T, H, D)), fit(v.expand(B, T, H, D)))]
        o = leakyattn.leaky_attention(*p, ld)
        return (o, *torch.autograd.grad(o, p, fit(g[:, None].expand(B, T, H, D))))
    for x, y in zip(run(False), run(True)):
        assert torch.equal(x, y)


def test_one_token_at_an_odd_distance(host):
    """T = 1: the distance between tokens is never used."""
    B, H, D = 3, 2, 64
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.zeros(B * H * D, device=DEV, dtype=dtype)
        x.copy_(rand(B * H * D, seed=1, dtype=dtype))
        odd = x.as_strided((B, 1, H, D), (H * D, 7, D, 1))
        ld = -torch.ones(H, device=DEV)
        assert torch.equal(leakyattn.leaky_attention(odd, odd, odd, ld), leakyattn.leaky_attention(*(x.view(B, 1, H, D),) * 3, ld))


@pytest.mark.parametrize("act", ("silu", "sigmoid"))
@pytest.mark.parametrize("gate", ("full", "row"))
def test_fp32_gates_far_from_zero(host, act, gate):
    """fp32: sigmoid to a few ulps wherever it is not subnormal, also where |gate| is large.  One row
    of D = 1 columns leaves x' = act(g) * +-1 (h = 2, eps = 0): relative error below 16 2^-24
    (exp 2 ulps, sum, quotient and products: 8 roundings, each at most 2^-23)."""
    g = torch.linspace(-80.0, 80.0, 4001, device=DEV)[:, None]
    if gate == "full":
        g = torch.cat((g, g.flip(0)), 1)
    D = g.shape[1] if gate == "full" else 2
    h, x = torch.full((4001, D), 2.0, device=DEV), torch.zeros(4001, D, device=DEV)
    got = normgate.norm_gate_residual(x, h, g, torch.ones(D, device=DEV), act=act, eps=0.0).double()
    s = torch.sigmoid(g.double())
    want = (s * g.double() if act == "silu" else s).expand(4001, D)
    assert ((got - want).abs() <= 16 * 2.0 ** -24 * want.abs() + 1e-37).all()
    # and its derivative: sum over the row of 1 * (+-1) * act'(g)
    gq = g.clone().requires_grad_()
    got, = torch.autograd.grad(normgate.norm_gate_residual(x, h, gq, torch.ones(D, device=DEV), act=act, eps=0.0).sum(), gq)
    d = s * (1 - s) if act == "sigmoid" else s * (1 + g.double() * (1 - s))
    want = d if gate == "full" else d * D
    # 1 - s loses what s has rounded away near 1: an absolute 2^-24 of the larger term
    near = 2.0 ** -22 * (s if act == "sigmoid" else s * (1 + g.double().abs())) * (1 if gate == "full" else D)
    assert ((got.double() - want).abs() <= 16 * 2.0 ** -24 * want.abs() + near + 1e-37).all()


def test_the_model_under_autocast(host):
    """Linear layers in bf16 around an fp32 stream.  Without spikes (a threshold that nothing reaches), whose
    flips would be large, some ten values on the way to a logit are rounded to bf16, 2^-8 each: below 2^-4."""
    from hard_resets_compose_b200.seqnet import SeqNet
    from tests.seq_refs import rel
    torch.manual_seed(3)
    net = SeqNet(vocab=50, width=64, heads=4, layers=1).cuda()
    net.theta = 1e9
    tok = torch.randint(0, 50, (3, 40), device=DEV)
    want = net(tok)
    with torch.autocast("cuda", torch.bfloat16):
        got = net(tok)
        got.float().sum().backward()
    assert rel(got, want) < 2.0 ** -4 and all(torch.isfinite(p.grad).all() for p in net.parameters())



def test_the_model_without_tokens(host):
    """No sequence, and sequences without a token, in every form of the model."""
    from hard_resets_compose_b200.seqnet import SeqNet
    net = SeqNet(vocab=50, width=64, heads=4, layers=2).cuda()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    tok, cache = torch.zeros(2, 0, dtype=torch.long, device=DEV), net.new_cache(3)
    for t in (tok, tok[:0], torch.zeros(0, 5, dtype=torch.long, device=DEV)):
        out = net(t)
        assert out.shape == (*t.shape, 50)
        out.sum().backward()
        assert not any(p.grad is not None and p.grad.any() for p in net.parameters())
    assert not net.prompt(tok, cache, i32(0, 2), i32(0, 0)).any()
    assert net.prompt(tok[:0], cache, i32(), i32()).shape == (0, 50)
    assert net.prompt(torch.zeros(0, 5, dtype=torch.long, device=DEV), cache, i32(), i32()).shape == (0, 50)
    assert net.step(torch.zeros(0, dtype=torch.long, device=DEV), cache, i32()).shape == (0, 50)


def test_calls_are_captured_into_graphs(host):
    """The status is not polled inside a capture (even where a poll is due), and replays give the same bits."""
    B, T, H, D = 2, 150, 2, 64
    q, k, v = (rand(B, T, H, D, seed=i, dtype=torch.bfloat16) for i in range(3))
    ld, w, table = -torch.ones(H, device=DEV), rand(D, seed=4), rand(10, D, seed=5)
    tok, state = torch.arange(6, device=DEV), rand(B, H, D, D, seed=6)

    def run(s):
        return (*leakyattn.leaky_attention(q, k, v, ld, state=state, return_state=True),
                leakyattn.leaky_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s), normgate.rms_norm(q, w),
                embed.embedding(tok, table), s)
    want = run(state.clone())
    s, side = state.clone(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(s)  # warm up
    torch.cuda.current_stream().wait_stream(side)
    time.sleep(0.03)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run(s)
    s.copy_(state)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
