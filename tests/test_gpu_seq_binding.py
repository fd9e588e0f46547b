"""The host binding of the sequence-model operators: the same bits, gradients and errors
as the Python functions behind it, over layouts that it takes and that it leaves to them."""
import pytest
import torch

from hard_resets_compose_b200 import _lib, embed, leakyattn, normgate

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _LeaveAll:
    """A binding that takes no call."""
    def __getattr__(self, name):
        return lambda *a: None


def both(monkeypatch, run):
    """run() through the binding and through the Python functions."""
    taken = []
    real = _lib.fast()

    class Watch:
        def __getattr__(self, name):
            def call(*a):
                out = getattr(real, name)(*a)
                taken.append(out is not None)
                return out
            return call
    monkeypatch.setattr(_lib, "fast", lambda: Watch())
    a = run()
    monkeypatch.setattr(_lib, "fast", lambda: _LeaveAll())
    b = run()
    monkeypatch.undo()
    return a, b, taken


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y)


def rand(*shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def test_binding_is_the_path_that_runs():
    w, t = rand(10, 8, seed=0), torch.arange(10, device=DEV)
    assert torch.equal(_lib.fast().embedding(t, w, 1.0), w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(7,), (3, 5), (0,)])
def test_embedding(monkeypatch, dtype, shape):
    w = rand(11, 24, seed=1, dtype=dtype)
    t = torch.randint(-1, 11, shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    dy = rand(*shape, 32, seed=3, dtype=dtype)[..., :24]

    def run():
        p = w.clone().requires_grad_(True)
        y = embed.embedding(t, p, 1.5)
        return (y.detach(), *torch.autograd.grad(y, p, dy))
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [True]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "row", "split", "dense"])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("needs", ["all", "x post", "h"])
def test_norm(monkeypatch, dtype, gate, pre, needs):
    T, B, D = 5, 3, 40
    t = {"x": rand(T, B, D, seed=1, dtype=dtype), "h": rand(T, B, D, seed=2, dtype=dtype),
         "gate": {"none": None, "row": rand(T, B, 1, seed=3, dtype=dtype),
                  "split": rand(T, B, 2 * D, seed=3, dtype=dtype).split(D, -1)[1],
                  "dense": rand(T, B, D, seed=3, dtype=dtype)}[gate],
         "post": rand(D, seed=4), "pre": rand(D, seed=5) if pre else None}
    g = rand(T, B, D, seed=6, dtype=dtype), rand(T, B, 2 * D, seed=7, dtype=dtype)[..., :D]

    def run():
        p = {k: None if v is None else v.detach() for k, v in t.items()}
        for k, v in p.items():
            if v is not None:
                v.requires_grad_(needs == "all" or k in needs.split())
        out = normgate.norm_gate_residual(p["x"], p["h"], p["gate"], p["post"], p["pre"], 0.5, "silu")
        out = out if pre else (out,)
        wanted = [v for v in p.values() if v is not None and v.requires_grad]
        return (*(o.detach() for o in out), *torch.autograd.grad(out, wanted, g[:len(out)]))
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [True]


@pytest.mark.parametrize("use", ["x", "n"])
def test_norm_gradient_of_one_output(monkeypatch, use):
    x, h, w = rand(6, 16, seed=1), rand(6, 16, seed=2), rand(16, seed=3)

    def run():
        p = [t.clone().requires_grad_(True) for t in (x, h, w, w)]
        xo, n = normgate.norm_gate_residual(p[0], p[1], None, p[2], p[3])
        return torch.autograd.grad((xo if use == "x" else n).sum(), p, allow_unused=True)
    a, b, _ = both(monkeypatch, run)
    same(a, b)


def test_rms_norm(monkeypatch):
    x, w = rand(4, 9, 64, seed=1).transpose(0, 1), rand(64, seed=2)  # its rows are not one list

    def run():
        p, q = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
        n = normgate.rms_norm(p, q)
        return (n.detach(), *torch.autograd.grad(n.sum(), (p, q)))
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [False]
    x = x.contiguous()
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [True]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("used", ["o", "state", "both"])
def test_attention(monkeypatch, dtype, state, used):
    B, T, H, Hk, Dk, Dv = 2, 150, 4, 2, 32, 64
    q, v = rand(B, T, H, Dk, seed=1, dtype=dtype), rand(B, T, Hk, Dv, seed=3, dtype=dtype)
    k = rand(B, T, 2 * Hk, Dk, seed=2, dtype=dtype)[:, :, ::2]
    ld = -torch.rand(H, generator=torch.Generator().manual_seed(4)).to(DEV)
    s0 = rand(B, H, Dk, Dv, seed=5) if state else None
    lengths = torch.tensor([T, 77], dtype=torch.int32, device=DEV) if state else None
    do, ds = rand(B, H, T, Dv, seed=6, dtype=dtype).transpose(1, 2), rand(B, H, Dk, Dv, seed=7)

    def run():
        p = [None if t is None else t.detach().requires_grad_(True) for t in (q, k, v, s0)]
        o, out = leakyattn.leaky_attention(p[0], p[1], p[2], ld, p[3], lengths, return_state=True)
        outs, gs = {"o": ((o,), (do,)), "state": ((out,), (ds,)), "both": ((o, out), (do, ds))}[used]
        g = torch.autograd.grad(outs, [t for t in p if t is not None], gs, allow_unused=True)
        return (o.detach(), out.detach(), *g)
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [True]


def test_attention_step(monkeypatch):
    B, H, Hk, D = 3, 4, 2, 32
    q, k, v = (rand(B, h, D, seed=i) for i, h in enumerate((H, Hk, Hk)))
    ld, s0 = -torch.ones(H, device=DEV), rand(5, H, D, D, seed=4)
    slots = torch.tensor([4, -1, 0], dtype=torch.int32, device=DEV)

    def run():
        s = s0.clone()
        return leakyattn.leaky_attention_step(q, k, v, ld, s, slots), s
    a, b, taken = both(monkeypatch, run)
    same(a, b)
    assert taken == [True]


def test_a_graph_of_the_gradient_is_refused_only_when_differentiated():
    w, t = rand(10, 8, seed=0).requires_grad_(True), torch.arange(10, device=DEV)
    y = embed.embedding(t, w)
    g, = torch.autograd.grad((y * y).sum(), w, create_graph=True)
    torch.testing.assert_close(g.detach(), 2 * w.detach(), rtol=0, atol=0)
    with pytest.raises(RuntimeError, match="not differentiable"):
        g.sum().backward()


def test_a_saved_input_changed_in_place_is_refused():
    x, w = rand(4, 16, seed=1).requires_grad_(True), rand(16, seed=2).requires_grad_(True)
    n = normgate.rms_norm(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.sum().backward()


def test_device_error_reaches_the_caller_of_the_backward():
    """A token past the table, reported by the poll in a later backward."""
    import time
    w = rand(10, 8, seed=0).requires_grad_(True)
    bad, good = torch.tensor([99], device=DEV), torch.tensor([1], device=DEV)
    _lib.check_device("before")
    embed.embedding(bad, w.detach())
    torch.cuda.synchronize()
    try:
        with pytest.raises(_lib.LifbError) as e:
            for _ in range(5):
                embed.embedding(good, w).sum().backward()
                torch.cuda.synchronize()
                time.sleep(0.03)
        assert e.value.device_code == 102
    finally:
        with pytest.raises(_lib.LifbError):
            _lib.check_device("after", reset=True)
    _lib.check_device("cleared")
