"""Norms around a block with gate and residual (csrc/normgate.cu) against
64 bits.

Bound, relative (Frobenius) per output: a row's sums take at most 16 terms a
thread and 10 joining steps, so a mean is off by at most 26 2^-24, its rsqrt
by half that and two ulps; with the products and expf (2 ulps) around them
fewer than 64 roundings of 2^-24 reach a value: 4e-6; the sums over rows of
the weights' gradients add their own (R terms in groups, random in sign:
below 4e-6 at these sizes too).  The residual stream and the gradients can
cancel to a few times less than their terms: 1e-5.  An output of a 16-bit
type is rounded once more, by at most u."""
import pytest
import torch

from tests.seq_refs import U, norm_gate, rel

pytestmark = pytest.mark.gpu
TOL = 1e-5


def make(R, D, dtype, gate, wdtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed + R + 31 * D)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, h = rnd(R, D).to(dtype), (2 * rnd(R, D)).to(dtype)
    gt = None if gate == "none" else rnd(R, D if gate == "full" else 1).to(dtype)
    post, pre = (1 + 0.1 * rnd(D)).to(wdtype), (1 + 0.1 * rnd(D)).to(wdtype)
    return x, h, gt, post, pre, rnd(R, D).to(dtype), rnd(R, D).to(dtype)


def reference(ts, scale, act, eps, dx, dn):
    d = [None if t is None else t.detach().double().requires_grad_() for t in ts]
    xo, n = norm_gate(*d, scale, act, eps)
    outs, ups = zip(*[(o, u.double()) for o, u in ((xo, dx), (n, dn)) if o is not None and u is not None and o.requires_grad])
    live = [t for t in d if t is not None]
    grads = iter(torch.autograd.grad(outs, live, ups, allow_unused=True))
    return xo.detach(), None if n is None else n.detach(), [None if t is None else next(grads) for t in d]


def tol(t):
    return TOL + (U[t.dtype] if t.dtype != torch.float32 else 0.0)


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("R,D,gate,act", ((1, 1, "full", "silu"), (5, 3, "row", "sigmoid"), (33, 7, "full", "none"),
                                          (4, 64, "none", "silu"), (300, 256, "full", "silu"),
                                          (1500, 256, "row", "sigmoid"), (7, 257, "full", "sigmoid"),
                                          (20, 1000, "row", "silu"), (40, 1024, "full", "silu"),
                                          (9, 2050, "full", "silu"), (700, 2048, "full", "silu"),
                                          (3, 4672, "row", "none"), (11, 4096, "none", "silu"), (5, 5001, "full", "silu"),
                                          (2, 8192, "full", "sigmoid"), (3, 8191, "full", "silu")))
def test_against_fp64(cuda, dtype, R, D, gate, act):
    from hard_resets_compose_b200.normgate import norm_gate_residual
    wdtype = torch.float32 if R % 2 else dtype
    *ts, dx, dn = make(R, D, dtype, gate, wdtype)
    leaves = [None if t is None else t.clone().requires_grad_() for t in ts]
    x, n = norm_gate_residual(*leaves, residual_scale=0.5, act=act, eps=1e-5)
    live = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad((x, n), live, (dx, dn)))
    rx, rn, rg = reference(ts, 0.5, act, 1e-5, dx, dn)
    assert rel(x, rx) <= tol(x) and rel(n, rn) <= tol(n)
    for name, t, want in zip(("x", "h", "gate", "post", "pre"), leaves, rg):
        if t is None:
            continue
        got = next(grads)
        assert got.dtype == t.dtype and got.shape == t.shape
        # D = 1: rmsnorm is +-1 almost exactly, so its gradient is what cancellation leaves
        if D > 1 or name not in ("h", "x", "gate"):
            assert rel(got, want) <= tol(got), name
    # the forward without gradients gives the same bits
    with torch.no_grad():
        x2, n2 = norm_gate_residual(*ts, residual_scale=0.5, act=act, eps=1e-5)
    assert torch.equal(x, x2) and torch.equal(n, n2)


@pytest.mark.parametrize("which", ("no pre", "rms_norm", "only dx", "only dn"))
def test_parts(cuda, which):
    from hard_resets_compose_b200.normgate import norm_gate_residual, rms_norm
    x, h, g, post, pre, dx, dn = make(77, 96, torch.float32, "full", torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, h, g, post, pre)]
    if which == "rms_norm":
        n = rms_norm(leaves[0], leaves[4], eps=1e-6)
        got = torch.autograd.grad(n, [leaves[0], leaves[4]], dn)
        d = [x.double().requires_grad_(), pre.double().requires_grad_()]
        rn = norm_gate(d[0], None, None, None, d[1], 1.0, "silu", 1e-6)[1]
        want = torch.autograd.grad(rn, d, dn.double())
        assert rel(n, rn.detach()) <= TOL
        assert all(rel(a, b) <= TOL for a, b in zip(got, want))
        return
    if which == "no pre":
        xo = norm_gate_residual(*leaves[:4], residual_scale=0.7)
        got = torch.autograd.grad(xo, leaves[:4], dx)
        _, _, want = reference([x, h, g, post, None], 0.7, "silu", 1e-6, dx, None)
    else:
        xo, n = norm_gate_residual(*leaves, residual_scale=0.7)
        ups = (dx, None) if which == "only dx" else (None, dn)
        got = torch.autograd.grad(xo if ups[0] is not None else n, leaves, ups[0] if ups[0] is not None else ups[1],
                                  allow_unused=True)
        _, _, want = reference([x, h, g, post, pre], 0.7, "silu", 1e-6, *ups)
    for a, b in zip(got, want):
        assert (a is None or not a.any()) if b is None else rel(a, b) <= TOL


def test_difference(cuda):
    """x' is linear in x and in post_weight: a central difference of any step is
    exact up to rounding; h and the gate by a small step in 64 bits are the
    reference's gradients already."""
    from hard_resets_compose_b200.normgate import norm_gate_residual
    x, h, g, post, pre, dx, _ = make(64, 48, torch.float32, "full", torch.float32)
    d = torch.randn_like(post)
    p = post.clone().requires_grad_()
    dp, = torch.autograd.grad(norm_gate_residual(x, h, g, p), p, dx)
    with torch.no_grad():
        diff = ((norm_gate_residual(x, h, g, post + d) - norm_gate_residual(x, h, g, post - d)).double() / 2 * dx.double()).sum()
        mag = (norm_gate_residual(x.abs(), h.abs(), g.abs(), post.abs() + d.abs(), act="none").double() * dx.abs().double()).sum()
    assert abs(diff - (dp.double() * d.double()).sum()) <= 1e-5 * mag


def test_strides_and_streams(cuda):
    from hard_resets_compose_b200.normgate import norm_gate_residual, rms_norm
    x, h, g, post, pre, dx, dn = make(24, 40, torch.bfloat16, "full", torch.bfloat16)
    ref = norm_gate_residual(x, h, g, post, pre)
    big = torch.randn(24, 200, device="cuda").to(torch.bfloat16)
    big[:, 8:48], big[:, 48:88], big[:, 88:128] = x, h, g
    got = norm_gate_residual(big[:, 8:48], big[:, 48:88], big[:, 88:128], post, pre)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    odd = torch.empty(24, 41, dtype=torch.bfloat16, device="cuda")
    odd[:, 1:] = x  # rows that are not 16-byte aligned take the element form: the same sums in another order
    got = norm_gate_residual(odd[:, 1:], h, g, post, pre)
    assert rel(got[0], ref[0]) <= 2 * tol(x) and rel(got[1], ref[1]) <= 2 * tol(x)
    three = norm_gate_residual(x.view(2, 12, 40), h.view(2, 12, 40), g.view(2, 12, 40), post, pre)
    assert torch.equal(three[1].view(24, 40), ref[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = norm_gate_residual(x, h, g, post, pre)
    side.synchronize()
    assert torch.equal(s[0], ref[0])
    # expanded and transposed gradients
    xq = x.clone().requires_grad_()
    n = rms_norm(xq, pre)
    a, = torch.autograd.grad(n, xq, dn, retain_graph=True)
    b, = torch.autograd.grad(n, xq, dn.t().contiguous().t(), retain_graph=True)
    assert torch.equal(a, b)
    c, = torch.autograd.grad(n.float().sum(), xq)
    assert torch.isfinite(c).all()


def test_empty_zero_and_non_finite_rows(cuda):
    from hard_resets_compose_b200.normgate import norm_gate_residual
    x, h, g, post, pre, dx, dn = make(10, 32, torch.float32, "full", torch.float32)
    e = [t[:0].clone().requires_grad_() for t in (x, h, g)] + [post.clone().requires_grad_(), pre.clone().requires_grad_()]
    xo, n = norm_gate_residual(*e)
    gr = torch.autograd.grad((xo, n), e, (dx[:0], dn[:0]))
    assert n.shape == (0, 32) and not gr[3].any() and not gr[4].any()
    x[2] = h[2] = 0.0          # rsqrt(eps), nothing infinite
    h[5, 3] = float("nan")
    g[7, 0] = -1e30            # sigmoid 0, and 0 * -1e30 stays -0
    xo, n = norm_gate_residual(x, h, g, post, pre)
    ok = torch.ones(10, dtype=torch.bool, device="cuda")
    ok[5] = False
    assert torch.isfinite(xo[ok]).all() and torch.isfinite(n[ok]).all() and not n[2].any()
    assert torch.isnan(n[5]).all()


def test_weight_gradients_repeat(cuda):
    from hard_resets_compose_b200.normgate import norm_gate_residual
    x, h, g, post, pre, dx, dn = make(5000, 256, torch.bfloat16, "row", torch.float32)
    runs = []
    for _ in range(3):
        leaves = [post.clone().requires_grad_(), pre.clone().requires_grad_()]
        runs.append(torch.autograd.grad(norm_gate_residual(x, h, g, *leaves), leaves, (dx, dn)))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_refusals(cuda):
    from hard_resets_compose_b200.normgate import norm_gate_residual, rms_norm
    x, h, g, post, pre, _, _ = make(4, 8, torch.float32, "full", torch.float32)
    for bad in (lambda: norm_gate_residual(x, h[:, :4], g, post, pre), lambda: norm_gate_residual(x, h, g[:3], post, pre),
                lambda: norm_gate_residual(x, h, g, post[:4], pre), lambda: norm_gate_residual(x, h, g, post, pre, act="gelu"),
                lambda: norm_gate_residual(x, None, g, post, pre), lambda: rms_norm(x, None),
                lambda: rms_norm(torch.zeros(1, 8193, device="cuda"), torch.zeros(8193, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: norm_gate_residual(x.double(), h, g, post, pre), lambda: norm_gate_residual(x, h.half(), g, post, pre),
                lambda: norm_gate_residual(x, h, g, post.half(), pre)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        rms_norm(x.cpu(), pre.cpu())


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("R,D,gate", ((9, 12, "full"), (40, 30, "row"), (33, 260, "full"), (21, 1030, "row"),
                                      (300, 2052, "full"), (200, 5140, "row"), (150, 5142, "full"), (3, 8186, "none")))
def test_rows_of_narrower_vectors(cuda, dtype, R, D, gate):
    """Widths that 8 or 4 bytes divide and 16 do not, and addresses that only those fit."""
    test_against_fp64(cuda, dtype, R, D, gate, "silu")


def test_vectors_follow_the_addresses(cuda):
    """The same rows at every offset: the same values, whatever vectors they are read in (sums in another order)."""
    from hard_resets_compose_b200.normgate import norm_gate_residual
    for dtype in (torch.float32, torch.bfloat16):
        R, D = 50, 512
        ts = make(R, D, dtype, "full", torch.float32)[:5]
        rx, rn, _ = reference(ts, 1.0, "silu", 1e-6, *make(R, D, dtype, "full", torch.float32)[5:])
        for at in (0, 1, 2, 4, 6, 8):
            def moved(t):
                wide = torch.full((R, D + 16), float("nan"), device=cuda, dtype=dtype)
                wide[:, at:at + D] = t
                return wide[:, at:at + D]
            with torch.no_grad():
                x, n = norm_gate_residual(moved(ts[0]), moved(ts[1]), moved(ts[2]), ts[3], ts[4])
            assert rel(x, rx) <= tol(x) and rel(n, rn) <= tol(n)
