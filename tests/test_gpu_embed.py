"""Embedding and its gradient (csrc/embed.cu) against 64-bit sums.

Bounds, elementwise: the forward multiplies once in fp32 and rounds once; the
gradient adds the m rows of a token and multiplies by the scale in fp32 (at
most m + 2 roundings of sums no larger than the terms' absolute sum A), then
rounds once: |error| <= (m + 2) 2^-24 A + u |y|."""
import pytest
import torch

from tests.seq_refs import U

pytestmark = pytest.mark.gpu
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def make(n, V, D, dtype, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n + 7 * V + 13 * D)
    if kind == "one":
        tok = torch.full((n,), V // 2, device="cuda")
    elif kind == "skew":
        tok = (V * torch.rand(n, device="cuda", generator=g) ** 4).long().clamp(max=V - 1)
    else:
        tok = torch.randint(0, V, (n,), device="cuda", generator=g)
    if n > 4 and kind != "one":
        tok[torch.randint(0, n, (n // 4,), device="cuda", generator=g)] = -1
    W = torch.randn(V, D, device="cuda", generator=g).to(dtype)
    dy = torch.randn(n, D, device="cuda", generator=g).to(dtype)
    return tok, W, dy


def check_grad(dw, tok, dy, scale, V):
    live = tok >= 0
    t, d = tok[live], dy.double()[live]
    ref = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    mag, cnt = torch.zeros_like(ref), torch.zeros(V, dtype=torch.float64, device=dy.device)
    ref.index_add_(0, t, d)
    mag.index_add_(0, t, d.abs())
    cnt.index_add_(0, t, torch.ones_like(t, dtype=torch.float64))
    ref, mag = ref * scale, mag * abs(scale)
    tiny = 2.0 ** -24 if dy.dtype == torch.float16 else 0.0  # fp16's subnormal step
    bound = (cnt[:, None] + 2) * 2.0 ** -24 * mag + (U[dy.dtype] * ref.abs() if dy.dtype != torch.float32 else 0) + tiny
    assert ((dw.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D,kind", ((1, 1, 1, "even"), (2, 700, 256, "even"), (64, 3, 8, "even"),
                                        (65, 3, 24, "skew"), (1000, 700, 256, "even"), (1023, 1024, 33, "skew"),
                                        (4097, 1025, 40, "skew"), (3000, 50001, 64, "skew"), (777, 9, 100, "one"),
                                        (70001, 700, 16, "even"), (66000, 200003, 8, "skew"), (128, 5, 264, "one"),
                                        (129, 2, 1000, "even")))
def test_embedding(cuda, dtype, n, V, D, kind):
    from hard_resets_compose_b200.embed import embedding
    tok, W, dy = make(n, V, D, dtype, kind)
    scale = 1.7
    for t in (tok, tok.int()):
        Wq = W.clone().requires_grad_()
        y = embedding(t, Wq, scale)
        ref = torch.where((tok >= 0)[:, None], W.double()[tok.clamp(min=0)] * scale, 0.0)
        assert ((y.double() - ref).abs() <= (2.0 ** -23 + U[dtype]) * ref.abs() + (2.0 ** -24 if dtype == torch.float16 else 0)).all()
        dw, = torch.autograd.grad(y, Wq, dy)
        assert dw.dtype == dtype and dw.shape == W.shape
        check_grad(dw, tok, dy, scale, V)
        again, = torch.autograd.grad(embedding(t, Wq, scale), Wq, dy)
        assert torch.equal(dw, again)  # the order of the sums is fixed


def test_embedding_difference(cuda):
    """y is linear in the weight: (y(W + d) - y(W - d)) / 2 . dy = dW . d."""
    from hard_resets_compose_b200.embed import embedding
    tok, W, dy = make(500, 37, 12, torch.float32, "skew")
    d = torch.randn_like(W)
    W.requires_grad_()
    dw, = torch.autograd.grad(embedding(tok, W, 0.5), W, dy)
    with torch.no_grad():
        diff = ((embedding(tok, W + d, 0.5) - embedding(tok, W - d, 0.5)).double() / 2 * dy.double()).sum()
        mag = ((embedding(tok, W.abs() + d.abs(), 0.5)).double() * dy.double().abs()).sum()
    assert abs(diff - (dw.double() * d.double()).sum()) <= 600 * 2.0 ** -24 * mag


def test_shapes_strides_streams(cuda):
    from hard_resets_compose_b200.embed import embedding
    tok, W, dy = make(60, 11, 16, torch.bfloat16, "even")
    wide = torch.zeros(11, 48, dtype=torch.bfloat16, device="cuda")
    wide[:, 16:32] = W
    ref = embedding(tok, W)
    assert torch.equal(embedding(tok, wide[:, 16:32]), ref)          # a row stride
    assert torch.equal(embedding(tok, W.t().contiguous().t()), ref)  # another order
    assert torch.equal(embedding(tok.view(3, 4, 5), W), ref.view(3, 4, 5, 16))
    off = torch.zeros(11 * 16 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(11, 16)
    off.copy_(W)
    assert torch.equal(embedding(tok, off), ref)                     # rows that are not 16-byte aligned
    assert embedding(tok[:0], W).shape == (0, 16)
    Wq = W.clone().requires_grad_()
    assert torch.autograd.grad(embedding(tok[:0], Wq).sum(), Wq)[0].abs().sum() == 0
    dy_t = dy.t().contiguous().t()
    a, = torch.autograd.grad(embedding(tok, Wq), Wq, dy)
    b, = torch.autograd.grad(embedding(tok, Wq), Wq, dy_t)
    assert torch.equal(a, b)
    c, = torch.autograd.grad(embedding(tok, Wq).sum(), Wq)           # an expanded gradient
    assert torch.equal(c[:, 0].float(), torch.bincount(tok[tok >= 0], minlength=11).float().to(c.dtype).float())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = embedding(tok, W)
    side.synchronize()
    assert torch.equal(got, ref)


def test_non_finite_stay_in_their_rows(cuda):
    from hard_resets_compose_b200.embed import embedding
    tok, W, dy = make(300, 20, 8, torch.float32, "even")
    tok[:2] = torch.tensor([3, -1], device="cuda")
    dy[0] = float("inf")
    dy[tok < 0] = float("nan")  # padding's gradient is not read
    Wq = W.clone().requires_grad_()
    dw, = torch.autograd.grad(embedding(tok, Wq), Wq, dy)
    ok = torch.ones(20, dtype=torch.bool, device="cuda")
    ok[3] = False
    assert torch.isfinite(dw[ok]).all() and torch.isinf(dw[3]).all()


def test_token_past_the_table_is_reported(cuda):
    from hard_resets_compose_b200 import _lib
    from hard_resets_compose_b200.embed import embedding
    lib = _lib.load()
    assert lib.lifb_check_device(1) == 0
    tok = torch.tensor([0, 5, 1], device="cuda")
    W = torch.ones(5, 4, device="cuda")
    y = embedding(tok, W)
    with pytest.raises(_lib.LifbError) as e:
        _lib.check_device("embedding", reset=True)
    assert e.value.device_code == 102
    assert y[1].abs().sum() == 0 and (y[[0, 2]] == 1).all()
    assert lib.lifb_check_device(0) == 0


def test_refusals(cuda):
    from hard_resets_compose_b200.embed import embedding
    W, tok = torch.zeros(5, 4, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError):
        embedding(tok, W[0])
    with pytest.raises(TypeError):
        embedding(tok, W.double())
    with pytest.raises(TypeError):
        embedding(tok.float(), W)
    with pytest.raises(RuntimeError):
        embedding(tok.cpu(), W)
