"""What the sequence-model operators owe autograd and their callers, on both host paths (the C++
binding and the Python functions)."""
import pytest
import torch

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
