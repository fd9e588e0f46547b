"""The sequence model's own bookkeeping (the decay's type, places of the cache, lengths)
on the CPU, its operators replaced by plain forms."""
import pytest
import torch

from hard_resets_compose_b200 import seqnet


@pytest.mark.parametrize("kind", ("bfloat16", "to", "half", "double"))
def test_the_decay_keeps_its_bits(kind):
    n = seqnet.SeqNet(vocab=5, width=32, heads=4, layers=2)
    before = [b.log_decay.clone() for b in n.blocks]
    n = n.to(torch.bfloat16) if kind == "to" else getattr(n, kind)()
    assert n.blocks[0].out.weight.dtype != torch.float32
    for b, d in zip(n.blocks, before):
        assert b.log_decay.dtype == torch.float32 and torch.equal(b.log_decay, d)
        assert dict(b.named_buffers())["log_decay"] is b.log_decay
