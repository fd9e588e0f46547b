"""Calls of different widths from several host threads at once, through the C entries (which run
without the interpreter's lock)."""
import threading

import pytest
import torch

from hard_resets_compose_b200 import _lib
from hard_resets_compose_b200._lib import LEAKY_ATTN, NORM_GATE

pytestmark = pytest.mark.gpu


def together(calls, rounds):
    """Each call in a thread of its own, `rounds` times; the statuses that were not 0."""
    failed, start = [], threading.Barrier(len(calls))

    def loop(i, call):
        start.wait()
        failed.extend((i, st) for st in (call() for _ in range(rounds)) if st)
    ts = [threading.Thread(target=loop, args=x) for x in enumerate(calls)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    return failed


def test_norm_gradients_of_two_widths(cuda):
    """512 and 4096 fp32 columns: one kernel, 36 and 64 KB of shared memory."""
    L = _lib.load()

    def call(D):
        x, h, dx, dh, w = (torch.randn(2, D, device=cuda) for _ in range(5))
        rstd, s = torch.ones(2, 2, device=cuda), torch.cuda.Stream()
        torch.cuda.synchronize()
        a = NORM_GATE.pack(x.data_ptr(), h.data_ptr(), 0, w.data_ptr(), 0, rstd.data_ptr(), 2, D, D, D, 0, 0, 1.0, 1e-6,
                           2, 0, 0)
        keep = (x, h, dx, dh, w, rstd, s)
        return lambda: (keep, L.lifb_norm_gate_bwd(a, dx.data_ptr(), D, None, D, dh.data_ptr(), None, None, None, None,
                                                   None, 0, s.cuda_stream))[1]
    assert not together([call(512), call(4096), call(512), call(4096)], 5000)


def test_attention_of_two_widths(cuda):
    """Odd widths, on the fp32 pipe: 20 and 80 KB of shared memory."""
    L = _lib.load()

    def call(D):
        x, ld, s = torch.randn(2, 8, 1, D, device=cuda), -torch.ones(1, device=cuda), torch.cuda.Stream()
        o = torch.empty_like(x)
        torch.cuda.synchronize()
        a = LEAKY_ATTN.pack(*(x.data_ptr(),) * 3, ld.data_ptr(), 0, 0, 2, 8, 1, 1, D, D, *(8 * D, D, D) * 3, 1.0, 0)
        keep = (x, ld, s, o)
        return lambda: (keep, L.lifb_leaky_attn_fwd(a, o.data_ptr(), None, None, 0, s.cuda_stream))[1]
    assert not together([call(9), call(127), call(9), call(127)], 5000)
