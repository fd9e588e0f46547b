"""Which memory layouts of a cache of states overlap, without a GPU."""
import itertools

import pytest

from hard_resets_compose_b200 import leakyattn


@pytest.mark.parametrize("n,h,mat", ((1, 1, 6), (1, 3, 4), (3, 1, 4), (3, 2, 4), (4, 3, 5)))
def test_overlap_against_every_element(n, h, mat):
    for s0, s1 in itertools.product(range(0, 4 * mat * max(n, h) // 2 + 2, 1), range(0, 3 * mat + 2)):
        cells = [i * s0 + j * s1 + e for i in range(n) for j in range(h) for e in range(mat)]
        assert leakyattn._overlap(n, s0, h, s1, mat) == (len(set(cells)) < len(cells)), (s0, s1)


def test_c_entries_refuse_misaligned_workspaces():
    """Their vector stores need 16 bytes (refused before anything is launched)."""
    from hard_resets_compose_b200 import _lib
    L = _lib.load()
    a = _lib.LEAKY_ATTN.pack(256, 256, 256, 256, 0, 0, 2, 300, 4, 2, 64, 64, *(1,) * 9, 1.0, 1)
    st = (_lib.c_i64 * 3)(1, 1, 1)
    big = 1 << 40
    assert L.lifb_leaky_attn_workspace_bytes(a, 0) and L.lifb_leaky_attn_workspace_bytes(a, 1)
    assert L.lifb_leaky_attn_fwd(a, 256, None, 264, big, None) == 3 and b"misaligned" in L.lifb_last_error()
    assert L.lifb_leaky_attn_bwd(a, 256, st, None, 256, 256, 256, None, 264, big, None) == 3
    n = _lib.NORM_GATE.pack(256, 256, 256, 256, 256, 256, 4, 8, 8, 8, 8, 8, 1.0, 1e-6, 0, 0, 0)
    assert L.lifb_norm_gate_bwd(n, 256, 8, 256, 8, 256, 256, 256, 256, 256, 260, big, None) == 3
