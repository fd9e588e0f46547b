"""Which memory layouts of a cache of states overlap, without a GPU."""
import itertools

import pytest

from hard_resets_compose_b200 import leakyattn


@pytest.mark.parametrize("n,h,mat", ((1, 1, 6), (1, 3, 4), (3, 1, 4), (3, 2, 4), (4, 3, 5)))
def test_overlap_against_every_element(n, h, mat):
    for s0, s1 in itertools.product(range(0, 4 * mat * max(n, h) // 2 + 2, 1), range(0, 3 * mat + 2)):
        cells = [i * s0 + j * s1 + e for i in range(n) for j in range(h) for e in range(mat)]
        assert leakyattn._overlap(n, s0, h, s1, mat) == (len(set(cells)) < len(cells)), (s0, s1)
