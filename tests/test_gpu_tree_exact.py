"""A node that sees one row gives that row's values, each rounded once: the row sets the exponents'
reference, so its weight is a power of two and its scales, as fp16 weights, need no rounding, in either
64-dim group. No reference counterpart."""
import numpy as np
import pytest

from tests import cache_ref as R
from tests.test_gpu_tree import Case
from tests.test_gpu_tree_tables import Wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("tile,D", [(16, 128), (16, 64), (128, 128), (128, 64), (256, 128)])
def test_one_row(va, fmt, tile, D):
    """Half of fp16's spacing, and the 1e-6 that fp32 scores and sums move a value by, against the steps that are left
    to a tie: less than a hundredth more."""
    G, Q = {16: 3, 128: 25, 256: 50}[tile], 5
    mask = np.array([[1 << i for i in range(Q)]] * 2, np.uint64)
    c = (Case if tile == 16 else Wide)(fmt, 2, 2 * G, 2, Q, D, 32, [Q, Q], mask=mask, seed=tile)
    assert va.tree_tile_rows(fmt, 2, 2 * G, 2, Q, c.max_pages * 32, D) == tile
    got = c.run(va, 1).astype(np.float64)
    for b in range(2):
        for h in range(2):
            v = c.rows(1, b, h)
            for i in range(Q):
                want = v[i]
                half = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64) / 2
                assert (np.abs(got[b, i, h * G:h * G + G] - want) <= 1.01 * half).all()
