"""Tree attention with V scales of very different sizes in one cache: the exponent
reference of a query row comes from what it sees alone, each position's score with that
position's own scale. The bound is test_gpu_tree's; where only rows that a node does not
see change, its output keeps its bits. No reference counterpart."""
import numpy as np
import pytest

from tests import cache_ref as R
from tests import test_gpu_tree as T
from tests.test_gpu_tree_tables import Wide

pytestmark = pytest.mark.gpu
SCALED = ["q8+", "q4+", "q3+", "f8+"]
LIM = {"q8+": 127, "q4+": 7, "q3+": 3}
LARGEST = np.float16(60000.0)


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


def case(tile, fmt, D, lens, seed, small):
    """Six nodes of four (tiles of 16), 16 (tiles of 128) or 32 (of 256) query heads a KV head; V of size `small`."""
    G, kind = {16: (4, T.Case), 128: (16, Wide), 256: (32, Wide)}[tile]
    c = kind(fmt, len(lens), 2 * G, 2, 6, D, 32, lens, seed=seed)
    c.sides[1][1] = (c.sides[1][1].astype(np.float32) * small).astype(np.float16)
    return c


def constant_row(fmt, D, dims, negative):
    """Bytes of a row whose first `dims` codes are the lowest (or 0), the others 0."""
    if fmt == "f8+":
        row = np.zeros(D, np.uint8)
        row[:dims] = 0xFE if negative else 0
        return row
    code = np.zeros(D, np.int64)
    code[:dims] = -LIM[fmt] if negative else 0
    if fmt == "q8+":
        return code.astype(np.int8).view(np.uint8)
    k = R.BITS[fmt]
    bits = ((code + LIM[fmt] + 1)[:, None] >> np.arange(k) & 1).astype(np.uint8).reshape(-1)
    return np.packbits(bits, bitorder="little")


@pytest.mark.parametrize("fmt", SCALED)
@pytest.mark.parametrize("tile,D", [(16, 128), (16, 64), (128, 128), (128, 64), (256, 128)])
@pytest.mark.parametrize("small", [0.1, 0.02, 0.004])
def test_large_scale_of_an_unseen_row(va, fmt, tile, D, small):
    """A drafted row with the largest finite scales reaches only the nodes that see it."""
    c = case(tile, fmt, D, [150, 6, 70], 3, small)
    j = 2
    clean = c.run(va, 2)
    for b in range(c.B):
        r = int(c.lens[b]) - 6 + j
        for codes, scales in c.sides:
            scales[c.table[b, r // 32], :, r % 32] = LARGEST
    want, mag = c.expect()
    got = c.run(va, 2)
    for b in range(c.B):
        for i in range(6):
            if not int(c.mask[b, i]) >> j & 1:
                err = np.abs(got[b, i].astype(np.float64) - want[b, i])
                assert (err <= T.bound(want[b, i], mag[b, i])).all()
                assert (got[b, i].view(np.uint16) == clean[b, i].view(np.uint16)).all()


@pytest.mark.parametrize("fmt", SCALED)
@pytest.mark.parametrize("tile,D", [(16, 128), (16, 64), (128, 128), (128, 64), (256, 128)])
@pytest.mark.parametrize("small", [0.1, 0.02, 0.004])
@pytest.mark.parametrize("at", [3, 200, 290])  # in a block of its own, inside, beside the drafted rows
def test_large_scale_of_a_row_without_weight(va, fmt, tile, D, small, at):
    """A row that every node sees, with the largest scales and a score of about -40."""
    c = case(tile, fmt, D, [300], 4, small)
    c.q[..., :16] = 4.0
    where = (c.table[0, at // 32], slice(None), at % 32)
    c.sides[0][0][where] = constant_row(fmt, D, 16, True)
    top = 448.0 if fmt == "f8+" else LIM[fmt]
    c.sides[0][1][where] = np.float16(40.0 * np.sqrt(D) / (16 * 4.0 * top))
    c.sides[1][1][where] = LARGEST
    c.check(va, 2)


@pytest.mark.parametrize("fmt", SCALED)
@pytest.mark.parametrize("tile", [16, 128, 256])
@pytest.mark.parametrize("small", [0.1, 1e-2, 1e-3, 1e-4])
def test_zero_row_among_small_ones(va, fmt, tile, small):
    """A V row of zeros, whose scales are 1 as the quantizer has them."""
    c = case(tile, fmt, 128, [200], 5, small)
    for at in (0, 77, 197):
        where = (c.table[0, at // 32], slice(None), at % 32)
        c.sides[1][0][where] = constant_row(fmt, 128, 0, False)
        c.sides[1][1][where] = np.float16(1.0)
    c.check(va, 2)


@pytest.mark.parametrize("fmt", SCALED)
@pytest.mark.parametrize("tile", [16, 128])
def test_scales_of_zero(va, fmt, tile):
    """Rows with scales of 0 beside others, with the highest scores, and a cache of nothing else."""
    c = case(tile, fmt, 128, [100, 40], 6, 1.0)
    for at in range(0, 100, 3):
        c.sides[1][1][c.table[0, at // 32], :, at % 32] = 0
    c.sides[0][1][c.table[0, 0], :, 0] *= np.float16(8.0)
    for at in range(40):
        c.sides[1][1][c.table[1, at // 32], :, at % 32] = 0
    got = c.check(va, 2)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("fmt", SCALED)
@pytest.mark.parametrize("tile", [16, 128])
def test_other_rows_leave_the_bits(va, fmt, tile):
    """A node's output has the same bits whatever the rows that it does not see hold."""
    c = case(tile, fmt, 128, [90], 7, 1.0)
    j = 1
    clean = c.run(va, 1)
    where = (c.table[0, (90 - 6 + j) // 32], slice(None), (90 - 6 + j) % 32)
    for k, v in ((1e-7, 1e-7), (900.0, 0.0), (np.nan, 3e4), (0.0, np.inf), (-np.inf, np.nan)):
        c.sides[0][1][where], c.sides[1][1][where] = np.float16(k), np.float16(v)
        got = c.run(va, 1)
        for i in range(6):
            if not int(c.mask[0, i]) >> j & 1:
                assert (got[0, i].view(np.uint16) == clean[0, i].view(np.uint16)).all()
