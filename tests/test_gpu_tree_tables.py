"""Tree attention through block tables that are much longer than the sequences: the
tables' size chooses the kernel's tiles, so these cases run the large ones."""
import numpy as np
import pytest

from tests import test_gpu_tree as T

pytestmark = pytest.mark.gpu
R = T.R


@pytest.fixture(scope="module")
def va():
    import torch
    assert torch.cuda.is_available()
    import voltattn_b200
    return voltattn_b200


class Wide(T.Case):
    """Tables of 2^23 / (query rows of all sequences) rows and more; places past a sequence are -1."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        rows = (1 << 23) // (self.B * self.Q * self.Hq) + self.page
        self.max_pages = max(self.max_pages, -(-rows // self.page))
        self.table = np.pad(self.table, ((0, 0), (0, self.max_pages - self.table.shape[1])), constant_values=-1)


@pytest.fixture(autouse=True)
def wide(monkeypatch):
    monkeypatch.setattr(T, "Case", Wide)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("shape", [s for s in T.SHAPES if s[1] // s[2] * s[3] > 16], ids=lambda s: "B{}_Hq{}_Hkv{}_Q{}_D{}_P{}".format(*s[:6]))
def test_shapes(va, fmt, shape):
    T.test_tree(va, fmt, shape)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("rows,D", [(17, 128), (33, 64), (64, 128), (65, 128), (66, 64), (96, 128), (128, 64), (128, 128), (129, 128), (130, 64),
                                    (256, 128), (257, 128), (320, 64)])
def test_tile_edges(va, fmt, rows, D):
    T.test_row_tile_edges(va, fmt, rows, D)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("rows", [40, 160])
def test_nothing_seen(va, fmt, rows):
    T.test_rows_that_see_nothing(va, fmt, rows)


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("G", [4, 8, 16])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_unseen(va, fmt, G, what):
    T.test_unseen_rows_have_no_influence(va, fmt, G, what)


@pytest.mark.parametrize("fmt", ["f16+", "bf16+", "f8+"])
@pytest.mark.parametrize("Hq", [32, 96])
def test_nan_entry(va, fmt, Hq):
    T.test_entry_of_nan_in_large_tiles(va, fmt, Hq)


@pytest.mark.parametrize("fmt", ["q8+", "f16+", "q3+", "bf16+"])
@pytest.mark.parametrize("G,Q", [(8, 4), (4, 32), (8, 32)])
def test_rising_scores(va, fmt, G, Q):
    T.test_growing_scores(va, fmt, G, Q)


@pytest.mark.parametrize("fmt", ["q4+", "f16+"])
@pytest.mark.parametrize("S", [0, 1, 2, 3, 40])
def test_uneven_lengths(va, fmt, S):
    """One long sequence among short, unused and barely drafted ones: windows that hold many
    tiles, and tiles that span many windows."""
    lens = [5000, 0, 64, 1, 700, 63, 65, 4, 130]
    nodes = [20, 0, 20, 1, 20, 2, 20, 0, 7]
    c = Wide(fmt, 9, 10, 2, 20, 128, 32, lens, nodes, seed=S)
    ws = None
    if S == 0:
        import torch
        ws = torch.zeros(va.tree_workspace_bytes(9, 10, 2, 20, 128, 24), dtype=torch.uint8, device="cuda")
    first = c.check(va, S, ws)
    assert (c.run(va, S, ws) == first).all()


@pytest.mark.parametrize("B", [32, 33, 75])
def test_more_sequences_than_lanes(va, B):
    rng = np.random.default_rng(B)
    lens = rng.integers(0, 400, B)
    nodes = np.minimum(rng.integers(0, 17, B), lens)
    c = Wide("q8+", B, 8, 1, 16, 64, 16, lens, nodes, seed=B)
    for S in (1, 2, 7):
        c.check(va, S)


def test_window_across_many_sequences(va):
    """More sequences than a window of a few CTAs' lanes: every window spans groups of 32 sequences."""
    B = 700
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 40, B)
    c = Wide("q4+", B, 8, 1, 16, 64, 8, lens, np.minimum(16, lens), seed=1)
    c.check(va, 2)
