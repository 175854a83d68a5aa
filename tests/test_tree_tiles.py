"""Which tile of query rows a tree-attention call takes: by the table's size, the query rows and the
format. No GPU."""
import pytest


@pytest.fixture(scope="module")
def va():
    import voltattn_b200
    return voltattn_b200


@pytest.mark.parametrize("fmt,D,few", [("q8+", 128, 64), ("q4+", 128, 64), ("q3+", 64, 64), ("bf16+", 128, 64), ("f8+", 64, 64),
                                       ("f8+", 128, 96), ("f16+", 128, 16), ("f16+", 64, 16)])
def test_query_rows(va, fmt, D, few):
    """Large tables: tiles of 16 up to `few` query rows (fp8 rows of 128 dims take the longest to convert)."""
    for Q, want in ((few // 2, 16), (few // 2 + 1, 128), (64, 128), (33, 16 if few > 66 else 128)):
        assert va.tree_tile_rows(fmt, 16, 16, 8, Q, 1 << 16, D) == want, Q
    assert va.tree_tile_rows(fmt, 16, 24, 8, 43, 1 << 16, D) == 256


@pytest.mark.parametrize("fmt,least", [("f16+", 21), ("q8+", 23), ("f8+", 23)])
def test_table_size(va, fmt, least):
    """128 query rows of one KV head: tiles of 16 up to 2^least positions times query rows."""
    rows = (1 << least) // 128
    assert va.tree_tile_rows(fmt, 1, 4, 1, 32, rows, 128) == 16
    assert va.tree_tile_rows(fmt, 1, 4, 1, 32, rows + 1, 128) == 128


def test_refusals(va):
    for bad in (("q4+", 0, 8, 2, 4, 100, 128), ("q4+", 1, 7, 2, 4, 100, 128), ("q4+", 1, 8, 2, 65, 100, 128), ("q4+", 1, 8, 2, 4, 0, 128),
                ("q4c+", 1, 8, 2, 4, 100, 128), ("q4+", 1, 8, 2, 4, 100, 96), ("f16", 1, 8, 2, 4, 100, 128)):
        with pytest.raises(va.VoltAttnError):
            va.tree_tile_rows(*bad)
