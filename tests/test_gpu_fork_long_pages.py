"""fork_pages with pages of which more than 2^31 bytes are copied. No reference counterpart."""
import pytest

pytestmark = pytest.mark.gpu


def test_copies_past_31_bits():
    import torch
    import voltattn_b200 as va
    D, page, rest = 128, 2 ** 24, 2 ** 23 + 16  # 256 bytes a row
    one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pools = [torch.zeros(2 * page * 2 * D, dtype=torch.uint8, device="cuda") for _ in "KV"]
    for i, p in enumerate(pools):
        p[:rest * 256].view(torch.int32).copy_(torch.arange(rest * 64, dtype=torch.int32, device="cuda") * (2 * i + 1))
    refs, table = one([1, 0]), one([[0]])
    nr, nt, nl, short = one([9, 9]), one([[9], [9]]), one([9, 9]), one([9])
    ws = torch.zeros(va.pages_workspace_bytes(2, 1, 2), dtype=torch.uint8, device="cuda")
    va.fork_pages("f16+", va.DeviceBufs(pools[0], pools[1], ws=ws), refs, table, one([rest]), one([0, 0]), nr, nt, nl, short, 1, 2, 1, 0, 1,
                  page, 2, D)
    assert nt.tolist() == [[0], [1]] and nl.tolist() == [rest, rest] and nr.tolist() == [1, 1] and short.tolist() == [0]
    for p in pools:
        a, b = p.view(2, -1)
        assert torch.equal(a[:rest * 256], b[:rest * 256]) and not b[rest * 256:].any()
