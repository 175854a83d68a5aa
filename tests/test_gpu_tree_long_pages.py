"""Tree attention over pages whose rows lie more than 2^31 bytes behind the page's start, and
the longest tables that the entry point takes. No reference counterpart."""
import ctypes as C

import numpy as np
import pytest

from tests import test_cache_ops_refusals as A


def test_longest_tables():
    """Positions stay below 2^31 with what the kernels add to them; longer tables are refused before any CUDA call."""
    import voltattn_b200 as va
    for page, pages in ((32, 2 ** 26 - 1), (8, 2 ** 28 - 1), (2 ** 31 - 8, 1)):
        assert A.tree(va, page=page, max_pages=pages, B=1) == A.TOO_LARGE


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,D", [("f16+", 128), ("bf16+", 128), ("q8+", 128), ("f16+", 64)])
@pytest.mark.parametrize("Q", [2, 32])
def test_rows_far_into_a_page(fmt, D, Q):
    """One page that is the whole cache. All rows but the last ones are zero (their weights count, their
    values do not), the last ones have scores of about 20."""
    import torch
    import voltattn_b200 as va
    wide = fmt != "q8+"
    rb = D * (2 if wide else 1)
    page = 2 ** 31 // rb + 1024
    near, n = 96, page - 40  # rows with values, rows in the cache
    gen = torch.Generator(device="cuda").manual_seed(D + Q)
    u = torch.randn(D, generator=gen, device="cuda")
    q = (u + 0.1 * torch.randn(1, Q, 1, D, generator=gen, device="cuda")).half()
    k = 20 * D ** 0.5 / float(u @ u) * u + 0.01 * torch.randn(near, D, generator=gen, device="cuda")
    v = torch.randn(near, D, generator=gen, device="cuda")

    def store(x):
        """The whole cache, its scales, and the last rows' values in 64 bits."""
        buf = torch.zeros(page * rb, dtype=torch.uint8, device="cuda")
        at = buf[(n - near) * rb:n * rb].view(near, rb)
        if wide:
            y = x.to(torch.float16 if fmt == "f16+" else torch.bfloat16)
            at.copy_(y.view(torch.uint8))
            return buf, None, y.double()
        s = (x.abs().view(near, D // 64, 64).amax(-1) / 127).half()
        c = (x.view(near, D // 64, 64) / s.float()[..., None]).round().clamp(-127, 127)
        at.copy_(c.to(torch.int8).view(near, D).view(torch.uint8))
        scales = torch.ones(page, D // 64, dtype=torch.float16, device="cuda")
        scales[n - near:n] = s
        return buf, scales, (c.double() * s.double()[..., None]).view(near, D)

    K, sK, kd = store(k)
    V, sV, vd = store(v)
    one = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    mask = one([[(2 << i) - 1 for i in range(Q)]], torch.int64)
    S = 64
    ws = torch.zeros(va.tree_workspace_bytes(1, 1, 1, Q, D, S), dtype=torch.uint8, device="cuda")
    out = torch.full((1, Q, 1, D), float("nan"), dtype=torch.float16, device="cuda")
    va.decode_tree(fmt, va.DeviceBufs(K, V, sK, sV, q, out, ws), mask, one([n]), one([Q]), one([[0]]), 1, 1, 1, 1, Q, page, 1, D, S=S)
    s = q[0, :, 0].double() @ kd.T / D ** 0.5
    i, j = torch.arange(Q, device="cuda")[:, None], torch.arange(near, device="cuda")[None, :]
    w = s.exp() * (j - (near - Q) <= i)
    total = w.sum(1) + (n - near)
    want, mag = (w @ vd) / total[:, None], (w @ vd.abs()) / total[:, None]
    err = (out[0, :, 0].double() - want).abs().cpu().numpy()
    from tests.test_gpu_tree import bound
    assert (err <= bound(want.cpu().numpy(), mag.cpu().numpy())).all()
    assert va.device_error() == 0
