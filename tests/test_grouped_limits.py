"""The most groups that gsplat_core.grouped takes: refusals on the host, and
calls next to 2^31 groups on the device."""
from __future__ import annotations

import ctypes as ct

import pytest
import torch

MOST = 2 ** 31 - 2


def test_more_groups_are_refused(gs):
    """What would not fit the C entry's 32 bits is refused, not cut off."""
    from gsplat_core import _lib as L
    from gsplat_core.grouped import group_offsets, grouped_linear_forward
    ids = torch.zeros(3, dtype=torch.int32)
    for groups in (MOST + 1, 2 ** 32 + 5):
        with pytest.raises(RuntimeError, match="2\\^31 - 1 groups"):
            group_offsets(ids, groups)
        w = torch.zeros(1).expand(groups, 1, 1)
        off = torch.zeros(1, dtype=torch.int32).expand(groups + 1)
        with pytest.raises(RuntimeError, match="2\\^31 - 1 groups"):
            grouped_linear_forward({"x": torch.zeros(3, 1), "weights": w, "offsets": off})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        group_offsets(ids, MOST)
    lib = gs.load()
    q = L.GroupedParams(6, 6, 2 ** 31 - 1, 4, 5, 0, 0, 0)
    assert lib.gs_grouped_linear_fwd(ct.byref(q), *[None] * 7) == L.GS_ERR_INVALID
    assert lib.gs_grouped_linear_bwd_workspace_size(ct.byref(q)) == 0


@pytest.mark.gpu
def test_offsets_of_the_most_groups(gs, cuda):
    """Every bound is written, and nothing in front of them: the ids lie at
    both ends, where a 32-bit count of the groups would turn negative."""
    from gsplat_core.grouped import group_offsets
    at = [0, 7, MOST - 2, MOST - 1]
    ids = torch.tensor(at, dtype=torch.int32, device="cuda")
    off = group_offsets(ids, MOST)
    assert off.numel() == MOST + 1
    edges = [0] + [a + 1 for a in at] + [MOST + 1]
    for i, (a, b) in enumerate(zip(edges, edges[1:])):
        assert bool((off[a:b] == i).all()), i


@pytest.mark.gpu
def test_products_of_the_most_groups(gs, cuda):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    at = [0, 7, 2 ** 30, MOST - 1]
    off = torch.zeros(MOST + 1, dtype=torch.int32, device="cuda")
    for a in at:
        off[a + 1:] += 1
    w = torch.ones((MOST, 1, 1), dtype=torch.bfloat16, device="cuda")
    for i, a in enumerate(at):
        w[a] = i + 2.0
    c = {"x": torch.tensor([[1.0], [2.0], [3.0], [4.0]], device="cuda").bfloat16(), "weights": w,
         "offsets": off}
    y = grouped_linear_forward(c)
    assert y.flatten().tolist() == [2.0, 6.0, 12.0, 20.0]
    g = grouped_linear_backward(c, None, torch.full_like(y, 2.0))
    assert g["v_x"].flatten().tolist() == [4.0, 6.0, 8.0, 10.0]
    vw = g["v_weights"].flatten()
    assert [vw[a].item() for a in at] == [2.0, 4.0, 6.0, 8.0]
    assert int(sum(torch.count_nonzero(part) for part in vw.split(2 ** 28))) == 4
