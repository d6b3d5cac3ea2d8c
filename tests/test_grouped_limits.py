"""The most groups that gsplat_core.grouped takes, and the scratch that its
backward asks for: refusals and sizes on the host, and calls at those
limits on the device."""
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


# dtype, K, M, row ids; whether a v_x of its own needs scratch
WANTED = [(0, 64, 64, 0, False), (0, 32, 3, 1, False), (1, 64, 64, 0, False), (1, 64, 64, 1, True),
          (2, 77, 45, 0, False), (2, 77, 45, 1, True), (1, 200, 136, 1, True)]


@pytest.mark.parametrize("dtype,K,M,ids,own", WANTED)
def test_scratch_is_for_what_is_wanted(gs, dtype, K, M, ids, own):
    """No partial sums of weights for v_x alone, no sums of shared rows for the
    weights alone; a gradient that is not named is refused."""
    from gsplat_core import _lib as L
    lib = gs.load()
    size = {}
    for wanted in range(8):
        q = L.GroupedParams(1000, 900 if ids else 1000, 70_000, K, M, dtype, 0, ids, 0, wanted)
        size[wanted] = lib.gs_grouped_linear_bwd_workspace_size(ct.byref(q))
    sums = 900 * K * 4 if own else 0
    assert sums <= size[1] <= sums + 256
    assert size[0] == size[3] == size[5] == size[7] and size[2] == size[4] == size[6]
    assert size[2] >= 4 * 70_000 * K * M
    assert size[7] - size[2] == size[1]
    one = ct.c_void_p(256)  # never followed: refused first
    for wanted, given in ((1, (None, one, None)), (6, (one, None, None)), (3, (one, one, one))):
        q = L.GroupedParams(1000, 900 if ids else 1000, 2, K, M, dtype, 0, ids, 0, wanted)
        assert lib.gs_grouped_linear_bwd(ct.byref(q), *[one] * 6, *given, one, 1 << 40,
                                         None) == L.GS_ERR_INVALID
    q = L.GroupedParams(1000, 1000, 2, K, M, dtype, 0, 0, 0, 8)
    assert lib.gs_grouped_linear_bwd_workspace_size(ct.byref(q)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,K,M,ids,own", WANTED)
def test_scratch_suffices(gs, cuda, dtype, K, M, ids, own):
    """With the scratch of each set of gradients, and not a byte past it, they
    have the bits of the whole (with row ids that name a row once, so that
    v_x has a fixed order)."""
    from gsplat_core import _lib as L
    lib = gs.load()
    dt = [torch.float32, torch.bfloat16, torch.float16][dtype]
    g = torch.Generator(device="cuda").manual_seed(dtype)
    R = 5000
    x, y, v = (torch.randn(R, k, generator=g, device="cuda").to(dt) for k in (K, M, M))
    w = torch.randn(3, M, K, generator=g, device="cuda").to(dt)
    off = torch.tensor([0, 1700, 1701, R], dtype=torch.int32, device="cuda")
    perm = torch.randperm(R, generator=g, device="cuda").to(torch.int32) if ids else None
    P = lambda t: None if t is None else ct.c_void_p(t.data_ptr())  # noqa: E731

    def run(wanted):
        q = L.GroupedParams(R, R, 3, K, M, dtype, 1, ids, 0, wanted)
        need = lib.gs_grouped_linear_bwd_workspace_size(ct.byref(q))
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        out = [torch.empty_like(t) if wanted & bit else None
               for t, bit in ((x, 1), (w, 2), (w[:, :, 0].contiguous(), 4))]
        torch.cuda.synchronize()
        assert lib.gs_grouped_linear_bwd(ct.byref(q), P(x), P(perm), P(off), P(w), P(y), P(v),
                                         *map(P, out), P(ws) if need else None, need, None) == 0
        torch.cuda.synchronize()
        assert bool((ws[need:] == 0x5A).all())
        return out

    whole = run(7)
    for wanted in range(1, 7):
        for got, want, name in zip(run(wanted), whole, ("v_x", "v_weights", "v_biases")):
            # v_x alone comes from another kernel than the 16-bit whole
            if got is not None and (name != "v_x" or wanted != 1):
                assert torch.equal(got, want), (wanted, name)
            elif got is not None:
                assert torch.allclose(got.float(), want.float(), rtol=2 ** -6, atol=1e-4)


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
