"""gsplat_core.dropout on the device against its definition: masks equal bit
for bit, kept values within the roundings of x / (1 - p)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _learned import TYPES, half_step, keep_mask, tiny

pytestmark = pytest.mark.gpu
SEED = 0x9E3779B97F4A7C15


def _x(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) + 3.0   # no zeros: the mask can be read off
    return x.to(dtype).cuda()


def _check(y, x, p, seed, step, rows):
    """The mask exactly; a kept value within the rounding of 1 / (1 - p) to
    fp32, that of the product (2^-24 each) and that to the type."""
    keep = torch.from_numpy(keep_mask(tuple(x.shape), p, seed, step, rows).copy())
    y64, x64 = y.double().cpu(), x.double().cpu()
    assert bool((y64[~keep] == 0).all())
    if p < 1:
        want = x64 / (1 - p)
        allow = (half_step(x.dtype) + 2 * 2.0 ** -24) * (1 + 2.0 ** -8) * want.abs() + tiny(x.dtype)
        bad = keep & ~((y64 - want).abs() <= allow)
        assert not bad.any(), (bad.nonzero()[:3], y64[bad][:3], want[bad][:3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,rows", [
    ((1,), True), ((0,), True), ((3,), False), ((1027,), True), ((10_001,), False), ((515, 1), True),
    ((129, 3), True), ((1000, 48), True), ((77, 37), True), ((300, 257), True), ((2, 70_001), True),
    ((300, 64), True), ((131, 16, 3), True), ((999, 37), False), ((4, 8192), False), ((5, 0), True)])
def test_dropout_matches_definition(gs, cuda, dtype, shape, rows):
    from gsplat_core.dropout import dropout_backward, dropout_forward
    x = _x(shape, TYPES[dtype])
    for p, seed, step in ((0.3, SEED, 5), (0.75, 12, 1 << 33)):
        y = dropout_forward(x, p, seed, step=step, rows=rows)
        _check(y, x, p, seed, step, rows)
        assert torch.equal(dropout_backward(x, p, seed, step=step, rows=rows), y)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 0.5, 1.0 - 2.0 ** -20, 1.0])
def test_edges_of_p(gs, cuda, p):
    from gsplat_core.dropout import dropout_forward
    x = _x((5000,), torch.float32)
    y = dropout_forward(x, p, 3, rows=True)
    if p in (0.0, 2.0 ** -33):
        assert torch.equal(y, x)
    elif p == 1.0:
        assert not y.any()
    else:
        _check(y, x, p, 3, 0, True)


@pytest.mark.parametrize("rows", [True, False])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_unaligned_and_strided(gs, cuda, rows, offset):
    """Views that start off a 16-byte boundary, in and out, and a strided x;
    what lies around out is left as it was."""
    from gsplat_core.dropout import dropout_forward
    for dtype in TYPES.values():
        base = _x((4000 + offset,), dtype)
        x = base[offset:].view(500, 8)
        y = dropout_forward(x, 0.4, 9, rows=rows)
        _check(y, x, 0.4, 9, 0, rows)
        buf = torch.full((4000 + offset + 5,), 7.0, dtype=dtype, device="cuda")
        out = buf[offset:offset + 4000].view(500, 8)
        dropout_forward(x, 0.4, 9, rows=rows, out=out)
        assert torch.equal(out, y)
        assert bool((buf[:offset] == 7).all()) and bool((buf[offset + 4000:] == 7).all())
        t = x.t()
        assert torch.equal(dropout_forward(t, 0.4, 9, rows=rows),
                           dropout_forward(t.contiguous(), 0.4, 9, rows=rows))


def test_non_finite_values(gs, cuda):
    """Dropped NaN and infinities are zeros; kept ones stay."""
    from gsplat_core.dropout import dropout_forward
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = torch.full((999, 5), bad, device="cuda")
        for rows in (True, False):
            y = dropout_forward(x, 0.5, 4, rows=rows).cpu()
            keep = torch.from_numpy(keep_mask((999, 5), 0.5, 4, 0, rows).copy())
            assert bool((y[~keep] == 0).all())
            assert bool(torch.isnan(y[keep]).all() if bad != bad else (y[keep] == bad).all())


def test_in_place_and_far_places(gs, cuda):
    """In place; and values whose place passes 2^32 bytes and 2^31 values."""
    from gsplat_core.dropout import dropout_forward
    x = _x((4097,), torch.float32)
    y = dropout_forward(x, 0.4, 9)
    assert dropout_forward(x, 0.4, 9, out=x) is x and torch.equal(x, y)
    buf = torch.zeros((4100,), device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        dropout_forward(buf[:4097], 0.4, 9, out=buf[3:])
    n = (1 << 31) + 4096 + 7
    big = torch.ones((n,), dtype=torch.bfloat16, device="cuda")
    dropout_forward(big, 0.5, 21, step=2, out=big)
    from _learned import philox
    for lo in (0, (1 << 31) - 512, n - 1024):
        lo -= lo % 4
        m = min(1024, n - lo)
        # words of the blocks from lo / 4 on: the counters are shifted by hand
        want = _words_at(lo, m, 21, 2) >= np.uint64(1 << 31)
        assert np.array_equal(big[lo:lo + m].float().cpu().numpy() > 0, want), lo
    assert philox(8, 21, 2).tolist() == _words_at(0, 8, 21, 2).tolist()
    share = float((big == 0).float().mean(dtype=torch.float64))
    assert abs(share - 0.5) < 5 * 0.5 / n ** 0.5


def _words_at(start, n, seed, step):
    import _learned
    real = np.arange
    try:  # the oracle's counters from start / 4 on
        _learned.np.arange = lambda k, dtype: real(start // 4, start // 4 + k, dtype=dtype)
        return _learned.philox(n, seed, step)
    finally:
        _learned.np.arange = real


def test_large_rows(gs, cuda):
    from gsplat_core.dropout import dropout_forward
    x = torch.ones((3_000_000, 48), device="cuda")
    y = dropout_forward(x, 0.2, 5, step=3, rows=True)
    keep = torch.from_numpy(keep_mask((3_000_000,), 0.2, 5, 3, True).copy()).cuda()
    assert torch.equal(y, torch.where(keep[:, None], torch.full_like(y, 1.25), torch.zeros_like(y)))


def test_step_tensor_graph_and_streams(gs, cuda):
    """A captured call draws the mask of the step that the tensor holds at
    replay; a call on another stream."""
    from gsplat_core.dropout import dropout_forward
    x = _x((10_000, 3), torch.float32)
    step = torch.tensor([4], dtype=torch.int64, device="cuda")
    dropout_forward(x, 0.3, 8, step=step, rows=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = dropout_forward(x, 0.3, 8, step=step, rows=True)
        step += 1
    for it in range(3):
        g.replay()
        assert torch.equal(y, dropout_forward(x, 0.3, 8, step=4 + it, rows=True)), it
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = dropout_forward(x, 0.3, 8, step=6, rows=True)
    side.synchronize()
    assert torch.equal(z, y)
    neg = torch.tensor(-1, dtype=torch.int64, device="cuda")
    assert torch.equal(dropout_forward(x, 0.3, -1, step=neg),
                       dropout_forward(x, 0.3, (1 << 64) - 1, step=(1 << 64) - 1))


def test_autograd(gs, cuda):
    from gsplat_core import autograd as A
    x = _x((700, 6), torch.float32).requires_grad_(True)
    v = torch.randn(700, 6, device="cuda")
    y = A.dropout(x, 0.25, 11, 2, rows=True)
    y.backward(v)
    keep = torch.from_numpy(keep_mask((700, 6), 0.25, 11, 2, True).copy()).cuda()
    scale = torch.tensor(1 / 0.75, device="cuda")
    assert torch.equal(x.grad, torch.where(keep, v * scale, torch.zeros_like(v)))
    # against a difference: y is linear in x, so the quotient is exact up to
    # rounding (values below 16, a step of 1: 2^-24 16 per value and side)
    with torch.no_grad():
        d = torch.ones_like(x)
        quot = ((A.dropout(x + d, 0.25, 11, 2, True) - A.dropout(x, 0.25, 11, 2, True)) * v)
        assert ((quot - x.grad).abs() <= 4 * 16 * 2.0 ** -23 * v.abs()).all()
    # a step tensor changed before the backward is refused, not redrawn
    step = torch.tensor([1], dtype=torch.int64, device="cuda")
    y = A.dropout(x, 0.25, 11, step)
    step += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
