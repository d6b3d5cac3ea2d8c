"""Long and deep sums of gsplat_core.grouped, all of one sign, so that what an
accumulator loses at each addition does not cancel, and gradients next to
the smallest that 16 bits hold.  The sums that they are compared with are
64-bit products on the device."""
from __future__ import annotations

import math

import pytest
import torch

from _learned import TYPES, tiny

pytestmark = pytest.mark.gpu

BITS = {torch.float32: 24, torch.bfloat16: 8, torch.float16: 11}


CUTS = {torch.float32: 2, torch.bfloat16: 4, torch.float16: 4}


def _bound(steps, joined, dtype):
    """How far a sum of one sign may be off, of its value.

    The tensor core cuts sums to fp32.  A step of 16 products loses as much as
    four cuts do at most, one of 8 fp32 products as much as two (on the device
    growing sums lost 3.0 and 1.2 times 2^-25 a step).  A cut loses between 0 and 2^-23 of
    the partial sum, half of that on average, and the partial sums are half of
    the last on average: 2^-25.  The spread of the cuts, and that of ``joined``
    rounded additions of partial sums (2^-24 at most, either way), both with
    the partial sums' squares at a third of the last's, as six standard
    deviations.  fp32 factors are taken apart to 2^-22 each, and the product of
    two remainders: 3 2^-22."""
    cuts = steps * CUTS[dtype]
    spread = math.sqrt(cuts / 3) * 2.0 ** -23 / math.sqrt(12), math.sqrt(joined / 9) * 2.0 ** -24
    return cuts * 2.0 ** -25 + 6 * math.hypot(*spread) + (3 * 2.0 ** -22 if dtype == torch.float32 else 0)


def _assert_sums(got, want, bound, extra=0.0, what=""):
    """|got - want| within bound |want| + extra and half a step of the type."""
    off = bound * want.abs() + extra
    step = torch.exp2(torch.floor(torch.log2(want.abs() + off)) - BITS[got.dtype])
    allow = off + step + tiny(got.dtype)
    d = (got.double() - want).abs()
    bad = ~(d <= allow)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()}, worst "
                           f"{((d - step) / want.abs())[bad].max():.3g} past the rounding, "
                           f"allowed {bound:.3g}")


def _positive(R, G, K, M, dtype, seed, top=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    c = {"x": rand(R, K).to(dtype), "weights": rand(G, M, K).to(dtype), "biases": rand(G, M).to(dtype)}
    return c, (0.1 + 0.8 * rand(R, M)).to(dtype), (top * rand(R, M)).to(dtype)


def _weight_sums(x, y, v, act, edges):
    v = v.double() * y.double() * (1 - y.double()) if act == "sigmoid" else v.double()
    x = x.double()
    spans = list(zip(edges, edges[1:]))
    return (torch.stack([v[a:b].T @ x[a:b] for a, b in spans]),
            torch.stack([v[a:b].sum(0) for a, b in spans]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_long_group_in_one_pass(gs, cuda, dtype, act):
    """The whole backward in one kernel: 16-bit rows, up to 128 features.  An
    accumulator takes 4 tiles of 8 steps, then come 11 pieces and 148 places.
    (Of 32 tiles it would be 2.5e-5 low.)"""
    from gsplat_core.grouped import grouped_linear_backward
    R, edges = 800_000, [0, 700, 800_000]
    c, y, v = _positive(R, 2, 128, 128, TYPES[dtype], 3, top=1 / 16)
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    got = grouped_linear_backward(c, y, v, activation=act, wanted=("v_weights", "v_biases"))
    w, b = _weight_sums(c["x"], y, v, act, edges)
    # v_z behind the sigmoid: three roundings of 2^-24, two parts of 16 bits
    extra = (3 * 2.0 ** -24 + 2.0 ** (-22 if dtype == "fp16" else -16)) if act == "sigmoid" else 0.0
    bound = _bound(32, 160, TYPES[dtype]) + extra
    _assert_sums(got["v_weights"], w, bound, what="v_weights")
    _assert_sums(got["v_biases"], b, _bound(0, 1200, TYPES[dtype]) + extra, what="v_biases")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
@pytest.mark.parametrize("R,K,M", [(600_000, 200, 130), (40_000, 1024, 1024)])
def test_long_group_of_wide_rows(gs, cuda, dtype, act, R, K, M):
    """16-bit rows past 128 features: the second shape has four CTAs to a tile
    of the weights, 10,000 rows each.  An accumulator takes 8 panels of 4 steps,
    then come up to 20 pieces and 74 places.  v_biases: a thread's rows of a
    piece, and the same."""
    from gsplat_core.grouped import grouped_linear_backward
    edges = [0, 700, R]
    c, y, v = _positive(R, 2, K, M, TYPES[dtype], 4, top=1 / 16)
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    got = grouped_linear_backward(c, y, v, activation=act, wanted=("v_weights", "v_biases"))
    w, b = _weight_sums(c["x"], y, v, act, edges)
    extra = (3 * 2.0 ** -24 + 2.0 ** (-22 if dtype == "fp16" else -16)) if act == "sigmoid" else 0.0
    _assert_sums(got["v_weights"], w, _bound(32, 94, TYPES[dtype]) + extra, what="v_weights")
    _assert_sums(got["v_biases"], b, _bound(0, 300, TYPES[dtype]) + extra, what="v_biases")


@pytest.mark.parametrize("act", ["none", "sigmoid"])
@pytest.mark.parametrize("K,M", [(64, 64), (64, 100), (32, 3)])
def test_long_group_fp32(gs, cuda, act, K, M):
    """An accumulator takes 4 panels of 4 steps, registers then 43 of them, then
    come 148 places (few outputs have no accumulator: a lane's 10 runs of 4
    rows up to 32 lanes, 8 warps and 296 places).  Kept in one accumulator a
    CTA's 675 steps would lose 2.3e-5, six times what is allowed here."""
    from gsplat_core.grouped import grouped_linear_backward
    R, edges = 800_000, [0, 700, 800_000]
    c, y, v = _positive(R, 2, K, M, torch.float32, 5)
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    got = grouped_linear_backward(c, y, v, activation=act, wanted=("v_weights", "v_biases"))
    w, b = _weight_sums(c["x"], y, v, act, edges)
    extra = 3 * 2.0 ** -24 if act == "sigmoid" else 0.0
    _assert_sums(got["v_weights"], w, _bound(16, 400, torch.float32) + extra, what="v_weights")
    _assert_sums(got["v_biases"], b, _bound(0, 400, torch.float32) + extra, what="v_biases")


@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("K,M,act", [(16384, 40, "none"), (6001, 70, "sigmoid"), (2048, 128, "relu"),
                                     (777, 33, "none")])
def test_deep_rows_fp32(gs, cuda, gathered, K, M, act):
    """Forward and v_x through many features: an accumulator takes 8 panels of
    4 additions, and up to 64 pieces are added up in fp32."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    R, edges = 300, [0, 130, 131, 131, 300]
    spans = list(zip(edges, edges[1:]))
    c, _, _ = _positive(R, 4, K, M, torch.float32, 6)
    if act == "sigmoid":  # z of order one, so that y says something of it
        c["weights"] /= K / 4
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    ids = torch.randperm(R, generator=torch.Generator().manual_seed(1)).cuda()
    rows = c["x"].double()
    if gathered:
        c["row_ids"] = ids.to(torch.int32)
        rows = rows[ids]
    z = torch.cat([rows[a:b] @ c["weights"][g].double().T + c["biases"][g].double()
                   for g, (a, b) in enumerate(spans)])
    y = grouped_linear_forward(c, activation=act)
    bound = _bound(32, 64, torch.float32)
    if act == "sigmoid":  # dy = y (1 - y) dz, and eight units of its own
        want = torch.sigmoid(z)
        off = bound * z * want * (1 - want) + 8 * 2.0 ** -24 * want
        assert bool(((y.double() - want).abs() <= off).all())
    else:
        _assert_sums(y, z, bound, what="y")
    # v_x: the same with M and K in each other's place
    c, _, v = _positive(R, 4, M, K, torch.float32, 7)
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    if gathered:
        c["row_ids"] = ids.to(torch.int32)
    y = torch.full_like(v, 0.25)
    vz = {"none": 1.0, "relu": 1.0, "sigmoid": 0.1875}[act] * v.double()
    want = torch.cat([vz[a:b] @ c["weights"][g].double() for g, (a, b) in enumerate(spans)])
    got = grouped_linear_backward(c, y, v, activation=act, wanted=("v_x",))["v_x"]
    if gathered:
        got = got[ids]
    _assert_sums(got, want, bound + (3 * 2.0 ** -24 if act == "sigmoid" else 0.0), what="v_x")


@pytest.mark.parametrize("gathered", [False, True])
@pytest.mark.parametrize("K,M,R", [(64, 16, 200_000), (77, 45, 50_000), (200, 136, 50_000), (32, 3, 50_000)])
@pytest.mark.parametrize("size", ["1e-6", "2^-24", "1"])
def test_small_gradients_of_fp16_behind_a_sigmoid(gs, cuda, gathered, K, M, R, size):
    """v_z = v_y y (1 - y) is below fp16's normal range, or all of its range,
    before it is multiplied: it is carried to 2^-22 of itself and to 2^-36,
    and its sums are right where fp16 holds them."""
    from gsplat_core.grouped import grouped_linear_backward
    half = torch.float16
    top = {"1e-6": 1e-6, "2^-24": 2.0 ** -24, "1": 1.0}[size]
    c, y, v = _positive(R, 2, K, M, half, 8)
    v = torch.full_like(v, top) if top < 1 else v / 64
    edges = [0, 900, R]
    c["offsets"] = torch.tensor(edges, dtype=torch.int32, device="cuda")
    w = c["weights"] = c["weights"] * (1 if top == 1 else 256)  # so that v_x is in fp16's range
    rows = c["x"]
    if gathered:
        ids = torch.randperm(R, generator=torch.Generator().manual_seed(1)).cuda()
        c["row_ids"] = ids.to(torch.int32)
        rows = rows[ids]
    vz = v.double() * y.double() * (1 - y.double())
    want_w, want_b = _weight_sums(rows, y, v, "sigmoid", edges)
    want_x = torch.cat([vz[:900] @ w[0].double(), vz[900:] @ w[1].double()])
    # of itself: two parts, three roundings; below: half a step of the second part
    part = 2.0 ** -22 + 3 * 2.0 ** -24
    low = lambda other: 2.0 ** -36 * other.double().abs().sum(0)  # noqa: E731
    for wanted in (("v_x", "v_weights", "v_biases"), ("v_x",)):
        got = grouped_linear_backward(c, y, v, activation="sigmoid", wanted=wanted)
        x = got["v_x"][ids] if gathered else got["v_x"]
        for s, g in ((slice(0, 900), 0), (slice(900, R), 1)):
            _assert_sums(x[s], want_x[s], _bound(9, 4, half) + part, low(w[g]), what="v_x")
            if "v_weights" in got:
                _assert_sums(got["v_weights"][g], want_w[g], _bound(32, 400, half) + part,
                             low(rows[s]), what="v_weights")
                _assert_sums(got["v_biases"][g], want_b[g], _bound(0, 400, half) + part,
                             what="v_biases")
