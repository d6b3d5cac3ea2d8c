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
