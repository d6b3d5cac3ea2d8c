"""gsplat_core.grouped on the device against the same sums in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _learned import TYPES, assert_sums, half_step, linear, tiny

pytestmark = pytest.mark.gpu

# (group sizes, N (0: no row ids), K, M)
SHAPES = [
    ([1], 0, 1, 1), ([1], 0, 16, 3), ([257], 0, 16, 3), ([128, 128], 0, 32, 32),
    ([127, 0, 129, 1, 0], 0, 64, 64), ([0, 0, 300], 90, 64, 64), ([50, 0, 7, 1000], 400, 32, 3),
    ([333, 444], 0, 128, 128), ([200, 1, 3], 60, 77, 45), ([77, 78], 0, 3, 64), ([500], 700, 48, 16),
    ([130, 131], 0, 200, 130), ([65], 0, 300, 257), ([40, 41], 33, 257, 20), ([3] * 70, 100, 20, 12),
    ([2500, 1800, 3000], 5000, 64, 32), ([64], 0, 65, 33), ([4097], 0, 8, 100), ([300], 0, 520, 40),
]

# up to 8 outputs, of rows that fill one to 32 lanes, and the first past that
FEW = [
    ([1000], 0, 32, 1), ([300, 0, 77], 500, 64, 3), ([257, 4], 0, 128, 4), ([90, 91], 60, 100, 2),
    ([513], 700, 48, 8), ([40] * 40, 100, 16, 5), ([333], 0, 250, 3), ([129, 1], 99, 7, 7),
    ([700], 0, 256, 8), ([2000, 3000], 1500, 4, 4), ([65], 0, 129, 3), ([65], 80, 257, 3),
    ([31, 1, 1, 64], 20, 8, 6), ([5], 3, 1, 8)]
# more features than shared memory holds weights of
MANY = [([150, 90], 0, 3700, 24), ([150, 90], 60, 24, 3700), ([140], 0, 1000, 40)]


def _case(sizes, N, K, M, dtype, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    R, G = sum(sizes), len(sizes)
    rand = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    c = {"x": rand(N or R, K).to(dtype).cuda(),
         "weights": (rand(G, M, K) / K ** 0.5).to(dtype).cuda(),
         "offsets": torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32).cuda()}
    if bias:
        c["biases"] = rand(G, M).to(dtype).cuda()
    if N:
        c["row_ids"] = torch.randint(0, N, (R,), generator=g, dtype=torch.int32).cuda()
    return c, rand(R, M).to(dtype).cuda()


def _parts(c):
    return c["x"], c["weights"], c["offsets"], c.get("biases"), c.get("row_ids")


def _check_forward(c, y, act):
    """Activations: relu does not enlarge an error, the sigmoid quarters it;
    it is off by at most eight units itself (exp, sum, quotient)."""
    want, mag = linear(*_parts(c), act=act)["y"]
    extra = 8 * 2.0 ** -24 if act == "sigmoid" else 0.0
    assert_sums(y, want, mag, c["x"].shape[1] + 1, c["x"].dtype, extra, "y")


def _check_backward(c, y, v_y, got, act):
    """v_z = v y (1 - y) takes three roundings of 2^-24 in fp32 (none for
    relu): within the twelve extra products' units.  16-bit v_z is carried
    in two 16-bit parts: off by 2^-16 of itself at most (bf16; fp16 2^-22,
    and by 2^-25 where it is subnormal), on top of the magnitude."""
    want = linear(*_parts(c), act=act, v_y=v_y, y=y)
    x, w, off = c["x"], c["weights"], c["offsets"]
    dt = x.dtype
    R = v_y.shape[0]
    hits = R if "row_ids" in c else 1   # rows that may meet in one row of x
    for k, terms in (("v_x", w.shape[1] + (hits if "row_ids" in c else 0)), ("v_weights", R),
                     ("v_biases", R)):
        if k not in got:
            continue
        val, mag = want[k]
        extra = 0.0
        if act == "sigmoid" and dt != torch.float32:
            extra = 2.0 ** -15 * mag
            if dt == torch.float16:
                other = {"v_x": w.double().abs().sum(1).max().item() * (1 if hits == 1 else R),
                         "v_weights": x.double().abs().sum(0).max().item() * hits, "v_biases": R}
                extra = extra + 2.0 ** -25 * other[k]
        assert_sums(got[k], val, mag, terms, dt, extra, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,N,K,M", SHAPES + FEW + MANY)
@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
def test_grouped_matches_64_bits(gs, cuda, dtype, sizes, N, K, M, act):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case(sizes, N, K, M, TYPES[dtype], bias=act != "none")
    y = grouped_linear_forward(c, activation=act)
    _check_forward(c, y, act)
    got = grouped_linear_backward(c, y, v_y, activation=act)
    assert set(got) == {"v_x", "v_weights"} | ({"v_biases"} if "biases" in c else set())
    _check_backward(c, y, v_y, got, act)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_that_are_not_aligned(gs, cuda, dtype):
    """Every operand starts one value off, so no access may be wide."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([70, 0, 200], 150, 32, 16, TYPES[dtype])

    def off(t):
        b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        b[1:] = t.reshape(-1)
        return b[1:].view(t.shape)

    s = {k: off(t) for k, t in c.items()}
    y = grouped_linear_forward(s, activation="relu")
    _check_forward(c, y, "relu")
    _check_backward(c, y, v_y, grouped_linear_backward(s, off(y), off(v_y), activation="relu"), "relu")


def test_rows_outside_groups_and_ids_outside_x(gs, cuda):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([200, 300, 100], 50, 32, 24, torch.float32)
    c["offsets"] = torch.tensor([30, 170, 170, 420], dtype=torch.int32, device="cuda")
    c["row_ids"][100:110] = -1
    c["row_ids"][250:260] = 50
    c["row_ids"][300] = 2 ** 31 - 1
    for act in ("none", "sigmoid"):
        y = grouped_linear_forward(c, activation=act)
        assert not y[:30].any() and not y[420:].any()
        _check_forward(c, y, act)
        _check_backward(c, y, v_y, grouped_linear_backward(c, y, v_y, activation=act), act)
    # no row ids: rows of x outside every group get zero gradients
    c, v_y = _case([200, 300, 100], 0, 32, 24, torch.float32)
    c["offsets"] = torch.tensor([30, 170, 170, 420], dtype=torch.int32, device="cuda")
    y = grouped_linear_forward(c, activation="sigmoid")
    got = grouped_linear_backward(c, y, v_y, activation="sigmoid")
    assert not got["v_x"][:30].any() and not got["v_x"][420:].any()
    _check_backward(c, y, v_y, got, "sigmoid")


def test_offsets_that_do_not_ascend_stay_in_bounds(gs, cuda):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([200, 300, 100, 5], 0, 16, 8, torch.float32)
    for off in ([0, 500, 100, 600, 605], [-7, 3, 1000, 2, 9999], [605, 0, 0, 0, 0], [5, 5, 5, 5, 5]):
        c["offsets"] = torch.tensor(off, dtype=torch.int32, device="cuda")
        y = grouped_linear_forward(c)
        grouped_linear_backward(c, y, v_y)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(gs, cuda, dtype):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    for N in (0, 9):
        c, v_y = _case([0, 0], N, 8, 4, TYPES[dtype])
        y = grouped_linear_forward(c, activation="relu")
        assert y.shape == (0, 4)
        got = grouped_linear_backward(c, y, v_y, activation="relu")
        assert got["v_x"].shape == c["x"].shape
        for t in got.values():
            assert not t.any()
    # ids into an x without rows: every row reads zeros
    c, _ = _case([5, 6], 4, 8, 4, TYPES[dtype])
    c["x"] = c["x"][:0]
    assert torch.equal(grouped_linear_forward(c), c["biases"].repeat_interleave(
        torch.tensor([5, 6], device="cuda"), dim=0))
    # and their gradients: none for x, zeros for the weights, v_y's sums for the biases
    for K, M in ((8, 4), (16, 16), (77, 45), (200, 9)):
        c, v_y = _case([5, 6], 4, K, M, TYPES[dtype])
        c["x"] = c["x"][:0]
        g = grouped_linear_backward(c, None, v_y)
        assert g["v_x"].shape == (0, K) and not g["v_weights"].any()
        want = torch.stack([v_y[:5].double().sum(0), v_y[5:].double().sum(0)]).cpu()
        assert_sums(g["v_biases"], want, v_y.double().abs().sum(0).cpu().expand(2, M), 11, TYPES[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,M", [(64, 64), (20, 7)])
def test_non_finite_values(gs, cuda, dtype, K, M):
    """A NaN or an infinity reaches exactly what the formula has it reach,
    with the formula's sign; in fp32 so do values next to the largest."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    dt = TYPES[dtype]
    c, v_y = _case([300, 200], 0, K, M, dt, bias=False)
    big = torch.finfo(dt).max
    for r, v in ((3, float("nan")), (140, float("inf")), (141, float("-inf")), (310, float("inf"))):
        c["x"][r, r % K] = v
    c["x"][200] = 0.0
    c["x"][200, 5] = big / 4
    c["weights"][1, 2, 1] = float("inf")
    y = grouped_linear_forward(c)
    want, _ = linear(*_parts(c))["y"]
    fine = torch.isfinite(want)
    got = y.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    assert bool(torch.isfinite(got[fine]).all())
    # one product: fp32 factors are carried to 2^-22 of themselves each, which
    # is 8 half steps of 2^-24, and the two partial sums and their join take a
    # rounding of up to a step each; 16-bit ones are exact up to the last
    assert torch.allclose(got[200], want[200], rtol=(8 + 6) * half_step(dt), atol=0)
    # the backward: a NaN row of v_y stays in its row of v_x, its column of v_weights
    c, v_y = _case([300, 200], 0, K, M, dt, bias=True)
    y = grouped_linear_forward(c)
    v_y[7, 3], v_y[400, 1] = float("nan"), float("inf")
    g = grouped_linear_backward(c, y, v_y)
    ref = linear(*_parts(c), v_y=v_y, y=y)
    for k in g:
        want = ref[k][0]
        got = g[k].double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), k
        inf = torch.isinf(want)
        assert torch.equal(got[inf], want[inf]), k


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time(gs, cuda, dtype):
    """Everything but the atomic sums of shared rows has a fixed order; with
    ids that name a row once v_x has one too."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([5000, 1, 0, 7000], 0, 64, 48, TYPES[dtype])
    c["row_ids"] = torch.randperm(12001, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    y = grouped_linear_forward(c, activation="relu")
    one = grouped_linear_backward(c, y, v_y, activation="relu")
    for _ in range(3):
        assert torch.equal(y, grouped_linear_forward(c, activation="relu"))
        two = grouped_linear_backward(c, y, v_y, activation="relu")
        for k in one:
            assert torch.equal(one[k], two[k]), k


def test_wanted_gradients(gs, cuda):
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([500, 300], 200, 64, 32, torch.float32)
    y = grouped_linear_forward(c, activation="sigmoid")
    for wanted in (("v_x",), ("v_weights",), ("v_biases",), ("v_weights", "v_biases"), ()):
        got = grouped_linear_backward(c, y, v_y, activation="sigmoid", wanted=wanted)
        assert set(got) == set(wanted)
        _check_backward(c, y, v_y, got, "sigmoid")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,M,N", [(64, 32, 0), (77, 45, 300), (32, 3, 300), (200, 40, 0)])
def test_wanted_gradients_of_each_kernel(gs, cuda, dtype, K, M, N):
    """Any subset gives the bits of the whole (v_x of shared rows: within
    their tolerance, their order is not fixed)."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([500, 0, 300], N, K, M, TYPES[dtype])
    y = grouped_linear_forward(c, activation="relu")
    whole = grouped_linear_backward(c, y, v_y, activation="relu")
    _check_backward(c, y, v_y, whole, "relu")
    for wanted in (("v_x",), ("v_weights",), ("v_biases",), ("v_x", "v_biases")):
        got = grouped_linear_backward(c, y, v_y, activation="relu", wanted=wanted)
        assert set(got) == set(wanted)
        _check_backward(c, y, v_y, got, "relu")
        for k in wanted:
            if k != "v_x":
                assert torch.equal(got[k], whole[k]), k


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(gs, cuda, dtype):
    """Inputs that are not contiguous are taken as they read."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    c, v_y = _case([200, 70], 150, 32, 24, TYPES[dtype])
    s = {"x": c["x"].t().contiguous().t(), "weights": c["weights"].transpose(1, 2).contiguous().transpose(1, 2),
         "biases": c["biases"].repeat_interleave(2, dim=1)[:, ::2],
         "offsets": c["offsets"].repeat_interleave(3)[::3], "row_ids": c["row_ids"].repeat_interleave(2)[::2]}
    assert not any(t.is_contiguous() for t in s.values())
    y = grouped_linear_forward(s, activation="sigmoid")
    assert torch.equal(y, grouped_linear_forward(c, activation="sigmoid"))
    g = grouped_linear_backward(s, y.t().contiguous().t(), v_y.t().contiguous().t(), activation="sigmoid")
    _check_backward(c, y, v_y, g, "sigmoid")


def test_no_second_derivative(gs, cuda):
    """A second derivative is refused instead of being zero."""
    from gsplat_core import autograd as A
    c, _ = _case([20], 0, 8, 4, torch.float32)
    x = c["x"].clone().requires_grad_(True)
    for y in (A.grouped_linear(x, c["weights"], c["offsets"], activation="sigmoid"),
              A.dropout(x, 0.5, 1)):
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_graphs_and_streams(gs, cuda):
    """Two captured graphs replayed on two streams at once, with other
    calls, and a call on a side stream: each has its own scratch."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    cases = [_case([3000, 2000], 4000, 64, 64, torch.bfloat16, seed=i) for i in range(2)]
    want, graphs, outs = [], [], []
    for c, v in cases:
        y = grouped_linear_forward(c, activation="relu")
        want.append((y, grouped_linear_backward(c, y, v, activation="relu")))
    torch.cuda.synchronize()
    for c, v in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = grouped_linear_forward(c, activation="relu")
            outs.append((y, grouped_linear_backward(c, y, v, activation="relu")))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (y, gy), (z, gz), (c, v) in zip(want, outs, cases):
        assert torch.equal(y, z)
        assert torch.equal(gy["v_weights"], gz["v_weights"])
        assert torch.equal(gy["v_biases"], gz["v_biases"])
        _check_backward(c, z, v, gz, "relu")


@pytest.mark.parametrize("n,groups", [(0, 0), (0, 3), (1, 1), (1000, 7), (70_000, 1), (500, 2000)])
def test_group_offsets(gs, cuda, n, groups):
    from gsplat_core.grouped import group_offsets
    ids = np.sort(np.random.default_rng(n).integers(0, max(groups, 1), size=n)).astype(np.int32)
    off = group_offsets(torch.from_numpy(ids).cuda(), groups)
    assert np.array_equal(off.cpu().numpy(), np.searchsorted(ids, np.arange(groups + 1)))


def test_autograd_and_differences(gs, cuda):
    """Gradients through autograd against central differences of the 64-bit
    forward along one direction per leaf."""
    from gsplat_core import autograd as A
    c, v = _case([60, 0, 90], 40, 24, 10, torch.float32)
    leaves = {k: c[k].clone().requires_grad_(True) for k in ("x", "weights", "biases")}
    y = A.grouped_linear(leaves["x"], leaves["weights"], c["offsets"], leaves["biases"],
                         c["row_ids"], "sigmoid")
    y.backward(v)
    g = torch.Generator().manual_seed(3)
    for k, leaf in leaves.items():
        d = torch.randn(leaf.shape, generator=g, dtype=torch.float64)
        h = 1e-4
        f = []
        for s in (h, -h):
            q = dict(c)
            q[k] = c[k].double().cpu() + s * d
            f.append(float((linear(*_parts(q), act="sigmoid")["y"][0] * v.double().cpu()).sum()))
        want = (f[0] - f[1]) / (2 * h)
        got = float((leaf.grad.double().cpu() * d).sum())
        # h^2 of the third derivative, and fp32 sums of 10^4 products
        assert abs(got - want) <= 1e-4 * abs(want) + 1e-3, (k, got, want)
    # a leaf that wants no gradient gets none, and none is computed
    x = c["x"].clone().requires_grad_(True)
    A.grouped_linear(x, c["weights"], c["offsets"], None, c["row_ids"]).backward(v)
    assert x.grad is not None


def test_large_offsets_pass_32_bits(gs, cuda):
    """R M and R K beyond 2^31 values: the last rows are right."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    R, K, M = 17_000_000, 130, 128
    x = torch.zeros((R, K), dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, K, device="cuda").to(torch.bfloat16)
    w = (torch.randn(2, M, K, device="cuda") / 11).to(torch.bfloat16)
    off = torch.tensor([0, R - 100, R], dtype=torch.int32, device="cuda")
    c = {"x": x, "weights": w, "offsets": off}
    y = grouped_linear_forward(c)
    tail = {"x": x[-300:].contiguous(), "weights": w,
            "offsets": torch.tensor([0, 200, 300], dtype=torch.int32, device="cuda")}
    _check_forward(tail, y[-300:], "none")
    assert not y[:-300].any()
    v = torch.zeros_like(y)
    v[-300:] = torch.randn(300, M, device="cuda").to(torch.bfloat16)
    g = grouped_linear_backward(c, y, v)
    assert not g["v_x"][:-300].any()
    g["v_x"] = g["v_x"][-300:].contiguous()
    _check_backward(tail, y[-300:].contiguous(), v[-300:].contiguous(), g, "none")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
@pytest.mark.parametrize("K,M", [(16, 16), (24, 72)])
def test_long_group(gs, cuda, dtype, act, K, M):
    """Many tiles of one group for every CTA: sums that leave the accumulators
    in between are neither lost nor added twice.  All positive, so that the
    magnitude is the value.  One accumulator takes at most 32 tiles of 8
    additions (each of up to 16 products), then come at most 48 pieces and 296
    places: 1000 additions one after the other are an upper bound."""
    from gsplat_core.grouped import grouped_linear_backward
    R = 800_000
    g = torch.Generator(device="cuda").manual_seed(2)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda").to(TYPES[dtype])  # noqa: E731
    c = {"x": rand(R, K), "weights": rand(2, M, K), "biases": rand(2, M),
         "offsets": torch.tensor([0, 700, R], dtype=torch.int32, device="cuda")}
    y, v_y = rand(R, M), rand(R, M)
    got = grouped_linear_backward(c, y, v_y, activation=act, wanted=("v_weights", "v_biases"))
    want = linear(*_parts(c), act=act, v_y=v_y, y=y)
    for k in got:
        val, mag = want[k]
        extra = 0.0
        if act == "sigmoid" and dtype != "fp32":
            extra = 2.0 ** -15 * mag + (2.0 ** -25 * R if dtype == "fp16" else 0.0)
        if dtype == "fp16":
            _half_sums(got[k], val, mag, extra, k)
        else:
            assert_sums(got[k], val, mag, 1000, TYPES[dtype], extra, k)


def _half_sums(got, val, mag, extra, what):
    """fp16 overflows at 65504: infinite exactly where the sum is past it (by
    more than the tolerance), else within the tolerance."""
    far = val > 65520 * (1 + 1e-3)
    assert bool(torch.isinf(got.cpu()[far]).all()), what
    near = val < 65520 * (1 - 1e-3)
    ex = extra[near] if isinstance(extra, torch.Tensor) else extra
    assert_sums(got.cpu()[near], val[near], mag[near], 1000, torch.float16, ex, what)


def test_many_groups(gs, cuda):
    """More groups than a grid is high, most of them of one row or none."""
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    rng = np.random.default_rng(5)
    sizes = rng.integers(0, 3, size=70_000)
    for K, M in ((4, 2), (8, 16)):
        c, v_y = _case(sizes.tolist(), 0, K, M, torch.float32)
        y = grouped_linear_forward(c, activation="relu")
        row = torch.from_numpy(np.repeat(np.arange(70_000), sizes)).cuda()
        z = torch.einsum("rk,rmk->rm", c["x"].double(), c["weights"][row].double()) + c["biases"][row]
        assert torch.allclose(y.double(), z.clamp(min=0), rtol=1e-6, atol=1e-5)
        g = grouped_linear_backward(c, y, v_y, activation="relu")
        v = torch.where(y > 0, v_y, torch.zeros_like(v_y)).double()
        vw = torch.zeros(70_000, M, K, dtype=torch.float64, device="cuda").index_add_(
            0, row, v[:, :, None] * c["x"].double()[:, None])
        assert torch.allclose(g["v_weights"].double(), vw, rtol=1e-6, atol=1e-5)
        vb = torch.zeros(70_000, M, dtype=torch.float64, device="cuda").index_add_(0, row, v)
        assert torch.allclose(g["v_biases"].double(), vb, rtol=1e-6, atol=1e-5)
        vx = torch.einsum("rm,rmk->rk", v, c["weights"][row].double())
        assert torch.allclose(g["v_x"].double(), vx, rtol=1e-6, atol=1e-5)


def test_no_wait_gave_up(gs, cuda):
    """Last in this file: no bounded wait of the calls above ran out."""
    from gsplat_core import grouped
    grouped.check()
