"""The dropout and the grouped products as they are used together: a step of
a splat model whose colours are learned per camera, on the packed rows, and
the image-fitting iteration with dropped Gaussians."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from _learned import assert_sums, keep_mask, linear

pytestmark = pytest.mark.gpu


def T(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.mark.parametrize("channels,hidden", [(3, False), (8, True)])
def test_packed_step_with_learned_colors(gs, cuda, channels, hidden):
    from gsplat_core import packed as P, synthetic as S
    from gsplat_core.dropout import dropout_backward, dropout_forward
    from gsplat_core.grouped import grouped_linear_backward, grouped_linear_forward
    sc = S.config3(seed=6, n=60_000)
    idx = np.sort(np.random.default_rng(7).choice(sc.n, size=20_000, replace=False))
    cams, K, N, ts = 3, 16, idx.size, 16
    Ks = np.repeat(sc.Ks[:1], cams, 0).copy()
    Ks[:, :2, :] /= 8
    W, H = sc.width // 8, sc.height // 8
    tw, th = (W + 15) // 16, (H + 15) // 16
    proj = gs.projection_ewa_3dgs_fused_forward(
        {"means": T(sc.means[idx][None]), "quats": T(sc.quats[idx][None]),
         "scales": T(sc.scales[idx][None]), "viewmats": T(S.orbit(cams, 4.0)[None]), "Ks": T(Ks[None])},
        W, H)
    pk = P.pack_projection(proj)
    img = pk["image_ids"].cpu().numpy()
    assert np.array_equal(pk["image_offsets"].cpu().numpy(), np.searchsorted(img, np.arange(cams + 1)))
    g = torch.Generator().manual_seed(1)
    feats = torch.randn(N, K, generator=g).cuda()
    wide = 32 if hidden else K
    w1 = (torch.randn(cams, 32, K, generator=g) / 4).cuda()
    w2 = (torch.randn(cams, channels, wide, generator=g) / wide ** 0.5).cuda()
    b2 = torch.randn(cams, channels, generator=g).cuda()
    opac = T(sc.opacities[idx])
    drop = (0.3, 17, 5, True)
    # forward: whole Gaussians dropped, colours from the features per camera
    opac_kept = dropout_forward(opac, *drop)
    rows = feats
    if hidden:
        first = {"x": feats, "weights": w1, "offsets": pk["image_offsets"], "row_ids": pk["gaussian_ids"]}
        h = grouped_linear_forward(first, activation="relu")
        hd = dropout_forward(h, 0.5, 18, 5)
        second = {"x": hd, "weights": w2, "biases": b2, "offsets": pk["image_offsets"]}
        colors = grouped_linear_forward(second, activation="sigmoid")
        rows = hd
    else:
        colors = P.camera_colors_forward(feats, w2, b2, pk)
    ids = None if hidden else pk["gaussian_ids"]
    want, mag = linear(rows, w2, pk["image_offsets"], b2, ids, "sigmoid")["y"]
    assert_sums(colors, want, mag, wide + 1, torch.float32, 8 * 2.0 ** -24, "colors")
    it = P.intersect_tile_packed_forward(pk, cams, ts, tw, th)
    rin = {"means2d": pk["means2d"], "conics": pk["conics"], "colors": colors,
           "opacities": opac_kept[pk["gaussian_ids"].long()]}
    out = P.rasterize_packed_forward(rin, it, cams, W, H, ts)
    # the dropped Gaussians leave the image: as if their rows were not there
    keep = T(keep_mask((N,), 0.3, 17, 5, True).copy())
    gone = dict(rin, opacities=rin["opacities"] * keep[pk["gaussian_ids"].long()])
    assert torch.equal(P.rasterize_packed_forward(gone, it, cams, W, H, ts)["render_colors"],
                       out["render_colors"])
    cot = {"v_render_colors": torch.randn(out["render_colors"].shape, generator=g).cuda(),
           "v_render_alphas": torch.zeros_like(out["render_alphas"])}
    rb = P.rasterize_packed_backward(rin, it, out, cot, cams, W, H, ts)
    # backward through the colours to the features
    if hidden:
        gr = grouped_linear_backward(second, colors, rb["v_colors"], activation="sigmoid")
        ref = linear(hd, w2, pk["image_offsets"], b2, None, "sigmoid", rb["v_colors"], colors)
        v_h = dropout_backward(gr["v_x"], 0.5, 18, 5)
        assert bool((v_h[~T(keep_mask(tuple(h.shape), 0.5, 18, 5, False).copy())] == 0).all())
        g1 = grouped_linear_backward(first, h, v_h, activation="relu")
        ref1 = linear(feats, w1, pk["image_offsets"], None, pk["gaussian_ids"], "relu", v_h, h)
        assert_sums(g1["v_x"], *ref1["v_x"], 32 + cams, torch.float32, what="v_features")
        assert_sums(g1["v_weights"], *ref1["v_weights"], img.size, torch.float32, what="v_w1")
    else:
        gr = P.camera_colors_backward(feats, w2, b2, pk, colors, rb["v_colors"])
        ref = linear(feats, w2, pk["image_offsets"], b2, pk["gaussian_ids"], "sigmoid",
                     rb["v_colors"], colors)
        assert_sums(gr["v_features"], *ref["v_x"], channels + cams, torch.float32, what="v_features")
    assert_sums(gr["v_weights"], *ref["v_weights"], img.size, torch.float32, what="v_weights")
    assert_sums(gr["v_biases"], *ref["v_biases"], img.size, torch.float32, what="v_biases")
    v_opac = torch.zeros(N, device="cuda").index_add_(0, pk["gaussian_ids"].long(), rb["v_opacities"])
    v_opac = dropout_backward(v_opac, *drop)
    assert bool((v_opac[~keep] == 0).all()) and bool((v_opac[keep] != 0).any())


def test_fit_step_with_dropout(gs, cuda):
    """An iteration with dropout moves exactly the kept Gaussians' moments,
    renders the dropped ones not at all, and draws anew each iteration; with
    dropout 0 it is the iteration without it, bit for bit in its inputs."""
    from gsplat_core import fitting
    from test_gpu_fitting import _problem
    means, quats, ls, cl, ol, view, K, target, size = _problem(n=2000, size=64, seed=4)
    mk = lambda **kw: fitting.ImageFitStep(means, quats, ls, cl, ol, view, K, target, size, size,  # noqa: E731
                                           **kw)
    fit = mk(dropout=0.4, dropout_seed=33)
    seen = np.zeros(2000, bool)
    for it in range(3):
        o = fit.opacities.clone()
        fit.run()
        keep = keep_mask((2000,), 0.4, 33, it, True)
        kt = T(keep.copy())
        used = fit.opacities_kept
        assert bool((used[~kt] == 0).all())
        assert torch.equal(used[kt], o[kt] * torch.tensor(1 / 0.6, device="cuda"))
        assert bool((fit.step.v_opacities[~kt] == 0).all())
        assert bool((fit.step.v_colors[0][~kt] == 0).all())
        seen |= keep
        m = fit.m1[:, 13].cpu().numpy()
        assert (m[~seen] == 0).all() and (m[seen] != 0).any()
    a, b = mk(), mk(dropout=0.0, dropout_seed=5)
    assert float(a.run()) == pytest.approx(float(b.run()), rel=1e-6)


def test_captured_training_step(gs, cuda):
    """Forward and backward through autograd in one captured graph, with a
    new mask at each replay: the gradients of an eager step of that mask."""
    from gsplat_core import autograd as A
    g = torch.Generator().manual_seed(4)
    x = torch.randn(900, 16, generator=g).cuda().requires_grad_(True)
    w = (torch.randn(3, 24, 16, generator=g) / 4).cuda().requires_grad_(True)
    b = torch.randn(3, 24, generator=g).cuda().requires_grad_(True)
    off = torch.tensor([0, 300, 320, 900], dtype=torch.int32, device="cuda")
    v = torch.randn(900, 24, generator=g).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def run(at):
        h = A.dropout(A.grouped_linear(x, w, off, b, None, "relu"), 0.3, 7, at)
        return torch.autograd.grad(h, (x, w, b), v)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(step)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = run(step)
    for it in (0, 3, 11):
        step.fill_(it)
        graph.replay()
        for got, want in zip(grads, run(it)):
            assert torch.equal(got, want), it
