"""Refusals of the dropout and the grouped products, raised before the
device is touched, and the host side of their C entries (no GPU needed)."""
from __future__ import annotations

import ctypes as ct
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from _learned import keep_mask, philox

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_philox_known_answers():
    """The published test vectors of Philox4x32 with 7 and 10 rounds, for
    counter and key zero."""
    assert philox(4, 0, 0, 7).tolist() == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    assert philox(4, 0, 0, 10).tolist() == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_mask_rate_and_independence():
    """A sixth dropped within five standard deviations; two steps, and two
    seeds, agree where chance has them agree."""
    n, p = 200_000, 1.0 / 6.0
    a, b, c = (keep_mask((n,), p, s, t, True) for s, t in ((7, 0), (7, 1), (8, 0)))
    for m in (a, b, c):
        assert abs((~m).mean() - p) < 5 * (p * (1 - p) / n) ** 0.5
    q = p * p + (1 - p) ** 2
    for m in (b, c):
        assert abs((a == m).mean() - q) < 5 * (q * (1 - q) / n) ** 0.5


@pytest.mark.parametrize("kw,match", [
    (dict(p=1.5), r"p must be in \[0, 1\]"), (dict(p=-0.1), r"p must be in"),
    (dict(p=float("nan")), r"p must be in"), (dict(x=torch.zeros(3, dtype=torch.int32)), "float32"),
    (dict(x=torch.zeros(3, dtype=torch.float64)), "float32"), (dict(x=None), "tensor"),
    (dict(x=torch.zeros(()), rows=True), "at least one dimension"),
    (dict(step=torch.zeros(1)), "one int64"), (dict(step=torch.zeros(2, dtype=torch.int64)), "one int64"),
    (dict(out=torch.zeros(4)), "out must be"), (dict(out=torch.zeros(3, dtype=torch.float16)), "out must be"),
    (dict(), "no CPU fallback")])
def test_dropout_refusals(gs, kw, match):
    from gsplat_core.dropout import dropout_forward
    a = dict(x=torch.zeros(3), p=0.5, seed=1)
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        dropout_forward(**a)


def test_dropout_rows_too_wide(gs):
    from gsplat_core.dropout import dropout_forward
    with pytest.raises(RuntimeError, match="fewer than 2\\^24"):
        dropout_forward(torch.zeros(1).expand(2, 1 << 24), 0.5, 1, rows=True)


def _inputs(**kw):
    a = {"x": torch.zeros(6, 4), "weights": torch.zeros(2, 5, 4),
         "offsets": torch.zeros(3, dtype=torch.int32)}
    a.update(kw)
    return {k: v for k, v in a.items() if v is not None}


@pytest.mark.parametrize("kw,match", [
    (dict(x=None), "missing input: x"), (dict(weights=None), "missing input: weights"),
    (dict(offsets=None), "missing input: offsets"),
    (dict(x=torch.zeros(6)), r"x must have shape"), (dict(x=torch.zeros(6, 4).double()), "x must have"),
    (dict(weights=torch.zeros(2, 5, 3)), "weights must have"),
    (dict(weights=torch.zeros(2, 5, 4).half()), "weights must have"),
    (dict(weights=torch.zeros(2, 0, 4)), "at least 1"),
    (dict(weights=torch.zeros(1, 1, 4).expand(2, 16385, 4)), "at most 16384"),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), "offsets must have"),
    (dict(offsets=torch.zeros(3, dtype=torch.int64)), "offsets must have"),
    (dict(biases=torch.zeros(2, 4)), "biases must have"),
    (dict(row_ids=torch.zeros(6, dtype=torch.int64)), "row_ids must have"),
    (dict(), "no CPU fallback")])
def test_grouped_refusals(gs, kw, match):
    from gsplat_core.grouped import grouped_linear_forward
    with pytest.raises(RuntimeError, match=match):
        grouped_linear_forward(_inputs(**kw))


def test_grouped_call_refusals(gs):
    from gsplat_core.grouped import group_offsets, grouped_linear_backward, grouped_linear_forward
    with pytest.raises(RuntimeError, match="activation must be"):
        grouped_linear_forward(_inputs(), activation="gelu")
    good, v = torch.zeros(6, 5), torch.zeros(6, 4)
    with pytest.raises(RuntimeError, match="y must have"):
        grouped_linear_backward(_inputs(), None, good, activation="relu")
    with pytest.raises(RuntimeError, match="v_y must have"):
        grouped_linear_backward(_inputs(), good, v, activation="relu")
    with pytest.raises(RuntimeError, match="wanted"):
        grouped_linear_backward(_inputs(), good, good, wanted=("v_offsets",))
    with pytest.raises(RuntimeError, match="1-D int32"):
        group_offsets(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(RuntimeError, match="negative number"):
        group_offsets(torch.zeros(3, dtype=torch.int32), -1)


def test_fit_dropout_refused(gs):
    from gsplat_core.fitting import ImageFitStep
    for p in (1.0, -0.5, float("nan")):
        with pytest.raises(RuntimeError, match="dropout must be"):
            ImageFitStep(*[None] * 8, 8, 8, device=torch.device("cpu"), dropout=p)


def test_c_entries_refuse_before_launch(gs):
    from gsplat_core import _lib as L
    lib = gs.load()

    def drop(rows=4, width=4, p=0.5, dtype=0, by_row=0):
        q = L.DropoutParams(rows, width, 1, 0, p, dtype, by_row)
        return lib.gs_dropout(ct.byref(q), None, None, None, None)

    assert drop(rows=0) == L.GS_OK and drop(width=0) == L.GS_OK
    for kw in (dict(), dict(rows=-1), dict(p=1.01), dict(p=float("nan")), dict(dtype=3),
               dict(width=1 << 24, by_row=1), dict(rows=1 << 40, width=1 << 40)):
        assert drop(**kw) == L.GS_ERR_INVALID, kw
    assert lib.gs_group_offsets(-1, None, 2, None, None) == L.GS_ERR_INVALID
    assert lib.gs_group_offsets(4, None, 2, None, None) == L.GS_ERR_INVALID

    def prm(rows=6, n=6, G=2, K=4, M=5, dtype=0, act=0, ids=0):
        return L.GroupedParams(rows, n, G, K, M, dtype, act, ids)

    fwd = lambda q: lib.gs_grouped_linear_fwd(ct.byref(q), *[None] * 7)  # noqa: E731
    assert fwd(prm(rows=0, n=0)) == L.GS_OK
    for q in (prm(), prm(n=5), prm(rows=-1), prm(G=0), prm(K=0), prm(M=0), prm(dtype=5), prm(act=3),
              prm(K=16385), prm(M=16385), prm(rows=2 ** 31 - 4000, n=2 ** 31 - 4000),
              prm(rows=2 ** 31, n=2 ** 31)):
        assert fwd(q) == L.GS_ERR_INVALID
        assert lib.gs_last_error()
    bwd = lambda q: lib.gs_grouped_linear_bwd(ct.byref(q), *[None] * 10, 0, None)  # noqa: E731
    assert bwd(prm()) == L.GS_OK            # nothing wanted
    assert bwd(prm(G=0)) == L.GS_ERR_INVALID
    assert lib.gs_grouped_linear_bwd_workspace_size(ct.byref(prm(G=0))) == 0
    # 16-bit gradients of shared rows are added up in fp32 scratch; what is too small is refused
    q = prm(dtype=1, ids=1)
    need = lib.gs_grouped_linear_bwd_workspace_size(ct.byref(q))
    assert need >= 4 * 6 * 4
    one = ct.c_void_p(256)                  # never followed: refused first
    assert lib.gs_grouped_linear_bwd(ct.byref(q), one, one, one, one, one, one, one, one, one,
                                     one, need - 1, None) == L.GS_ERR_WORKSPACE


def test_param_layouts(gs, tmp_path):
    from gsplat_core import _lib as L
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    pairs = {"gs_dropout_params": L.DropoutParams, "gs_grouped_params": L.GroupedParams}
    body = "".join(f'printf("%zu ", sizeof({c}));' + "".join(
        f'printf("%zu ", offsetof({c}, {f}));' for f, _ in t._fields_) for c, t in pairs.items())
    (tmp_path / "l.c").write_text('#include <stddef.h>\n#include <stdio.h>\n#include "gsplat_b200.h"\n'
                                  "int main(void) {" + body + "return 0;}\n")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o",
                    str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True,
                                          text=True).stdout.split()]
    assert got == [v for t in pairs.values()
                   for v in [ct.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]]
