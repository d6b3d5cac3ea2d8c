"""Products of ragged groups of rows with one weight matrix per group: a
learned layer per camera (appearance, exposure, hidden features) over the
packed rows, which are sorted by camera.  No counterpart in the reference.

    off = group_offsets(packed["image_ids"], I)
    inputs = {"x": features, "weights": W, "biases": b, "offsets": off,
              "row_ids": packed["gaussian_ids"]}
    colors = grouped_linear_forward(inputs, activation="sigmoid")   # [nnz, M]
    ...                                                # rasterize, backward
    g = grouped_linear_backward(inputs, colors, v_colors, activation="sigmoid")

With ``row_ids`` the rows of x are gathered as they are read, so that no
[nnz, K] copy of the Gaussians' features is made; the backward adds the rows
of one Gaussian up.  Everything runs on the current stream and nothing waits
for the device, so the calls can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as ct

import torch

from . import _lib
from ._lib import GroupedParams, on_device_of
from ._lib import check as check_status

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_WANTED = {"v_x": 1, "v_weights": 2, "v_biases": 4}
_GROUPS_MOST = 2 ** 31 - 2
_ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2}


def _ptr(t):
    return None if t is None else t.data_ptr()


def group_offsets(ids, groups):
    """[groups + 1] int32 bounds of the rows of each id in the sorted int32
    ``ids`` (packed["image_ids"], or any rows sorted by group): group g's
    rows are off[g] .. off[g + 1] - 1."""
    if ids.dim() != 1 or ids.dtype != torch.int32:
        raise RuntimeError("group_offsets: ids must be a 1-D int32 tensor.")
    if int(groups) < 0:
        raise RuntimeError("group_offsets: negative number of groups.")
    if int(groups) > _GROUPS_MOST:
        raise RuntimeError("group_offsets: 2^31 - 1 groups or more.")
    if not ids.is_cuda:
        raise RuntimeError("group_offsets: ids must be a CUDA tensor (there is no CPU fallback).")
    ids = ids.contiguous()
    off = torch.empty((int(groups) + 1,), dtype=torch.int32, device=ids.device)
    lib = _lib.load()
    check_status(on_device_of(ids, lambda stream: lib.gs_group_offsets(
        ids.numel(), _ptr(ids), int(groups), _ptr(off), stream)), "group_offsets")
    return off


def _validated(inputs, activation):
    """The inputs, contiguous, and the call's params; shapes and types are
    checked before the device is touched."""
    for k in ("x", "weights", "offsets"):
        if inputs.get(k) is None:
            raise RuntimeError(f"grouped_linear missing input: {k}")
    x, w, off = inputs["x"], inputs["weights"], inputs["offsets"]
    b, ids = inputs.get("biases"), inputs.get("row_ids")
    dtype = x.dtype
    if x.dim() != 2 or dtype not in _DTYPES:
        raise RuntimeError("grouped_linear: x must have shape [rows, K] and type float32, "
                           "bfloat16 or float16.")
    n, K = x.shape
    if w.dim() != 3 or w.shape[2] != K or w.dtype != dtype:
        raise RuntimeError("grouped_linear: weights must have shape [G, M, K] and x's type.")
    G, M, _ = w.shape
    if min(G, M, K) < 1 or max(M, K) > 16384:
        raise RuntimeError("grouped_linear: G, M and K must be at least 1, M and K at most 16384.")
    if G > _GROUPS_MOST:
        raise RuntimeError("grouped_linear: 2^31 - 1 groups or more.")
    if off.shape != (G + 1,) or off.dtype != torch.int32:
        raise RuntimeError("grouped_linear: offsets must have shape [G + 1] and type int32.")
    if b is not None and (b.shape != (G, M) or b.dtype != dtype):
        raise RuntimeError("grouped_linear: biases must have shape [G, M] and x's type.")
    if ids is not None and (ids.dim() != 1 or ids.dtype != torch.int32):
        raise RuntimeError("grouped_linear: row_ids must have shape [rows] and type int32.")
    if activation not in _ACTIVATIONS:
        raise RuntimeError("grouped_linear: activation must be none, relu or sigmoid.")
    at = x.get_device()  # -1: the host
    if (w.get_device() != at or off.get_device() != at or (b is not None and b.get_device() != at)
            or (ids is not None and ids.get_device() != at)):
        raise RuntimeError("grouped_linear: inputs on different devices.")
    R = n if ids is None else ids.shape[0]
    if max(R, n) >= 2 ** 31 - 4096:
        raise RuntimeError("grouped_linear: 2^31 - 4096 rows or more.")
    p = GroupedParams(R, n, G, K, M, _DTYPES[dtype], _ACTIVATIONS[activation], int(ids is not None))
    return p, (x.contiguous(), w.contiguous(), off.contiguous(),
               None if b is None else b.contiguous(), None if ids is None else ids.contiguous())


def _on_cuda(t):
    if not t.is_cuda:
        raise RuntimeError("grouped_linear: inputs must be CUDA tensors (there is no CPU "
                           "fallback).")


def grouped_linear_forward(inputs, activation="none"):
    """y [R, M] = activation(x[id(r)] W[g]^T + b[g]) for the rows r of group
    g, offsets[g] <= r < offsets[g + 1].

    inputs: x [R, K] -- or [N, K] with row_ids [R] int32, which name the row
    of x that each row reads -- weights [G, M, K], offsets [G + 1] int32
    ascending, biases [G, M] (optional).  x, weights and biases share one
    type, float32, bfloat16 or float16; sums are in float32 and y is rounded
    once.  activation: none, relu or sigmoid.  Rows outside every group are
    zeros; a row id outside [0, N) reads zeros."""
    p, (x, w, off, b, ids) = _validated(inputs, activation)
    _on_cuda(x)
    y = x.new_empty((p.rows, p.out_features))
    lib = _lib.load()
    check_status(on_device_of(x, lambda stream: lib.gs_grouped_linear_fwd(
        ct.byref(p), _ptr(x), _ptr(ids), _ptr(off), _ptr(w), _ptr(b), _ptr(y), stream)),
        "grouped_linear_forward")
    return y


def grouped_linear_backward(inputs, y, v_y, activation="none",
                            wanted=("v_x", "v_weights", "v_biases")):
    """Gradients {"v_x" like x, "v_weights" [G, M, K], "v_biases" [G, M]} --
    those named in ``wanted``, v_biases only where inputs has biases -- from
    the forward's output ``y`` (not read for activation "none") and its
    gradient ``v_y`` [R, M].  With row_ids, v_x sums the rows that read one
    row of x with fp32 atomics (their order is not fixed); the other sums
    have a fixed order."""
    p, (x, w, off, b, ids) = _validated(inputs, activation)
    R, M = p.rows, p.out_features
    if activation != "none" and (y is None or y.shape != (R, M) or y.dtype != x.dtype):
        raise RuntimeError("grouped_linear: y must have shape [rows, M] and x's type.")
    if v_y is None or v_y.shape != (R, M) or v_y.dtype != x.dtype:
        raise RuntimeError("grouped_linear: v_y must have shape [rows, M] and x's type.")
    if set(wanted) - {"v_x", "v_weights", "v_biases"}:
        raise RuntimeError("grouped_linear: wanted names v_x, v_weights and v_biases.")
    y = y.contiguous() if activation != "none" else None
    v_y = v_y.contiguous()
    if v_y.device != x.device or (y is not None and y.device != x.device):
        raise RuntimeError("grouped_linear: inputs on different devices.")
    _on_cuda(x)
    out = {}
    if "v_x" in wanted:
        out["v_x"] = torch.empty_like(x)
    if "v_weights" in wanted:
        out["v_weights"] = torch.empty_like(w)
    if "v_biases" in wanted and b is not None:
        out["v_biases"] = torch.empty_like(b)
    if not out:
        return out
    p.wanted = sum(_WANTED[k] for k in out)  # scratch for these alone
    lib = _lib.load()

    def call(stream):
        need = lib.gs_grouped_linear_bwd_workspace_size(ct.byref(p))
        ws = off.new_empty((need + 3) // 4)
        return lib.gs_grouped_linear_bwd(
            ct.byref(p), _ptr(x), _ptr(ids), _ptr(off), _ptr(w), _ptr(y), _ptr(v_y),
            _ptr(out.get("v_x")), _ptr(out.get("v_weights")), _ptr(out.get("v_biases")),
            _ptr(ws), need, stream)

    check_status(on_device_of(x, call), "grouped_linear_backward")
    return out


def check(device=None):
    """Waits for the current stream of ``device`` (None: the current one) and
    raises if a bounded on-device wait of a grouped_linear call on that device
    gave up since the last check: what that call gave is void.  Until then the
    calls behind it on the device raise, too (the backward of a step, or the
    next step, without waiting for anything); after it they run again."""
    lib = _lib.load()
    with torch.cuda.device(device):
        check_status(lib.gs_grouped_linear_check(torch.cuda.current_stream().cuda_stream),
                     "grouped_linear")
