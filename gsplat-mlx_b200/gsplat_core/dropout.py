"""Dropout with a mask from a counter-based generator that is never stored:
whole Gaussians of a training step (their opacities, features or SH rows), or
single hidden features.  No counterpart in the reference.

    opac = dropout_forward(opacities, 0.1, seed, step=it, rows=True)
    ...                                          # render, backward
    v_opacities = dropout_backward(v_opac, 0.1, seed, step=it, rows=True)

The mask is a function of (seed, step, index): the backward draws it again,
every rank of a camera-sharded step draws the same one, and all tensors of
one Gaussian (rows=True) are dropped together whatever their width or type.
Kept values are scaled by 1 / (1 - p).  The generator is Philox4x32-7; see
``gs_dropout`` in include/gsplat_b200.h for the exact rule.
"""
from __future__ import annotations

import ctypes as ct

import torch

from . import _lib
from ._lib import DropoutParams, check, on_device_of

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_U64 = (1 << 64) - 1


def dropout_forward(x, p, seed, step=0, rows=False, out=None):
    """x with each value -- or, with ``rows``, each x[i] as a whole -- dropped
    with probability ``p`` in [0, 1] and the others divided by 1 - p (fp32,
    bf16 or fp16; p = 1 gives zeros).  A dropped place is an exact zero
    whatever x holds there.  ``seed`` is an integer (mod 2^64); ``step`` an
    integer, or an int64 CUDA tensor of one element that the kernel reads
    when it runs (a captured graph then draws another mask at each replay).
    ``out`` may be a contiguous tensor like x, or x itself."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise RuntimeError("dropout: x must be a float32, bfloat16 or float16 tensor.")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout: p must be in [0, 1], got {p}.")
    if rows and x.dim() == 0:
        raise RuntimeError("dropout: rows=True needs a tensor with at least one dimension.")
    n = x.shape[0] if x.dim() else 1
    width = x.numel() // n if n else 0
    if rows and width >= 1 << 24:
        raise RuntimeError("dropout: rows=True takes rows of fewer than 2^24 values.")
    step_dev = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != x.device:
            raise RuntimeError("dropout: a step tensor must be one int64 on x's device.")
        step, step_dev = 0, step
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype
                            or out.device != x.device or not out.is_contiguous()):
        raise RuntimeError("dropout: out must be contiguous, with x's shape, type and device.")
    if not x.is_cuda:
        raise RuntimeError("dropout: x must be a CUDA tensor (there is no CPU fallback).")
    x = x.contiguous()
    y = torch.empty_like(x) if out is None else out
    size = x.numel() * x.element_size()
    if out is not None and 0 < abs(y.data_ptr() - x.data_ptr()) < size:
        raise RuntimeError("dropout: out overlaps x without being x.")
    prm = DropoutParams(n, width, int(seed) & _U64, int(step) & _U64, p, _DTYPES[x.dtype],
                        int(bool(rows)))
    lib = _lib.load()
    check(on_device_of(x, lambda stream: lib.gs_dropout(
        ct.byref(prm), x.data_ptr(), None if step_dev is None else step_dev.data_ptr(),
        y.data_ptr(), stream)), "dropout")
    return y


def dropout_backward(v_y, p, seed, step=0, rows=False, out=None):
    """The gradient of x from that of y: the forward's map (same p, seed,
    step and rows) on ``v_y``, its mask drawn again."""
    return dropout_forward(v_y, p, seed, step, rows, out)
