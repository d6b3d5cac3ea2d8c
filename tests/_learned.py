"""64-bit forms of the dropout and the grouped products, and the rounding
that the kernels may add, shared by their tests."""
from __future__ import annotations

import numpy as np
import torch

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def philox(n, seed, step, rounds=7):
    """Words 0..n-1 of Philox4x32 (Salmon et al. 2011) under key seed, with
    the counters (i / 4, step)."""
    u = np.uint64
    block = np.arange((n + 3) // 4, dtype=u)
    low = u(0xFFFFFFFF)
    c = [block & low, block >> u(32), np.full_like(block, step & 0xFFFFFFFF),
         np.full_like(block, (step >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(rounds):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def keep_mask(shape, p, seed, step, rows):
    n = shape[0] if rows else int(np.prod(shape))
    keep = philox(n, seed, step) >= np.uint64(round(p * 2.0 ** 32))
    if rows:
        return np.broadcast_to(keep.reshape((-1,) + (1,) * (len(shape) - 1)), shape)
    return keep.reshape(shape)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the type's subnormals."""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134,
            torch.float16: 2.0 ** -25}[dtype]


def linear(x, w, off, b=None, ids=None, act="none", v_y=None, y=None):
    """The grouped product (and, with v_y and the forward's y, its reverse
    mode) in 64 bits on the host: {name: (value, magnitude)}; magnitude is
    the sum of the absolute values of what is added up."""
    d = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, w, b = d(x), d(w), d(b)
    G, M, K = w.shape
    edges = [int(v) for v in off.tolist()]
    R = x.shape[0] if ids is None else ids.numel()
    at = torch.arange(R) if ids is None else ids.cpu().long()
    ok = (at >= 0) & (at < x.shape[0])
    rows = x.new_zeros((R, K))
    rows[ok] = x[at[ok]]
    if v_y is None:
        z, mag, live = x.new_zeros((R, M)), x.new_zeros((R, M)), torch.zeros(R, dtype=torch.bool)
        for g in range(G):
            s = slice(edges[g], edges[g + 1])
            z[s] = rows[s] @ w[g].T + (b[g] if b is not None else 0)
            mag[s] = rows[s].abs() @ w[g].abs().T + (b[g].abs() if b is not None else 0)
            live[s] = True
        a = z.clamp(min=0) if act == "relu" else torch.sigmoid(z) if act == "sigmoid" else z
        return {"y": (torch.where(live[:, None], a, torch.zeros_like(a)), mag)}
    v, y = d(v_y), d(y)
    if act == "relu":
        v = torch.where(y > 0, v, torch.zeros_like(v))
    elif act == "sigmoid":
        v = v * y * (1 - y)
    out = {"v_x": [torch.zeros_like(x), torch.zeros_like(x)],
           "v_weights": [torch.zeros_like(w), torch.zeros_like(w)],
           "v_biases": [w.new_zeros((G, M)), w.new_zeros((G, M))]}
    for i, f in enumerate((lambda t: t, torch.abs)):
        for g in range(G):
            s = slice(edges[g], edges[g + 1])
            o = ok[s]
            out["v_x"][i].index_add_(0, at[s][o], f(v[s][o]) @ f(w[g]))
            out["v_weights"][i][g] = f(v[s]).T @ f(rows[s])
            out["v_biases"][i][g] = f(v[s]).sum(0)
    return {k: tuple(t) for k, t in out.items()}


def assert_sums(got, want, mag, terms, dtype, extra=0.0, what=""):
    """|got - want| within what fp32 sums of ``terms`` products may be off.

    A product of two fp32 values taken apart into two 11-bit parts each is
    off by at most 3 2^-22 = 12 2^-24 of itself (two remainders of 2^-22 and
    the product of the low parts), a 16-bit one is exact.  Each of the
    ``terms`` additions and the final ones (accumulators joined, bias) loses
    at most one unit in the last place, 2^-23, of a partial sum that the
    magnitude bounds: 2 (terms + 10) 2^-24 with ten for the joining.  Then
    one rounding to the type.  ``extra``: absolute, from before the sum."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {got.shape} != {want.shape}"
    allow = (2 * (terms + 10) + 12) * 2.0 ** -24 * mag + half_step(dtype) * want.abs()
    allow = allow * (1 + 2.0 ** -7) + tiny(dtype) + extra
    bad = ~((got - want).abs() <= allow)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance, first at "
        f"{bad.nonzero()[0].tolist()}: {got[bad][0]} vs {want[bad][0]} (allowed {allow[bad][0]:.3g})")
