"""Cases for the grouped products and the counter-based dropout.

Both serve a splat model whose colours are learned per camera.  The packed
rows of a batch of cameras are sorted by camera, a ragged number for each;
``grouped_linear`` multiplies every row's Gaussian's features by its camera's
weights, and ``dropout`` drops Gaussians (whole rows) or hidden features with
a mask that is a function of (seed, step, index) and is never stored.

``own`` false: the operators in elementary torch operations, in 32 bits.
``own`` true: the calls that a user makes of gsplat_core.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "gsplat-mlx_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from gsplat_core import dropout, grouped
    return dropout, grouped


# ------------------------------------------------------------------- cases

def _drop(name, n, width, dtype, rows, p, direction):
    return {"name": name, "op": "dropout", "n": n, "width": width, "dtype": dtype, "rows": rows,
            "p": p, "direction": direction}


def _lin(name, rows, groups, gaussians, k, m, dtype, act, direction, bias=True, skew=1.0):
    """gaussians > 0: the rows gather their features from that many."""
    return {"name": name, "op": "grouped_linear", "rows": rows, "groups": groups,
            "gaussians": gaussians, "k": k, "m": m, "dtype": dtype, "act": act,
            "direction": direction, "bias": bias, "skew": skew}


def listed():
    return [
        # opacities of a 10,000-Gaussian scene, one camera: launch latency
        _drop("drop 10k opacities", 10_000, 1, "fp32", True, 0.1, "fwd"),
        # the gradient of the opacities at 1 M Gaussians
        _drop("drop 1M opacities bwd", 1_000_000, 1, "fp32", True, 0.1, "bwd"),
        # SH degree 3 rows (16 x 3 floats) of 3 M Gaussians, whole Gaussians
        _drop("drop 3M SH rows", 3_000_000, 48, "fp32", True, 0.2, "fwd"),
        # hidden features of the visible rows of one 1297x840 view
        _drop("drop hidden bf16", 316_527, 128, "bf16", False, 0.5, "fwd"),
        # odd width, half precision, the backward
        _drop("drop odd fp16 bwd", 999_983, 37, "fp16", False, 0.25, "bwd"),
        # one small image's rows to colours: launch latency
        _lin("one camera 257 rows", 257, 1, 0, 16, 3, "fp32", "sigmoid", "fwd"),
        # one 1297x840 view of 1 M Gaussians: the visible ones' features to hidden ones
        _lin("view 64-64 gather", 316_527, 1, 1_000_000, 64, 64, "fp32", "relu", "fwd"),
        # 32 cameras, 3 M Gaussians: features to colours
        _lin("32 views 32-3 gather", 4_000_000, 32, 3_000_000, 32, 3, "fp32", "sigmoid", "fwd"),
        # its training pass at 64 features
        _lin("8 views 64-64 gather bwd", 1_200_000, 8, 1_000_000, 64, 64, "fp32", "relu", "bwd"),
        # hidden layer in 16 bits, 32 cameras
        _lin("32 views 128-128 bf16", 2_000_000, 32, 0, 128, 128, "bf16", "relu", "fwd"),
        _lin("32 views 128-128 bf16 bwd", 2_000_000, 32, 0, 128, 128, "bf16", "relu", "bwd"),
        # odd sizes, groups of very unequal sizes and empty ones
        _lin("odd 77-45 fp16 bwd", 200_003, 19, 0, 77, 45, "fp16", "sigmoid", "bwd", skew=3.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _largest(op):
    return max(_cost(c) for c in listed() if c["op"] == op)


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 50.0


def draw(rng):
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    direction = rng.choice(["fwd", "bwd"])
    if rng.random() < 0.4:
        rows = rng.random() < 0.5
        width = rng.choice([1, 3, 4, 48]) if rows and rng.random() < 0.6 else _log_int(rng, 1, 256)
        case = _drop("", _log_int(rng, 100, 4_000_000), width, dtype, rows,
                     round(rng.uniform(0.02, 0.7), 3), direction)
    else:
        rows = _log_int(rng, 1, 4_000_000)
        gaussians = 0 if rng.random() < 0.5 else max(1, int(rows * rng.uniform(0.2, 3.0)))
        wide = [3, 16, 32, 48, 64, 128]
        k = rng.choice(wide) if rng.random() < 0.5 else _log_int(rng, 1, 200)
        m = rng.choice(wide) if rng.random() < 0.5 else _log_int(rng, 1, 200)
        case = _lin("", rows, _log_int(rng, 1, 64), gaussians, k, m, dtype,
                    rng.choice(["none", "relu", "sigmoid"]), direction, rng.random() < 0.8,
                    round(rng.uniform(0.2, 2.0), 2))
    del case["name"]
    size = "n" if case["op"] == "dropout" else "rows"
    over = _cost(case) / _largest(case["op"])
    if over > 1.0:  # as many rows as the largest listed case pays for
        case[size] = max(1, int(case[size] / over * 0.98))
        if case.get("gaussians"):
            case["gaussians"] = max(1, int(case["gaussians"] / over * 0.98))
    return case


def work(case):
    es = _BYTES[case["dtype"]]
    if case["op"] == "dropout":
        # a dropped row is written but need not be read
        return {"bytes": case["n"] * case["width"] * es * (2.0 - (case["p"] if case["rows"] else 0)),
                "flops": float(case["n"] * case["width"])}
    r, g, k, m = case["rows"], case["groups"], case["k"], case["m"]
    n = case["gaussians"]
    weights = g * (m * k + (m if case["bias"] else 0)) * es
    x = (min(r, n) if n else r) * k * es + (4 * r if n else 0) + 4 * (g + 1)
    y = r * m * es
    if case["direction"] == "fwd":
        return {"bytes": float(x + weights + y), "flops": 2.0 * r * k * m}
    read_y = 0 if case["act"] == "none" else y
    return {"bytes": float(x + 2 * weights + y + read_y + (n or r) * k * es),
            "flops": 4.0 * r * k * m}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _group_sizes(case, seed):
    """Ragged sizes: skew 0 is even, larger is more unequal; of 8 groups or
    more some are empty (a camera that sees nothing)."""
    r, g = case["rows"], case["groups"]
    rng = np.random.default_rng(int(seed))
    share = np.exp(case["skew"] * rng.uniform(-0.6, 0.6, size=g))
    if g >= 8:
        share[rng.integers(0, g, size=g // 8)] = 0.0
    edge = np.floor(np.cumsum(share) / share.sum() * r + 0.5).astype(np.int64)
    edge[-1] = r
    return np.diff(np.minimum(edge, r), prepend=0)


def prepare(case, seed):
    g = _gen(seed)
    dt = _DTYPES[case["dtype"]]
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "dropout":
        x = torch.randn((case["n"], case["width"]), generator=g, device="cuda", dtype=dt)
        return {"case": case, "x": x, "seed": 0x9E3779B97F4A7C15 ^ int(seed), "step": 1000 + int(seed) % 977}
    r, k, m, n = case["rows"], case["k"], case["m"], case["gaussians"]
    sizes = _group_sizes(case, seed)
    counts = torch.from_numpy(sizes).cuda()
    offsets = torch.zeros(case["groups"] + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = counts.cumsum(0)
    group = torch.repeat_interleave(torch.arange(case["groups"], device="cuda"), counts,
                                    output_size=r)
    s = {"case": case, "offsets": offsets.to(torch.int32), "longest": int(sizes.max()),
         "x": rand(n or r, k).to(dt), "weights": (rand(case["groups"], m, k) / math.sqrt(k)).to(dt)}
    if n:  # each camera sees some of the Gaussians, in their order
        at = (torch.arange(r, device="cuda") - offsets[group]).double()
        at += torch.rand(r, generator=g, device="cuda", dtype=torch.float64)
        s["row_ids"] = (at * (n / counts[group].double())).long().clamp_(max=n - 1).to(torch.int32)
        del at
    if case["bias"]:
        s["biases"] = (0.1 * rand(case["groups"], m)).to(dt)
    if case["direction"] == "bwd":
        # what the forward gave, and what the rasterizer's backward gives
        s["y"] = _linear_forward(s).to(dt)
        s["v_y"] = rand(r, m).to(dt)
    return s


# -------------------------------------------------------------- plain forms

_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
_LOW = 0xFFFFFFFF


def _round(state, key):
    """One round of Philox4x32 (Salmon et al. 2011) on int64 tensors that
    hold 32-bit words; a product's bits 32 to 63 survive its sign."""
    c0, c1, c2, c3 = state
    k0, k1 = key
    p0, p1 = c0 * _M0, c2 * _M1
    return (((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW)


def _words(n, seed, step, device):
    """The first n 32-bit words of Philox4x32-7: word i is output i % 4 of
    the counter (i / 4, step) under the key seed."""
    block = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    zero = torch.zeros_like(block)
    keys = [((seed + r * _W0) & _LOW, ((seed >> 32) + r * _W1) & _LOW) for r in range(7)]
    start = (block & _LOW, block >> 32, zero + (step & _LOW), zero + (step >> 32))
    return torch.stack(functools.reduce(_round, keys, start), dim=1).reshape(-1)[:n]


def _dropout(s):
    x, case = s["x"], s["case"]
    n = case["n"] if case["rows"] else x.numel()
    keep = _words(n, s["seed"], s["step"], x.device) >= int(round(case["p"] * 2.0 ** 32))
    keep = keep.view(-1, 1) if case["rows"] else keep.view(x.shape)
    return torch.where(keep, x.float() * (1.0 / (1.0 - case["p"])), 0.0).to(x.dtype)


def _padded(s):
    """Each row's group and its place in a [groups, longest] layout."""
    off = s["offsets"].long()
    row = torch.arange(s["case"]["rows"], device=off.device)
    group = torch.searchsorted(off[1:], row, right=True)
    return group, row - off[group]


def _to_groups(s, v, at):
    pad = v.new_zeros((s["case"]["groups"], s["longest"], v.shape[1]))
    pad[at] = v
    return pad


def _rows_of_x(s):
    x = s["x"].float()
    return x[s["row_ids"].long()] if "row_ids" in s else x


def _linear_forward(s):
    at = _padded(s)
    z = torch.bmm(_to_groups(s, _rows_of_x(s), at), s["weights"].float().transpose(1, 2))[at]
    if "biases" in s:
        z = z + s["biases"].float()[at[0]]
    act = s["case"]["act"]
    return torch.clamp(z, min=0.0) if act == "relu" else torch.sigmoid(z) if act == "sigmoid" else z


def _rows_product(a, b):
    """Sum over each group's rows of a[row]^T b[row], a run of 4096 rows at a
    time: one long fp32 sum would lose what the 4096-row ones keep."""
    n = a.shape[1]
    a, b = (torch.nn.functional.pad(t, (0, 0, 0, -n % 4096)).reshape(-1, 4096, t.shape[2])
            for t in (a, b))
    return torch.bmm(a.transpose(1, 2), b).view(-1, (n + 4095) // 4096, a.shape[2], b.shape[2]).sum(1)


def _linear_backward(s):
    at = _padded(s)
    y, v = s["y"].float(), s["v_y"].float()
    act = s["case"]["act"]
    v = v * (y > 0) if act == "relu" else v * y * (1.0 - y) if act == "sigmoid" else v
    v = _to_groups(s, v, at)
    v_rows = torch.bmm(v, s["weights"].float())[at]
    if "row_ids" in s:
        v_rows = torch.zeros_like(s["x"], dtype=torch.float32).index_add_(0, s["row_ids"].long(), v_rows)
    out = {"v_x": v_rows.to(s["x"].dtype),
           "v_weights": _rows_product(v, _to_groups(s, _rows_of_x(s), at)).to(s["x"].dtype)}
    if "biases" in s:
        out["v_biases"] = v.sum(1).to(s["x"].dtype)
    return out


# --------------------------------------------------------------------- run

def run(s):
    case = s["case"]
    if own:
        dropout, grouped = _package()
        if case["op"] == "dropout":
            call = dropout.dropout_forward if case["direction"] == "fwd" else dropout.dropout_backward
            return call(s["x"], case["p"], s["seed"], step=s["step"], rows=case["rows"])
        inputs = {k: s[k] for k in ("x", "weights", "offsets", "biases", "row_ids") if k in s}
        if case["direction"] == "fwd":
            return grouped.grouped_linear_forward(inputs, activation=case["act"])
        return grouped.grouped_linear_backward(inputs, s["y"], s["v_y"], activation=case["act"])
    if case["op"] == "dropout":
        return _dropout(s)
    if case["direction"] == "fwd":
        return _linear_forward(s).to(s["x"].dtype)
    return _linear_backward(s)


# ------------------------------------------------------------------- exact

def _exact_words(n, seed, step):
    """The same words with numpy's unsigned 64-bit integers."""
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    mask, shift = np.uint64(_LOW), np.uint64(32)
    c = [block & mask, block >> shift, np.full_like(block, step & _LOW),
         np.full_like(block, step >> 32)]
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(7):
        a, b = c[0] * np.uint64(_M0), c[2] * np.uint64(_M1)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & mask,
             (a >> shift) ^ c[3] ^ np.uint64(k1), a & mask]
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    return np.stack(c, axis=1).reshape(-1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        n = case["n"] if case["rows"] else case["n"] * case["width"]
        keep = _exact_words(n, s["seed"], s["step"]) >= np.uint64(round(case["p"] * 2.0 ** 32))
        keep = torch.from_numpy(keep).cuda().view(case["n"], -1)
        x = s["x"].double()
        return torch.where(keep, x / (1.0 - case["p"]), torch.zeros_like(x))
    edges = s["offsets"].tolist()
    w = s["weights"].double()
    xs = s["x"]
    ids = s["row_ids"].long() if "row_ids" in s else None
    spans = [(g, a, b) for g, (a, b) in enumerate(zip(edges, edges[1:])) if b > a]
    if case["direction"] == "fwd":
        out = torch.empty((case["rows"], case["m"]), dtype=torch.float64, device="cuda")
        for g, a, b in spans:
            z = (xs[ids[a:b]] if ids is not None else xs[a:b]).double() @ w[g].T
            if case["bias"]:
                z += s["biases"][g].double()
            out[a:b] = z.relu() if case["act"] == "relu" else (
                1.0 / (1.0 + torch.exp(-z)) if case["act"] == "sigmoid" else z)
        return out
    v_x = torch.zeros(xs.shape, dtype=torch.float64, device="cuda")
    v_w = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    v_b = torch.zeros(w.shape[:2], dtype=torch.float64, device="cuda")
    for g, a, b in spans:
        y, v = s["y"][a:b].double(), s["v_y"][a:b].double()
        if case["act"] == "relu":
            v = torch.where(y > 0, v, torch.zeros_like(v))
        elif case["act"] == "sigmoid":
            v = v * (y - y * y)
        x = (xs[ids[a:b]] if ids is not None else xs[a:b]).double()
        if ids is not None:
            v_x.index_add_(0, ids[a:b], v @ w[g])
        else:
            v_x[a:b] = v @ w[g]
        v_w[g], v_b[g] = v.T @ x, v.sum(0)
    out = {"v_x": v_x, "v_weights": v_w}
    if case["bias"]:
        out["v_biases"] = v_b
    return out
