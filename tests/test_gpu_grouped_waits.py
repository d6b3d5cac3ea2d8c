"""Waits inside the grouped_linear kernels that run out: of copies that never
count as arrived, or a tensor-core tile that never counts as done.  The call
says so and returns, and the device goes on."""
from __future__ import annotations

import ctypes as ct

import pytest
import torch

pytestmark = pytest.mark.gpu

# N: rows of x where they are gathered (0: not), `off`: values that x starts past
# 16 bytes.  Forward: how rows arrive (TMA; gathered; copied); backward: each
# kernel, and each way of its operands
FORWARD = [("fp32", 64, 64, 0, 0, "relu"), ("bf16", 128, 128, 0, 0, "none"),
           ("fp32", 64, 64, 500, 0, "none"), ("fp16", 64, 32, 500, 0, "sigmoid"),
           ("fp32", 65, 33, 0, 0, "none"), ("fp16", 77, 45, 300, 0, "relu"),
           ("fp32", 1000, 40, 0, 0, "none"), ("bf16", 64, 64, 0, 1, "none")]
BACKWARD = [("fp32", 64, 64, 0, 0, "none"), ("fp32", 64, 64, 500, 0, "relu"),
            ("fp32", 64, 100, 500, 0, "sigmoid"), ("fp32", 65, 33, 0, 0, "relu"),
            ("fp32", 65, 64, 300, 0, "none"), ("bf16", 128, 128, 0, 0, "relu"),
            ("fp16", 64, 64, 0, 0, "sigmoid"), ("bf16", 64, 64, 500, 0, "relu"),
            ("fp16", 77, 45, 0, 0, "sigmoid"), ("bf16", 200, 136, 0, 0, "none"),
            ("fp16", 201, 140, 300, 0, "sigmoid"), ("bf16", 64, 64, 0, 1, "none")]
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
ACTS = {"none": 0, "relu": 1, "sigmoid": 2}


def P(t):
    return None if t is None else ct.c_void_p(t.data_ptr())


class Call:
    """The C entries on one problem."""

    def __init__(self, gs, dtype, K, M, N, off, act, R=60_000):
        from gsplat_core import _lib
        self.L, self.lib = _lib, gs.load()
        dt, g = TYPES[dtype], torch.Generator(device="cuda").manual_seed(1)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)  # noqa: E731
        n = N or R
        buf = torch.zeros(n * K + off, dtype=dt, device="cuda")
        self.x = buf[off:].view(n, K)
        self.x.copy_(rand(n, K))
        self.w, self.b = rand(3, M, K), rand(3, M)
        self.off = torch.tensor([0, 700, 700, R], dtype=torch.int32, device="cuda")
        self.ids = (torch.randint(0, N, (R,), generator=g, device="cuda", dtype=torch.int32)
                    if N else None)
        self.y, self.v = rand(R, M).sigmoid(), rand(R, M)
        self.sizes = (R, n, 3, K, M, list(TYPES).index(dtype), ACTS[act], int(bool(N)))

    def params(self, selftest, status):
        return self.L.GroupedParams(*self.sizes, selftest, 0, None if status is None else status.data_ptr())

    def forward(self, selftest=0, status=None):
        y, p = torch.empty_like(self.y), self.params(selftest, status)
        rc = self.lib.gs_grouped_linear_fwd(ct.byref(p), P(self.x), P(self.ids), P(self.off), P(self.w),
                                            P(self.b), P(y), None)
        return rc, [y]

    def backward(self, selftest=0, status=None):
        p = self.params(selftest, status)
        need = self.lib.gs_grouped_linear_bwd_workspace_size(ct.byref(p))
        ws = torch.empty((need + 3) // 4, dtype=torch.int32, device="cuda")
        out = [torch.zeros_like(t) for t in (self.w, self.b, self.x)]
        rc = self.lib.gs_grouped_linear_bwd(
            ct.byref(p), P(self.x), P(self.ids), P(self.off), P(self.w), P(self.y), P(self.v),
            P(out[2]), P(out[0]), P(out[1]), P(ws), need, None)
        torch.cuda.synchronize()
        return rc, out[:2] if self.ids is not None else out  # the atomic sums have no fixed order


@pytest.mark.parametrize("direction,dtype,K,M,N,off,act",
                         [("forward", *c) for c in FORWARD] + [("backward", *c) for c in BACKWARD])
def test_a_wait_that_gives_up_is_reported(gs, cuda, direction, dtype, K, M, N, off, act):
    """The call's own word is set, and nothing else: the next call gives the
    bits of the one before, and the device's word stays clear."""
    from gsplat_core import grouped
    call = getattr(Call(gs, dtype, K, M, N, off, act), direction)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc, want = call(status=status)
    assert rc == 0 and int(status) == 0
    assert call(selftest=1, status=status)[0] == 0
    torch.cuda.synchronize()
    assert int(status) == 1
    status.zero_()
    torch.cuda.synchronize()
    rc, got = call(status=status)
    torch.cuda.synchronize()
    assert rc == 0 and int(status) == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grouped.check()


def test_calls_behind_one_that_gave_up_raise(gs, cuda):
    """Without a word of its own a call that gave up is reported by the next
    calls on the device, through the functions, autograd and the packed
    colours, until check() has reported it; a call with a word still runs."""
    from gsplat_core import autograd as A, grouped, packed
    c = Call(gs, "fp32", 64, 64, 0, 0, "none")
    inputs = {"x": c.x, "weights": c.w, "offsets": c.off, "biases": c.b}
    want = grouped.grouped_linear_forward(inputs)
    x = c.x.clone().requires_grad_(True)
    y = A.grouped_linear(x, c.w, c.off, c.b)
    torch.cuda.synchronize()
    assert c.forward(selftest=1)[0] == 0
    torch.cuda.synchronize()
    ids = torch.arange(c.x.shape[0], dtype=torch.int32, device="cuda")
    for f in (lambda: grouped.grouped_linear_forward(inputs),
              lambda: grouped.grouped_linear_backward(inputs, None, c.v),
              lambda: torch.autograd.grad(y, x, c.v),
              lambda: packed.camera_colors_forward(c.x, c.w, c.b, {"image_offsets": c.off,
                                                                   "gaussian_ids": ids})):
        with pytest.raises(RuntimeError, match="gave up"):
            f()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc, own = c.forward(status=status)
    torch.cuda.synchronize()
    assert rc == 0 and int(status) == 0 and torch.equal(own[0], want)
    with pytest.raises(RuntimeError, match="gave up"):
        grouped.check()
    grouped.check()
    assert torch.equal(grouped.grouped_linear_forward(inputs), want)


def test_first_call_within_a_capture(gs, cuda):
    """The device's word is set up outside the graph that is being recorded."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from gsplat_core.grouped import check, grouped_linear_forward
c = {"x": torch.ones(300, 32, device="cuda"), "weights": torch.ones(1, 32, 32, device="cuda"),
     "offsets": torch.tensor([0, 300], dtype=torch.int32, device="cuda")}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = grouped_linear_forward(c)
graph.replay()
check()
assert bool((y == 32).all())
print("captured")
"""
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "gsplat-mlx_b200"))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
