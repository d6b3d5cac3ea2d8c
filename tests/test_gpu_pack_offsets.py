"""The packed rows' bounds by image, written by the pass that packs them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _projection(images, N, share, seed=0):
    g = torch.Generator().manual_seed(seed)
    visible = torch.rand(images, N, generator=g) < share
    if images > 2:
        visible[1] = False  # an image that sees nothing
    radii = (visible[..., None] * torch.randint(1, 9, (images, N, 2), generator=g)).to(torch.int32)
    return {"radii": radii.cuda(), "means2d": torch.rand(images, N, 2, generator=g).cuda(),
            "depths": torch.rand(images, N, generator=g).cuda(),
            "conics": torch.rand(images, N, 3, generator=g).cuda()}


@pytest.mark.parametrize("images,N", [(1, 1), (1, 5000), (3, 1), (7, 3), (500, 5), (4, 16), (5, 4096),
                                      (3, 10_007), (2, 65_536), (64, 1000)])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_image_offsets(gs, cuda, images, N, share):
    from gsplat_core.packed import pack_projection
    pr = _projection(images, N, share)
    pk = pack_projection(pr)
    ids = pk["image_ids"].cpu().numpy()
    assert ids.size == int((pr["radii"] > 0).all(-1).sum())
    off = pk["image_offsets"]
    assert off.dtype == torch.int32 and off.shape == (images + 1,)
    assert np.array_equal(off.cpu().numpy(), np.searchsorted(ids, np.arange(images + 1)))


@pytest.mark.parametrize("images,N", [(0, 7), (3, 0), (0, 0)])
def test_no_elements(gs, cuda, images, N):
    from gsplat_core.packed import pack_projection
    pk = pack_projection(_projection(images, N, 0.5))
    assert pk["image_ids"].numel() == 0
    assert pk["image_offsets"].tolist() == [0] * (images + 1)


def test_packing_costs_no_further_call(gs, cuda, monkeypatch):
    """The bounds come with the rows: the library is asked for the scratch's
    size, the count and the rows, and for nothing else."""
    from gsplat_core import grouped, packed
    real, asked = packed._lib.load(), []

    class Lib:
        def __getattr__(self, name):
            asked.append(name)
            return getattr(real, name)

    monkeypatch.setattr(packed._lib, "load", lambda: Lib())
    packed.pack_projection(_projection(3, 1000, 0.5))
    assert grouped._lib is packed._lib and len(asked) == 3, asked
