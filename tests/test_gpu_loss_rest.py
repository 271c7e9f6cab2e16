"""linear_cross_entropy's gradients on the GPU where the rounding of the target's entry decides (krsi_even_loss)."""
import pytest
import torch

import krsi_even_loss as C
import krsi_oracle as O
import linear_cross_entropy as L
from krsi_testutil import log

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])


def _verify(dt, ignored, unweighted):
    x, w, targets, dout, rank = C.inputs(dt, ignored, unweighted)
    r = O.linear_cross_entropy_64(x, w, targets, dout, reduction="none")
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    dx, dw = torch.autograd.grad(L.linear_cross_entropy(*leaves, targets, reduction="none"), leaves, dout)
    bx, bw = C.bounds(r, x.detach(), w.detach(), targets, rank)
    for name, got, ref, bound in (("dx", dx, r["dx"], bx), ("dw", dw, r["dw"], bw)):
        off = (got.double() - ref).abs()
        log(f"{name}: worst {(off / bound.clamp_min(1e-300)).max().item():.3f} of its bound")
        assert got.shape == ref.shape and bool((off <= bound).all()), name


@DTYPES
@pytest.mark.parametrize("ignored", [0, 100, 40000 - C.V], ids=["all count", "some ignored", "two pieces"])
def test_rounding_of_the_target_comes_back(dt, ignored):
    log(f"linear_cross_entropy, equal logits, {C.V} targets, {ignored} ignored {dt}")
    _verify(dt, ignored, 0)
