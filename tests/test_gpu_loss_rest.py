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


@DTYPES
def test_rows_without_weight_take_nothing_from_the_target(dt):
    """Rows of weight 0 behind the ones that count: the rest of the rows that count comes back all the same."""
    log(f"linear_cross_entropy, equal logits, rows of weight 0 last {dt}")
    _verify(dt, 100, C.V // 2)


@DTYPES
def test_rows_without_weight_have_no_gradient(dt):
    """dx of a row of weight 0 is 0 whatever the row holds, in one part and in parts that are added."""
    for rows, K, V in ((50, 128, 300), (40, 64, 9000)):
        log(f"linear_cross_entropy, NaN and infinities in rows of weight 0, x[{rows},{K}] w[{V},{K}] {dt}")
        g = torch.Generator().manual_seed(4)
        x = torch.randn(rows, K, generator=g).to(dt).cuda()
        w = (torch.randn(V, K, generator=g) / K ** 0.5).to(dt).cuda()
        targets = torch.randint(0, V, (rows,), generator=g).cuda()
        dout = torch.randn(rows, generator=g).cuda()
        dout[3:6] = 0.0
        (ref,) = torch.autograd.grad(L.linear_cross_entropy(x.requires_grad_(True), w, targets, reduction="none"), x, dout)
        odd = x.detach().clone()
        odd[3, 5], odd[4, 6], odd[5] = float("nan"), float("inf"), float("-inf")
        odd.requires_grad_(True)
        (dx,) = torch.autograd.grad(L.linear_cross_entropy(odd, w, targets, reduction="none"), odd, dout)
        assert not dx[3:6].any() and torch.equal(dx, ref)
