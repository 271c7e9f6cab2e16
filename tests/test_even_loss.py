"""The inputs and bounds of krsi_even_loss, on the CPU: they take gradients formed as the kernels form them, and none in which
what comes back of the target's rounding is missing, has the wrong sign or goes to the wrong place."""
import pytest
import torch

import krsi_even_loss as C
import krsi_oracle as O


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
def test_bounds_tell_a_missing_or_misplaced_rest(dt):
    x, w, targets, dout, rank = C.inputs(dt, ignored=100, unweighted=500, device="cpu")
    r = O.linear_cross_entropy_64(x, w, targets, dout, reduction="none")
    bx, bw = C.bounds(r, x, w, targets, rank)
    dx, dw = C.emulated(x, w, targets, dout)
    assert C.within(dx, r["dx"], bx) and C.within(dw, r["dw"], bw)
    for fault in ("none", "sign", "another row's", "another entry"):
        dx, dw = C.emulated(x, w, targets, dout, fault)
        assert not C.within(dx, r["dx"], bx) and not C.within(dw, r["dw"], bw), fault
    # Rows of weight 0 that take the place of the row that counts: dw alone.
    _, dw = C.emulated(x, w, targets, dout, "rows without weight")
    assert not C.within(dw, r["dw"], bw)
