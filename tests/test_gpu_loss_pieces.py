"""linear_cross_entropy's backward where the vocabulary is taken in several pieces and the sum of each piece's part of dx is
split, with per-row weights, ignored rows and targets at the pieces' ends, against 64 bits."""
import pytest
import torch

import _hip
import linear_cross_entropy as L
from krsi_testutil import log, seeded
from test_gpu_linear_cross_entropy import _inputs, _verify

pytestmark = pytest.mark.gpu

# Rows, V, the first piece's columns: two pieces of unlike widths; rows that no tile divides.
CASES = [(8192, 40001, 20224), (4099, 70001, 35072)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
@pytest.mark.parametrize("rows,V,width", CASES)
def test_pieces_with_split_sums(rows, V, width, dt):
    K = 64
    log(f"linear_cross_entropy in pieces and parts x[{rows},{K}] w[{V},{K}] {dt}")
    size = _hip.lib().krsi_linear_cross_entropy_bwd_workspace_bytes(rows, K, V)
    assert rows * width * 2 + 2 * rows * K * 4 < size < rows * V * 2  # dl of one piece, and fp32 parts of sums
    x, w, targets = _inputs(rows, K, V, dt)
    targets[:8] = torch.tensor([0, 1, width - 1, width, width + 1, V - 1, V - 2, width - 2])
    targets[9::7] = -100
    targets[200:232:2] = width
    dout = seeded((rows,), 5, dtype=torch.float32)
    dout[300:310] = 0.0
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = L.linear_cross_entropy(*leaves, targets, reduction="none")
    dx, dw = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    _verify(out, dx, dw, x, w, targets, dout, reduction="none", device="cuda")
    assert not dx[targets == -100].any() and not dx[300:310].any()
    again = torch.autograd.grad(out, leaves, dout)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])
