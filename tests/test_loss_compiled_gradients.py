"""linear_cross_entropy under torch.compile: its backward forms the gradients that are asked for, as the eager ones do."""
import pytest
import torch

import _hip
import _ops
import linear_cross_entropy as L
from krsi_testutil import log


@pytest.mark.parametrize("dx,dw", [(True, True), (True, False), (False, True)])
def test_shapes_of_the_gradients(dx, dw):
    """Without a GPU: what the op's shape function says for each choice."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(8, 64, dtype=torch.bfloat16), torch.empty(20, 64, dtype=torch.bfloat16)
        targets, stats, dout = torch.empty(8, dtype=torch.int64), torch.empty(9), torch.empty(())
        got = _ops.linear_cross_entropy_bwd_op(dout, x, w, targets, stats, -100, "mean", dx, dw)
    assert [g.shape for g in got] == [x.shape if dx else (0,), w.shape if dw else (0,)]


@pytest.mark.gpu
@pytest.mark.parametrize("dx,dw", [(True, True), (True, False), (False, True)])
def test_only_the_gradients_asked_for(dx, dw, monkeypatch):
    log(f"linear_cross_entropy compiled, dx {dx}, dw {dw}")
    g = torch.Generator().manual_seed(7)
    x = torch.randn(40, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_(dx)
    w = torch.randn(90, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_(dw)
    targets = torch.randint(0, 90, (40,), generator=g).cuda()
    leaves = [t for t in (x, w) if t.requires_grad]
    ref = torch.autograd.grad(L.linear_cross_entropy(x, w, targets), leaves)
    asked, backward = [], _hip.linear_cross_entropy_bwd

    def recorded(*args):
        out = backward(*args)
        asked.append([g is not None for g in out])
        return out

    monkeypatch.setattr(_hip, "linear_cross_entropy_bwd", recorded)
    fn = torch.compile(lambda a, b: L.linear_cross_entropy(a, b, targets), fullgraph=True)
    got = torch.autograd.grad(fn(x, w), leaves)
    assert asked == [[dx, dw]] and all(torch.equal(a, b) for a, b in zip(got, ref))
