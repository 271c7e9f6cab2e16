"""The class AdamW without a GPU: which tensors it steps, and when its lists are made. The launch is replaced by the same
arithmetic in torch, so the tests are of the class alone; what the kernels compute is tested on the GPU."""
import copy

import pytest
import torch

import _hip
import adamw as W


def _step(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas, eps, weight_decay, masters=None, scales=None,
          max_norm=None, norm=None, seed=0):
    share = 1.0 if norm is None else min(1.0, max_norm / (float(norm) + 1e-6))
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs)):
        if g is None:
            continue
        steps[i] += 1
        t, w = int(steps[i]), p if masters is None else masters[i]
        m.mul_(betas[0]).add_(g * share, alpha=1 - betas[0])
        v.mul_(betas[1]).add_((g * share).square(), alpha=1 - betas[1])
        w.mul_(1 - lr * weight_decay).sub_(
            lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps))
        if masters is not None:
            p.copy_(w)


@pytest.fixture(autouse=True)
def capturing(monkeypatch):
    """The launch replaced; {"now": whether a capture is on}."""
    state = {"now": False}
    monkeypatch.setattr(W, "adamw_step", _step)
    monkeypatch.setattr(W, "grad_norm", lambda gs: torch.stack([g.float().square().sum() for g in gs]).sum().sqrt())
    monkeypatch.setattr(_hip, "_on_gpu", lambda *ts: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["now"])
    return state


def _params(n=3, dt=torch.float32):
    return [torch.nn.Parameter(torch.full((4,), 1.0 + i, dtype=dt)) for i in range(n)]


def _grads(params, value=0.5):
    for p in params:
        p.grad = torch.full_like(p, value)


def _stepped(params, **kw):
    opt = W.AdamW(params, **{"lr": 0.1, **kw})
    _grads(params)
    opt.step()
    return opt


# ------------------------------------------------------------------ captures
def test_capture_right_after_loading(capturing):
    """Loaded states are listed when they are loaded: a step that is captured next records no making of the counts."""
    a, b = _params(), _params()
    opt, other = _stepped(a), W.AdamW(b, lr=0.1)
    other.load_state_dict(opt.state_dict())
    counts = [other.state[p]["step"] for p in b]
    _grads(b)
    capturing["now"] = True
    other.step()
    assert [other.state[p]["step"] for p in b] == [2, 2, 2]
    assert all(other.state[p]["step"] is t for p, t in zip(b, counts))  # the ones that later steps count on


@pytest.mark.parametrize("make", [copy.deepcopy, lambda opt: W.AdamW(_params())], ids=["copied", "new"])
def test_no_lists_are_made_in_a_capture(make, capturing):
    other = make(_stepped(_params()))
    params = other.param_groups[0]["params"]
    _grads(params)
    before = {p: dict(other.state[p]) for p in params}
    capturing["now"] = True
    with pytest.raises(RuntimeError, match="first step"):
        other.step()
    for p in params:
        assert other.state[p].keys() == before[p].keys() and all(t is before[p][k] for k, t in other.state[p].items())
    capturing["now"] = False
    other.step()
    capturing["now"] = True
    other.step()
