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


# ------------------------------- what state and param_groups hold at the time
def _same_as_new(opt, params):
    """That a step of opt moves params as one of a new optimizer does that is given opt's states."""
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = W.AdamW(copies, lr=opt.param_groups[0]["lr"])
    states = [{k: t.clone() for k, t in opt.state[p].items()} if opt.state.get(p) else {} for p in params]
    other.load_state_dict({"state": {i: s for i, s in enumerate(states) if s},
                           "param_groups": other.state_dict()["param_groups"]})
    _grads(params)
    _grads(copies)
    before = [p.detach().clone() for p in params]
    opt.step()
    other.step()
    for p, q, old in zip(params, copies, before):
        assert torch.equal(p, q) and not torch.equal(p, old)
        assert opt.state[p].keys() == other.state[q].keys()
        assert all(torch.equal(t, other.state[q][k]) for k, t in opt.state[p].items())


def test_parameter_replaced_in_its_group():
    params = _params()
    opt = _stepped(params)
    old, kept = params[0], params[0].detach().clone()
    params[0] = opt.param_groups[0]["params"][0] = torch.nn.Parameter(torch.full((6,), 2.0))
    _same_as_new(opt, params)
    assert torch.equal(old, kept) and int(opt.state[params[0]]["step"]) == 1


def test_group_taken_out_and_group_replaced():
    params = _params(4)
    opt = W.AdamW([{"params": params[:2]}, {"params": params[2:]}], lr=0.1)
    _grads(params)
    opt.step()
    gone = opt.param_groups.pop()["params"]
    kept = [p.detach().clone() for p in gone]
    _same_as_new(opt, params[:2])
    assert all(torch.equal(p, q) for p, q in zip(gone, kept))
    opt.param_groups[0] = {**opt.param_groups[0], "lr": 0.3}
    _same_as_new(opt, params[:2])
    opt.param_groups = [{**opt.param_groups[0], "params": params[1:3], "lr": 0.2}]
    kept = params[0].detach().clone()
    _same_as_new(opt, params[1:3])
    assert torch.equal(params[0], kept)


def test_states_cleared_and_replaced():
    params = _params()
    opt = _stepped(params)
    opt.state.clear()
    _same_as_new(opt, params)
    assert [int(opt.state[p]["step"]) for p in params] == [1, 1, 1] and len(opt.state_dict()["state"]) == 3
    opt.state[params[1]]["exp_avg"] = torch.full((4,), -3.0)
    _same_as_new(opt, params)
    opt.state[params[2]]["step"] = torch.tensor(40, dtype=torch.int32)
    _same_as_new(opt, params)
    assert int(opt.state[params[2]]["step"]) == 41
    s = opt.state[params[0]]
    s["exp_avg"], s["exp_avg_sq"] = s["exp_avg_sq"].abs(), s["exp_avg"].abs()
    _same_as_new(opt, params)
    del opt.state[params[0]]
    _same_as_new(opt, params)
    assert [int(opt.state[p]["step"]) for p in params] == [1, 5, 43]


def test_lists_stay_where_nothing_changed_and_are_not_made_in_a_capture(capturing):
    params = _params()
    opt = _stepped(params)
    counts = [opt.state[p]["step"] for p in params]
    opt.param_groups[0]["lr"] = 0.2
    opt.state[params[0]]["exp_avg"].zero_()
    _same_as_new(opt, params)
    assert all(opt.state[p]["step"] is t for p, t in zip(params, counts))
    capturing["now"] = True
    opt.step()
    opt.state[params[0]]["exp_avg"] = torch.zeros(4)
    with pytest.raises(RuntimeError, match="first step"):
        opt.step()
    assert all(opt.state[p]["step"] is t and int(t) == 3 for p, t in zip(params, counts))


# ------------------------------------------------ parameters without a gradient
def test_states_come_with_the_first_gradient(capturing):
    """A frozen parameter has no state, and may be of any kind and place; once it gets a gradient it begins as it is then."""
    frozen = torch.nn.Parameter(torch.ones(4, dtype=torch.bfloat16), requires_grad=False)
    indices = torch.nn.Parameter(torch.arange(3), requires_grad=False)
    odd = torch.nn.Parameter(torch.ones(3, 4).t(), requires_grad=False)
    params = [frozen, *_params(2), indices, odd]
    opt = W.AdamW(params, lr=0.1)
    _grads(params[1:3])
    opt.step()
    assert set(opt.state) == set(params[1:3]) and set(opt.state_dict()["state"]) == {1, 2}
    counts = [opt.state[p]["step"] for p in params[1:3]]
    params[1].grad = None  # without a gradient this time: its state stays, and so does its place
    opt.step()
    assert [int(t) for t in counts] == [1, 2] and all(opt.state[p]["step"] is t for p, t in zip(params[1:3], counts))
    with torch.no_grad():
        frozen.fill_(3.0)  # loaded
    frozen.requires_grad_(True)
    frozen.grad = torch.zeros_like(frozen)
    capturing["now"] = True
    with pytest.raises(RuntimeError, match="first step"):
        opt.step()
    capturing["now"] = False
    opt.step()
    assert torch.equal(opt.state[frozen]["master"], torch.full((4,), 3.0 * (1 - 0.1 * 0.01)))
    assert [int(opt.state[p]["step"]) for p in params[:3]] == [1, 1, 3]


def test_capture_right_after_loading_beside_a_frozen_parameter(capturing):
    a, b = _params(), _params()
    for ps in (a, b):
        ps[1].requires_grad_(False)
    opt, other = W.AdamW(a, lr=0.1), W.AdamW(b, lr=0.1)
    for p in (a[0], a[2]):
        p.grad = torch.ones_like(p)
    opt.step()
    other.load_state_dict(opt.state_dict())
    for p in (b[0], b[2]):
        p.grad = torch.ones_like(p)
    capturing["now"] = True
    other.step()
    assert [int(other.state[b[i]]["step"]) for i in (0, 2)] == [2, 2] and b[1] not in other.state


# --------------------------------------------------- masters and their parameters
def _bf16(value=0.9, n=3):
    params = [torch.nn.Parameter(torch.full((4,), value, dtype=torch.bfloat16)) for _ in range(n)]
    opt = _stepped(params, lr=1e-3, weight_decay=0.0)
    _grads(params, 0.25)  # small steps: the masters are between two bf16 numbers
    opt.step()
    assert all(not torch.equal(opt.state[p]["master"], p.float()) for p in params)
    return params, opt


CHANGES = {
    "filled": lambda p: p.fill_(5.0),
    "loaded": lambda p: p.copy_(torch.full((4,), 5.0)),
    "exchanged": lambda p: setattr(p, "data", torch.full((4,), 5.0, dtype=torch.bfloat16)),
}


@pytest.mark.parametrize("change", CHANGES)
def test_masters_follow_changed_parameters(change):
    params, opt = _bf16()
    masters = [opt.state[p]["master"].clone() for p in params]
    with torch.no_grad():
        CHANGES[change](params[1])
    opt.param_groups[0]["lr"] = 0.0
    opt.step()
    assert torch.equal(params[1], torch.full((4,), 5.0, dtype=torch.bfloat16))
    assert torch.equal(opt.state[params[1]]["master"], torch.full((4,), 5.0))
    assert all(torch.equal(opt.state[params[i]]["master"], masters[i]) for i in (0, 2))


def test_masters_keep_what_did_not_change():
    """A clamp that meets one element: the others' masters keep what is below their rounding. Then nothing changes, and
    nothing is taken over."""
    params, opt = _bf16()
    master = opt.state[params[0]]["master"].clone()
    with torch.no_grad():
        params[0][2] = 0.5
    opt.param_groups[0]["lr"] = 0.0
    opt.step()
    master[2] = 0.5
    assert torch.equal(opt.state[params[0]]["master"], master)
    taken = []
    with pytest.MonkeyPatch.context() as m:
        m.setattr(W, "_follow", lambda master, p: taken.append(p))
        opt.step()
        opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.ones(2, dtype=torch.bfloat16)))
        opt.param_groups[0]["params"][-1].grad = torch.ones(2, dtype=torch.bfloat16)
        opt.step()  # lists made again
    assert not taken


def test_change_before_the_lists_are_made_again():
    params, opt = _bf16()
    with torch.no_grad():
        params[0].fill_(5.0)
    opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.ones(2, dtype=torch.bfloat16)))
    opt.param_groups[0]["params"][-1].grad = torch.ones(2, dtype=torch.bfloat16)
    opt.param_groups[0]["lr"] = 0.0
    opt.step()
    assert torch.equal(params[0], torch.full((4,), 5.0, dtype=torch.bfloat16))


@pytest.mark.parametrize("model_first", [True, False])
def test_loading_keeps_the_masters(model_first):
    """Whichever is loaded first, the saved masters stand: they are what the saved parameters are the rounding of."""
    a, opt = _bf16()
    b = [torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16)) for _ in a]
    other = W.AdamW(b, lr=1e-3, weight_decay=0.0)

    def load_model():
        with torch.no_grad():
            for p, q in zip(a, b):
                q.copy_(p)

    if model_first:
        load_model()
    other.load_state_dict(opt.state_dict())
    if not model_first:
        load_model()
    _grads(a, 0.25)
    _grads(b, 0.25)
    opt.step()
    other.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], other.state[q]["master"])
    clone = copy.deepcopy(other)
    c = clone.param_groups[0]["params"]
    _grads(c, 0.25)
    with torch.no_grad():
        c[0].fill_(5.0)
    clone.step()
    other.step()
    assert (c[0] > 4.9).all() and all(torch.equal(clone.state[p]["master"], other.state[q]["master"])
                                      for p, q in zip(c[1:], b[1:]))


def test_changes_that_torch_does_not_count():
    params, opt = _bf16()
    masters = [opt.state[p]["master"].clone() for p in params]
    params[0].data.fill_(5.0)
    params[1].data[1] = float("nan")
    opt.masters_from_parameters()
    masters[0].fill_(5.0)
    masters[1][1] = float("nan")
    for p, t in zip(params, masters):
        assert torch.equal(opt.state[p]["master"].nan_to_num(7.0), t.nan_to_num(7.0))


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_states_under_another_default_dtype(default):
    torch.set_default_dtype(default)
    try:
        params = [torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16))]
        opt = W.AdamW(params, lr=0.1, state_bits=8)
        state = opt._new_state(params[0])
    finally:
        torch.set_default_dtype(torch.float32)
    assert {k: t.dtype for k, t in state.items()} == {
        "step": torch.int32, "exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.float8_e4m3fn, "scales": torch.float32,
        "master": torch.float32}
