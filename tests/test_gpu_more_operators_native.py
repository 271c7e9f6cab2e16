"""The native eager path of add_rmsnorm, quantize_rows and linear_8bit against their Python path: the same kernels, so
results are bitwise the same; what it hands back (None) runs or raises as the Python path does; saved tensors that come
back otherwise raise; captured, compiled and on another stream they give the eager results."""
import pytest
import torch

import _hip
import add_rmsnorm as A
import linear_8bit as L
from krsi_testutil import log, seeded

pytestmark = pytest.mark.gpu
EPS = 1e-6
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ids = lambda d: str(d).split(".")[-1]  # noqa: E731


def _inputs(dt, rows=37, n=200):
    return [seeded((rows, n), 1, dtype=dt), seeded((rows, n), 2, dtype=dt), seeded((n,), 3, std=0.1, mean=1.0, dtype=dt)]


def _same(a, b):
    return a is b is None or torch.equal(a.float(), b.float())


def _run(fn, inputs, needs, used):
    leaves = [t.detach().requires_grad_(n) for t, n in zip(inputs, needs)]
    out = fn(*leaves)
    outs = [o for o, u in zip(out, used) if u]
    g = [seeded(o.shape, 90 + i, dtype=o.dtype) for i, o in enumerate(outs)]
    grads = torch.autograd.grad(outs, [t for t in leaves if t.requires_grad], g, allow_unused=True)
    return [o.detach() for o in out] + list(grads)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_native_matches_python_path(dt):
    log(f"add_rmsnorm native against Python path {dt}")
    n = _hip.native()
    assert n is not _hip._NoNative
    inputs = _inputs(dt)
    leaves = [t.detach().requires_grad_(True) for t in inputs]
    assert n.add_rmsnorm(*leaves, EPS) is not None
    assert not isinstance(A.add_rmsnorm(*leaves, EPS)[0].grad_fn, torch.autograd.function.BackwardCFunction)
    for needs in [[True] * 3] + [[k == j for k in range(3)] for j in range(3)]:
        for used in ((1, 1), (1, 0), (0, 1)):
            if used == (0, 1) and needs == [False, False, True]:
                continue  # the stream does not depend on the weight
            for a, b in zip(_run(lambda *t: A.add_rmsnorm(*t, EPS), inputs, needs, used),
                            _run(lambda *t: A.AddRMSNorm.apply(*t, EPS), inputs, needs, used)):
                assert _same(a, b), (needs, used)
    with torch.no_grad():
        for a, b in zip(n.add_rmsnorm(*inputs, EPS), _hip.add_rmsnorm_fwd(*inputs, EPS)):
            assert torch.equal(a, b)
        for res in (inputs[1], None):
            for a, b in zip(n.add_rmsnorm_8bit(inputs[0], res, inputs[2], EPS), _hip.add_rmsnorm_8bit(inputs[0], res, inputs[2], EPS)):
                assert _same(a, b)
        for a, b in zip(n.quantize_rows(inputs[0]), _hip.quantize_rows(inputs[0])):
            assert _same(a, b)
        w, ws = _hip.quantize_rows(seeded((40, 208), 5))
        for rows in (3, 90):
            x = seeded((rows, 208), 6, dtype=dt)
            q, s = _hip.quantize_rows(x)
            for code, out_dt in enumerate((torch.bfloat16, torch.float16, torch.float32)):
                want = _hip.linear_8bit(q, w, ws, s, out_dt)
                assert torch.equal(n.linear_8bit(q, w, ws, s, code), want) and torch.equal(n.linear_8bit(x, w, ws, None, code), want)


def test_native_hands_back_what_is_not_plain():
    log("add_rmsnorm, linear_8bit: forms handed back")
    n = _hip.native()
    x, r, w = _inputs(torch.bfloat16, 4, 64)
    ok = [x, r, w, EPS]
    for i, bad in [(0, x.cpu()), (0, x.double()), (0, x.t()), (0, x[0]), (0, x[:0]), (1, r[:3]), (1, r.float()), (1, None), (1, r.t()),
                   (2, w[:63]), (2, w.float()), (3, 1), (0, torch.stack([x, x], 2)[..., 0])]:
        args = [bad if k == i else v for k, v in enumerate(ok)]
        assert n.add_rmsnorm(*args) is None, (i, bad)
        if not (i == 1 and bad is None):
            assert n.add_rmsnorm_8bit(*args) is None, (i, bad)
    assert n.add_rmsnorm(x, r, w) is None and n.add_rmsnorm(x, r, w, float("nan")) is None
    for bad in (x.cpu(), x.double(), x[0], x[:0], x.t(), None):
        assert n.quantize_rows(bad) is None
    q, s = _hip.quantize_rows(x)
    wq, ws = _hip.quantize_rows(seeded((32, 64), 4))
    ok = [q, wq, ws, s, 0]
    assert n.linear_8bit(*ok) is not None
    for i, bad in [(0, x), (0, q[:, :48]), (0, q[0]), (0, q.cpu()), (1, wq.float()), (1, wq[:, :48]), (2, ws[:5]), (2, ws.double()),
                   (3, s[:2]), (3, None), (4, 3), (4, None), (4, -1)]:
        assert n.linear_8bit(*[bad if k == i else v for k, v in enumerate(ok)]) is None, (i, bad)


def test_saved_tensor_hooks():
    log("add_rmsnorm: saved-tensor hooks")
    inputs = _inputs(torch.bfloat16)
    for fn in (lambda *t: A.add_rmsnorm(*t, EPS), lambda *t: A.AddRMSNorm.apply(*t, EPS)):
        plain = _run(fn, inputs, [True] * 3, (1, 1))
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.cpu(), lambda t: t.cuda()):
            hooked = _run(fn, inputs, [True] * 3, (1, 1))
        assert packed and all(torch.equal(a, b) for a, b in zip(plain, hooked))
        for unpack in (lambda t: t.cpu(), lambda t: t.float() if t.dtype != torch.float32 else t.double(),
                       lambda t: t.flatten()[:-1]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                with pytest.raises((ValueError, TypeError, RuntimeError, IndexError)):
                    _run(fn, inputs, [True] * 3, (1, 1))


def test_stream_changed_in_place_is_noticed():
    """The backward reads r: changing it between is an error, as for any saved output."""
    log("add_rmsnorm: r changed in place")
    leaves = [t.requires_grad_(True) for t in _inputs(torch.float32)]
    y, r = A.add_rmsnorm(*leaves, EPS)
    with torch.no_grad():
        r.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_double_backward_is_refused():
    log("add_rmsnorm: double backward")
    for fn in (A.add_rmsnorm, A.AddRMSNorm.apply):
        leaves = [t.requires_grad_(True) for t in _inputs(torch.float32)]
        y, r = fn(*leaves, EPS)
        g = torch.ones_like(y).requires_grad_(True)
        grads = torch.autograd.grad([y, r], leaves, [g, torch.ones_like(r)], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grads[0].sum(), leaves)


def test_unrecorded_calls():
    inputs = _inputs(torch.bfloat16)
    y, r = A.add_rmsnorm(*inputs, EPS)
    assert not y.requires_grad and y.grad_fn is None and not r.requires_grad
    with torch.inference_mode():
        y2, r2 = A.add_rmsnorm(*inputs, EPS)
        assert torch.equal(y2, y) and torch.equal(r2, r)
        q, s, _ = A.add_rmsnorm_8bit(*inputs, EPS)
    assert torch.equal(q.float(), A.add_rmsnorm_8bit(*inputs, EPS)[0].float())


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_compiled(dt):
    """Under torch.compile(fullgraph=True): forward, gradients and the 8-bit forms as eager."""
    log(f"add_rmsnorm compiled {dt}")
    torch._dynamo.reset()
    inputs = _inputs(dt, 16, 128)

    def block(x, res, w):
        y, r = A.add_rmsnorm(x, res, w, EPS)
        return y, r

    for a, b in zip(_run(torch.compile(block, fullgraph=True), inputs, [True] * 3, (1, 1)), _run(block, inputs, [True] * 3, (1, 1))):
        assert torch.equal(a, b)

    def eight(x, res, w, wq, ws):
        q, s, r = A.add_rmsnorm_8bit(x, res, w, EPS)
        q2, s2, _ = A.add_rmsnorm_8bit(r, None, w, EPS)
        return L.linear_8bit(q, wq, ws, x_scale=s), L.linear_8bit(q2, wq, ws, x_scale=s2), r

    with torch.no_grad():
        wq, ws = L.quantize_rows(seeded((48, 128), 9))
        for a, b in zip(torch.compile(eight, fullgraph=True)(*inputs, wq, ws), eight(*inputs, wq, ws)):
            assert torch.equal(a, b)


def test_captured_and_on_another_stream():
    """A captured forward and backward with new inputs in each replay, eager work between them; and on a side stream."""
    log("add_rmsnorm captured")
    inputs = _inputs(torch.bfloat16, 50, 1000)
    gy, gr = seeded((50, 1000), 7), seeded((50, 1000), 8)
    leaves = [t.detach().clone().requires_grad_(True) for t in inputs]

    def step(ts):
        y, r = A.add_rmsnorm(*ts, EPS)
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], ts, [gy, gr])]  # no graph outlives the step

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(leaves)
    side.synchronize()
    eager = [t.detach().clone().requires_grad_(True) for t in inputs]
    assert all(torch.equal(a, b) for a, b in zip(first, step(eager)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
        with torch.no_grad():
            codes = A.add_rmsnorm_8bit(*leaves, EPS)
    for i in range(4):
        with torch.no_grad():
            for t, e in zip(leaves, eager):
                t.copy_(seeded(tuple(t.shape), 20 + i))
                e.copy_(t)
        graph.replay()
        want = step(eager)
        with torch.no_grad():
            want_codes = A.add_rmsnorm_8bit(*eager, EPS)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(codes, want_codes)), i
