"""The native eager path of qk_norm_rope, embedding and linear_cross_entropy against their Python path (the
autograd.Function classes): the same kernels, so results are bitwise the same, over every form the native one
takes; what it hands back (None) runs or raises as the Python path does; saved tensors that come back
otherwise raise."""
import pytest
import torch

import _hip
import embedding as E
import linear_cross_entropy as L
import qk_norm_rope as Q
from krsi_testutil import log, seeded

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _cases(dt):
    """(public call, Python path, native entry, inputs, whether the native path takes the call)."""
    n = _hip.native()
    B, S, H, KH, D = 2, 9, 4, 2, 40
    cols = (H + 2 * KH) * D
    rope = Q.rope_table(30, 20)
    wide = seeded((B * S, cols + 16), 1, dtype=dt)
    wq, wk = (seeded((D,), i, std=0.1, mean=1.0, dtype=dt) for i in (2, 3))
    pos = torch.randint(0, 30, (B * S,), device="cuda")

    def qk(p, inter):
        dims = (B, S, H, KH, D, 1e-6, inter)
        return (lambda *t: Q.qk_norm_rope(*t, rope, B, S, H, D, 1e-6, kv_heads=KH, positions=p, interleaved=inter),
                lambda q, *t: Q.QKNormRope.apply(Q._in_place_layout(q, cols), *t, rope, p, *dims),
                lambda *t: n.qk_norm_rope(*t, rope, p, B, S, H, KH, D, 1e-6, int(inter)))

    tokens = torch.randint(0, 50, (3, 40), device="cuda")
    table = seeded((50, 24), 4, dtype=dt)

    def emb(t):
        return (lambda w: E.embedding(t, w, 2.5, padding_idx=1), lambda w: E.Embedding.apply(t, w, 2.5, 1),
                lambda w: n.embedding(t, w, 2.5, 1))

    cases = [
        (*qk(None, False), [wide[:, :cols].contiguous(), wq, wk], True),
        (*qk(pos, True), [wide, wq, wk], True),                                   # wider rows, read in place
        (*qk(pos.int(), False), [wide[:, 3:3 + cols], wq, wk], True),             # off alignment
        (*qk(pos.view(B, S), False), [wide, wq, wk], False),                      # positions to flatten
        (*qk(None, False), [wide[:, :cols].t().contiguous().t(), wq, wk], False),  # through a copy
        (*emb(tokens), [table], True),
        (*emb(tokens.int()[0, 0]), [table], True),
        (*emb(tokens.t()), [table], False),
        (*emb(tokens), [table.t().contiguous().t()], False),
    ]
    if dt != torch.float32:
        targets = torch.randint(0, 90, (70,), device="cuda")
        targets[::5] = 3
        x, w = seeded((70, 64), 5, dtype=dt), seeded((90, 64), 6, dtype=dt)
        for code, red in ((0, "none"), (1, "mean"), (2, "sum")):
            cases.append((lambda a, b, r=red: L.linear_cross_entropy(a, b, targets, ignore_index=3, reduction=r),
                          lambda a, b, r=red: L.LinearCrossEntropy.apply(a, b, targets, 3, r),
                          lambda a, b, c=code: n.linear_cross_entropy(a, b, targets, 3, c), [x, w], True))
        cases.append((lambda a, b: L.linear_cross_entropy(a, b, targets), lambda a, b: L.LinearCrossEntropy.apply(
            a, b, targets, -100, "mean"), lambda a, b: n.linear_cross_entropy(a, b, targets, -100, 1),
            [x.t().contiguous().t(), w], False))
    return cases


def _run(fn, inputs, needs):
    leaves = [t.detach().requires_grad_(n) for t, n in zip(inputs, needs)]
    out = fn(*leaves)
    g = seeded(out.shape, 99, dtype=out.dtype)
    return [out.detach(), *torch.autograd.grad(out, [t for t in leaves if t.requires_grad], g)]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: str(d).split(".")[-1])
def test_native_matches_python_path(dt):
    log(f"operators: native against Python path {dt}")
    assert _hip.native() is not _hip._NoNative
    for i, (fn, py, native, inputs, plain) in enumerate(_cases(dt)):
        log(f"case {i}")
        leaves = [t.detach().requires_grad_(True) for t in inputs]
        assert (native(*leaves) is not None) == plain
        assert isinstance(fn(*leaves).grad_fn, torch.autograd.function.BackwardCFunction) != plain
        for needs in [[True] * len(inputs)] + [[k == j for k in range(len(inputs))] for j in range(len(inputs))]:
            for a, b in zip(_run(fn, inputs, needs), _run(py, inputs, needs)):
                assert a.shape == b.shape and torch.equal(a, b)
        with torch.no_grad():
            assert (native(*inputs) is not None) == plain
            a, b = fn(*inputs), py(*inputs)
        assert not a.requires_grad and torch.equal(a, b)


def test_saved_tensor_hooks():
    """Saved tensors through hooks: to the CPU and back, bitwise the same; given back elsewhere, as another type or
    with another shape: an error."""
    log("operators: saved-tensor hooks")
    for fn, _, _, inputs, _ in _cases(torch.bfloat16):
        needs = [True] * len(inputs)
        plain = _run(fn, inputs, needs)
        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.cpu(), lambda t: t.cuda()):
            hooked = _run(fn, inputs, needs)
        assert packed and all(torch.equal(a, b) for a, b in zip(plain, hooked))
        for unpack in (lambda t: t.cpu(), lambda t: t.float() if t.dtype != torch.float32 else t.double(),
                       lambda t: t.flatten()[:-1]):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                with pytest.raises((ValueError, TypeError, RuntimeError, IndexError)):
                    _run(fn, inputs, needs)


def test_native_hands_back_what_is_not_plain():
    log("operators: forms handed back")
    n = _hip.native()
    rope = Q.rope_table(8, 8)
    qkv, w = seeded((8, 24), 1), seeded((8,), 2)
    tokens, table = torch.zeros(4, dtype=torch.int64, device="cuda"), seeded((5, 8), 3)
    x, targets = seeded((4, 64), 4), torch.zeros(4, dtype=torch.int64, device="cuda")
    qk = [qkv, w, w, rope, None, 1, 8, 1, 1, 8, 1e-6, 0]
    assert n.qk_norm_rope(*qk) is not None and n.embedding(tokens, table, 1.0, -1) is not None
    assert n.linear_cross_entropy(x, x, targets, -100, 1) is not None
    for i, bad in [(0, qkv.cpu()), (0, qkv.double()), (0, qkv[:, :16]), (1, w.float()), (2, w[:4]), (3, rope.double()),
                   (3, rope[:7]), (3, rope[:, :3]), (3, rope.clone().requires_grad_(True)), (4, tokens), (5, 2), (9, 12),
                   (10, 1), (11, 2), (0, None)]:
        assert n.qk_norm_rope(*[bad if k == i else v for k, v in enumerate(qk)]) is None, i
    for args in [(tokens.cpu(), table, 1.0, -1), (tokens.float(), table, 1.0, -1), (tokens, table.double(), 1.0, -1),
                 (tokens[:0], table, 1.0, -1), (tokens, table[0], 1.0, -1), (tokens, table, 1, -1), (tokens, table, 1.0)]:
        assert n.embedding(*args) is None
    for args in [(x.float(), x.float(), targets, -100, 1), (x, x[:, :32], targets, -100, 1), (x, x, targets[1:], -100, 1),
                 (x, x, targets, -100, 3), (x, x, targets, -100, None), (x[:0], x, targets[:0], -100, 1),
                 (x, x, targets.float(), -100, 1), (x.cpu(), x, targets, -100, 1)]:
        assert n.linear_cross_entropy(*args) is None


def test_calls_that_nothing_records():
    """With grad mode on and no input that requires a gradient: the same values, and no node."""
    log("operators: unrecorded calls")
    for fn, py, _, inputs, _ in _cases(torch.bfloat16):
        a = fn(*inputs)
        assert not a.requires_grad and a.grad_fn is None and torch.equal(a, py(*inputs))
        with torch.inference_mode():
            assert torch.equal(fn(*inputs), a)


def test_double_backward_is_refused():
    log("operators: double backward")
    for fn, _, _, inputs, _ in _cases(torch.bfloat16):
        leaves = [t.detach().requires_grad_(True) for t in inputs]
        out = fn(*leaves)
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out).requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grads[0].float().sum(), leaves)
