"""embedding (token lookup with scaling) on the GPU: the forward bitwise, the gradient against 64 bits.

Tolerance of the gradient, derived: a row's sum of c rows takes at most c - 1 additions in fp32 and one product,
each off by half a step (2^-24) of a value no larger than the sum of magnitudes, then one rounding to the type."""
import pytest
import torch

import embedding as E
import krsi_oracle as O
from _harness import selftest_autograd
from krsi_testutil import log, seeded
from test_gpu_graphs import _replay_matches

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
STEP = 2.0 ** -24


def _tokens(kind, n, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), V - 1)
    if kind == "two":  # two long runs and short ones between them
        t = torch.randint(0, V, (n,), generator=g)
        u = torch.rand(n, generator=g)
        return torch.where(u < 0.45, 0, torch.where(u < 0.9, V // 2, t))
    if kind == "low":  # ids that all lie in one narrow range
        return torch.randint(0, min(V, 64), (n,), generator=g)
    return torch.randint(0, V, (n,), generator=g)


def _check_grad(got, dout, tokens, V, scale, dt, padding_idx=None):
    ref, mag, count = O.embedding_grad_64(dout.cpu(), tokens.cpu(), V, scale, padding_idx)
    got = got.cpu().double()
    bound = torch.finfo(dt).eps / 2 * ref.abs() * (1 + STEP) + (count + 1) * STEP * mag
    if dt == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    off = (got - ref).abs()
    assert got.shape == ref.shape and bool((off <= bound).all()), (off - bound).max().item()
    assert (got[(count == 0)[:, 0]] == 0).all()


CASES = [  # n, V, D, tokens
    (1, 1, 1, "any"), (1, 5, 8, "any"), (2, 300, 3, "one"), (31, 256, 10, "any"), (32, 7, 72, "one"),
    (33, 1, 64, "one"), (33, 257, 1001, "two"), (64, 1000, 9, "low"), (95, 3, 513, "two"), (1000, 255, 40, "any"),
    (1025, 70001, 24, "any"), (4097, 50, 128, "any"), (5000, 4000, 17, "two"), (8191, 32128, 64, "low"),
    (20000, 30, 8, "two"), (700, 300000, 4, "any"), (3000, 2000, 4096, "two"), (66000, 900, 16, "one"),
]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: str(d).split(".")[-1])
@pytest.mark.parametrize("n,V,D,kind", CASES)
def test_forward_and_gradient(n, V, D, kind, dt):
    log(f"embedding n{n} V{V} D{D} {kind} {dt}")
    tokens = _tokens(kind, n, V).cuda()
    table = seeded((V, D), 1, dtype=dt).requires_grad_(True)
    scale = D ** 0.5
    out = E.embedding(tokens, table, scale)
    assert torch.equal(out, (table.detach()[tokens].float() * scale).to(dt))
    dout = seeded((n, D), 2, dtype=dt)
    (g,) = torch.autograd.grad(out, table, dout, retain_graph=True)
    _check_grad(g, dout, tokens, V, scale, dt)
    assert torch.equal(g, torch.autograd.grad(out, table, dout)[0])  # bitwise reproducible
    (g32,) = torch.autograd.grad(E.embedding(tokens.int(), table, scale), table, dout)
    assert torch.equal(g, g32)


@pytest.mark.parametrize("n", [50, 3000])
def test_padding_and_tokens_outside_the_table(n):
    """A token outside [0, V): a NaN row, no gradient. padding_idx: its row is looked up, its gradient stays zero."""
    V, D = 100, 36
    log(f"embedding padding and bad tokens n{n}")
    tokens = _tokens("any", n, V)
    tokens[::3] = 7
    tokens[1::10] = torch.tensor([-1, V, 1 << 40, -(1 << 40), -100]).repeat(n)[:len(tokens[1::10])]
    table = seeded((V, D), 1, dtype=torch.float32).requires_grad_(True)
    dout = seeded((n, D), 2, dtype=torch.float32)
    inside = (tokens >= 0) & (tokens < V)
    for pad in (7, 7 - V, None):
        out = E.embedding(tokens.cuda(), table, padding_idx=pad)
        assert torch.equal(out[inside], table.detach()[tokens[inside].cuda()])
        assert torch.isnan(out[~inside]).all()
        (g,) = torch.autograd.grad(out, table, dout)
        _check_grad(g, dout, tokens, V, 1.0, torch.float32, None if pad is None else 7)
    tokens[:] = 7
    (g,) = torch.autograd.grad(E.embedding(tokens.cuda(), table, padding_idx=7), table, dout)
    assert not g.any()


def test_shapes_and_layouts():
    """Any shape of tokens, also none and empty; strided tokens, tables and gradients."""
    log("embedding shapes and layouts")
    table = seeded((11, 20), 1)
    for shape in ((), (0,), (3, 0), (2, 3, 4)):
        tokens = torch.randint(0, 11, shape, device="cuda")
        leaf = table.detach().requires_grad_(True)
        out = E.embedding(tokens, leaf)
        assert out.shape == (*shape, 20) and torch.equal(out, table[tokens])
        dout = seeded(out.shape, 3)
        (g,) = torch.autograd.grad(out, leaf, dout)
        _check_grad(g, dout, tokens, 11, 1.0, torch.bfloat16)
    tokens = torch.randint(0, 11, (6, 8), device="cuda")
    wide = seeded((20, 13), 4)
    leaf = wide.t()[:11, 1:].detach().requires_grad_(True)  # transposed, off alignment
    out = E.embedding(tokens.t()[1:], leaf)
    assert torch.equal(out, leaf.detach()[tokens.t()[1:]])
    dout = seeded((19, 6, 7), 5).permute(2, 1, 0)
    (g,) = torch.autograd.grad(out, leaf, dout)
    _check_grad(g, dout, tokens.t()[1:], 11, 1.0, torch.bfloat16)
    base = seeded((5 * 16 + 1,), 6)
    odd = base[1:].view(5, 16)  # rows off every vector alignment
    assert torch.equal(E.embedding(tokens % 5, odd), odd[tokens % 5])


def test_infinities_and_nan_stay_in_their_rows():
    log("embedding infinities and NaN")
    tokens = torch.arange(200, device="cuda") % 10
    table = seeded((10, 16), 1, dtype=torch.float32)
    table[3, 2], table[4] = float("inf"), float("nan")
    leaf = table.requires_grad_(True)
    out = E.embedding(tokens, leaf, 2.0)
    assert torch.equal(out.nan_to_num(7.0), (leaf.detach() * 2)[tokens].nan_to_num(7.0))
    dout = seeded(out.shape, 2, dtype=torch.float32)
    dout[5], dout[6, 1] = float("nan"), float("inf")
    (g,) = torch.autograd.grad(out, leaf, dout)
    assert torch.isnan(g[5]).all() and g[6, 1] == float("inf")
    assert torch.isfinite(g[[0, 1, 2, 3, 4, 7, 8, 9]]).all()


def test_tables_past_two_to_the_31():
    """A table of more elements than 31 bits count: rows at its end."""
    V, D = 1 << 20, 2064
    log(f"embedding V{V} D{D}")
    table = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    table[-3:] = seeded((3, D), 1)
    tokens = torch.tensor([V - 1, 0, V - 3, V - 1, V - 2], device="cuda")
    leaf = table.requires_grad_(True)
    out = E.embedding(tokens, leaf)
    assert torch.equal(out, table.detach()[tokens])
    dout = seeded(out.shape, 2)
    (g,) = torch.autograd.grad(out, leaf, dout)
    _check_grad(g[-3:], dout[[0, 2, 3, 4]], tokens[[0, 2, 3, 4]] - (V - 3), 3, 1.0, torch.bfloat16)
    assert torch.equal(g[0], dout[1]) and not g[1:-3].any()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: str(d).split(".")[-1])
def test_graph_replay_matches_eager(dt):
    log(f"embedding graph replay {dt}")
    tokens = _tokens("two", 2000, 500).cuda()
    other = seeded((64, 256), 6)
    _replay_matches(lambda t: E.embedding(tokens, t, 3.0), [seeded((500, 48), 1, dtype=dt)],
                    seeded((2000, 48), 2, dtype=dt), lambda: other.float().square().sum(1))


def test_tokens_changed_between_replays():
    """A captured backward reads the tokens that its buffer holds at the replay."""
    log("embedding replay with other tokens")
    tokens, dout = _tokens("two", 900, 60).cuda(), seeded((900, 24), 2)
    table = seeded((60, 24), 1).requires_grad_(True)

    def step():
        return torch.autograd.grad(E.embedding(tokens, table), table, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = step()
    for kind in ("one", "any", "two"):
        tokens.copy_(_tokens(kind, 900, 60, seed=4))
        graph.replay()
        torch.cuda.synchronize()
        _check_grad(g, dout, tokens, 60, 1.0, torch.bfloat16)


def test_selftest_protocol_and_compile():
    log("selftest_autograd embedding + torch.compile(fullgraph)")
    torch.manual_seed(0)
    tokens = torch.randint(0, 700, (4, 100), device="cuda")
    res = selftest_autograd(lambda t: E.embedding(tokens, t, 8.0, padding_idx=3),
                            lambda t: E.reference(tokens, t, 8.0, padding_idx=3), [seeded((700, 64), 0)], time=False)
    assert res["pass"], res["checks"]
    assert res["compiled"].get("pass"), res["compiled"]


def test_refusals():
    log("embedding refusals")
    tokens, table = torch.zeros(4, dtype=torch.int64, device="cuda"), seeded((5, 8), 1)
    for error, args, kw in [(ValueError, (tokens.cpu(), table), {}), (TypeError, (tokens.float(), table), {}),
                            (TypeError, (tokens, table.double()), {}), (ValueError, (tokens, table[0]), {}),
                            (ValueError, (tokens, table[:0]), {}), (ValueError, (tokens, table), {"padding_idx": 5}),
                            (ValueError, (tokens, table), {"padding_idx": -6}),
                            (RuntimeError, (tokens, table, float("inf")), {})]:
        with pytest.raises(error):
            E.embedding(*args, **kw)
