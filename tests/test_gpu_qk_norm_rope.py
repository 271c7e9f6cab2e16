"""qk_norm_rope (the norm of query and key heads with the position rotation) on the GPU against its closed
form in 64 bits.

Tolerances, derived: an output is rounded once to its type (half a step, finfo.eps / 2 of the value); before
that it is a short chain of fp32 operations of half a step each on terms whose magnitudes the oracle gives.
The chain: D squares added (D steps, half of which reach r), and about 16 further operations; in dx the sum
dn x as well (D steps more). A weight's gradient adds one term per token and head, so as many steps again.
"""
import pytest
import torch

import krsi_oracle as O
import qk_norm_rope as Q
from _harness import selftest_autograd
from krsi_testutil import log, seeded
from test_gpu_graphs import _replay_matches

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6
STEP = 2.0 ** -24


def _inputs(B, S, H, KH, D, R, dt, seed=0, length=None):
    qkv = seeded((B * S, (H + 2 * KH) * D), seed, dtype=dt)
    wq, wk = (seeded((D,), seed + i, std=0.1, mean=1.0, dtype=dt) for i in (1, 2))
    return qkv, wq, wk, Q.rope_table(length or S, R)


def _check(name, got, ref, mag, steps, dt):
    got = got.cpu().double()
    bound = torch.finfo(dt).eps / 2 * ref.abs() + steps * STEP * mag
    if dt == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    worst = ((got - ref).abs() / bound.clamp_min(1e-300)).max().item() if ref.numel() else 0.0
    log(f"{name}: worst {worst:.3f} of its bound")
    assert got.shape == ref.shape and bool(((got - ref).abs() <= bound).all()), (name, worst)


def _verify(out, grads, dout, qkv, wq, wk, rope, pos, H, KH, D, inter, dt, eps=EPS):
    args = [t.detach().cpu() for t in (qkv, wq, wk, rope)]
    pos = pos.reshape(-1).cpu().long()
    tokens = len(pos)
    _check("out", out.detach(), *O.qk_norm_rope_64(*args, pos, H, KH, D, eps, inter), D / 2 + 16, dt)
    refs, mags = O.qk_norm_rope_grads_64(dout.cpu(), *args, pos, H, KH, D, eps, inter)
    for name, got, ref, mag, n in zip(("dqkv", "dwq", "dwk"), grads, refs, mags, (0, tokens * H, tokens * KH)):
        _check(name, got, ref, mag, 2.5 * D + 16 + n, dt)


CASES = [  # B, S, H, KH, D, R, interleaved, positions
    (1, 1, 1, 1, 8, 2, False, False),        # one token, one head: the smallest there is
    (1, 1, 1, 1, 128, 126, False, False),    # a pair width of one column
    (2, 7, 3, 1, 40, 20, True, False),
    (2, 70, 3, 3, 72, 72, False, False),     # head groups of 9 of 16 lanes
    (1, 129, 16, 4, 128, 64, True, False),   # few key heads, half of the columns rotate
    (3, 1, 32, 16, 128, 128, False, True),   # one step of generation
    (2, 33, 5, 5, 24, 10, False, True),      # R / 2 odd
    (1, 65, 33, 11, 96, 96, True, True),     # heads that no wave divides
    (2, 2049, 4, 2, 64, 64, False, False),   # more items than a backward's waves
    (1, 37, 1, 1, 72, 36, False, True),      # several tokens to a wave; chunks that share columns in both parts
    (2, 5, 1, 1, 8, 4, True, False),         # as many tokens to a wave as there are
    (1, 40, 2, 2, 72, 44, True, False),      # shared columns, adjacent pairs
    (3, 1, 7, 1, 104, 54, False, True),
]


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: str(d).split(".")[-1])
@pytest.mark.parametrize("B,S,H,KH,D,R,inter,positions", CASES)
def test_against_64_bits(B, S, H, KH, D, R, inter, positions, dt):
    log(f"qk_norm_rope B{B} S{S} H{H} KH{KH} D{D} R{R} interleaved {inter} positions {positions} {dt}")
    qkv, wq, wk, rope = _inputs(B, S, H, KH, D, R, dt, length=300 if positions else S)
    pos = torch.randint(0, 300, (B, S), generator=torch.Generator().manual_seed(3)).cuda() if positions else None
    dout = seeded(qkv.shape, 9, dtype=dt)
    leaves = [t.requires_grad_(True) for t in (qkv, wq, wk)]
    out = Q.qk_norm_rope(*leaves, rope, B, S, H, D, EPS, kv_heads=KH, positions=pos, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    implied = torch.arange(B * S) % S if pos is None else pos
    _verify(out, grads, dout, *leaves, rope, implied, H, KH, D, inter, dt)
    again = torch.autograd.grad(out, leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    if pos is not None:  # int32 positions name the same rows
        assert torch.equal(out, Q.qk_norm_rope(*leaves, rope, B, S, H, D, EPS, kv_heads=KH, positions=pos.int(),
                                               interleaved=inter))


@pytest.mark.parametrize("layout", ["wide", "slice_off_alignment", "column_stride", "rows_overlap", "one_row"])
def test_layouts(layout):
    """A wider tensor, a slice off every alignment, a transposed one, rows of stride 0 and a single row of any
    stride give what their contiguous copy gives; the gradient is zero outside the heads' columns."""
    B, S, H, D, dt = 2, 9, 3, 40, torch.bfloat16
    cols = 3 * H * D
    log(f"qk_norm_rope layout {layout}")
    wide = seeded((B * S, cols + 13), 1, dtype=dt)
    base, view = {
        "wide": lambda: (wide, lambda t: t),
        "slice_off_alignment": lambda: (wide, lambda t: t[:, 3:3 + cols]),
        "column_stride": lambda: (wide[:, :cols].t().contiguous(), lambda t: t.t()),
        "rows_overlap": lambda: (wide[:1, :cols].contiguous(), lambda t: t.expand(B * S, cols)),
        "one_row": lambda: (wide[:1, :cols].contiguous(), lambda t: t.as_strided((1, cols), (1, 1))),
    }[layout]()
    if layout == "one_row":
        B, S = 1, 1
    _, wq, wk, rope = _inputs(1, S, H, H, D, D, dt)
    dout = seeded((B * S, cols), 5, dtype=dt)
    base.requires_grad_(True)
    out = Q.qk_norm_rope(view(base), wq, wk, rope, B, S, H, D, EPS)
    (got,) = torch.autograd.grad(out, base, dout)
    flat = view(base.detach())[:, :cols].clone(memory_format=torch.contiguous_format).requires_grad_(True)
    ref = Q.qk_norm_rope(flat, wq, wk, rope, B, S, H, D, EPS)
    assert torch.equal(out, ref)
    (dflat,) = torch.autograd.grad(ref, flat, dout)
    leaf = base.detach().requires_grad_(True)
    (want,) = torch.autograd.grad(view(leaf)[:, :cols], leaf, dflat)
    assert torch.equal(got, want)


def test_positions_outside_the_table():
    """NaN in the rotated columns of their own token's query and key heads, and nowhere else."""
    log("qk_norm_rope positions outside the table")
    B, S, H, KH, D, R = 1, 6, 4, 2, 64, 32
    qkv, wq, wk, rope = _inputs(B, S, H, KH, D, R, torch.float32, length=50)
    pos = torch.tensor([0, -1, 49, 50, 1 << 40, 7], device="cuda")
    good = torch.where((pos >= 0) & (pos < 50), pos, 0)
    out = Q.qk_norm_rope(qkv, wq, wk, rope, B, S, H, D, EPS, kv_heads=KH, positions=pos)
    ref = Q.qk_norm_rope(qkv, wq, wk, rope, B, S, H, D, EPS, kv_heads=KH, positions=good)
    bad = torch.zeros(S, H + 2 * KH, D, dtype=torch.bool, device="cuda")
    bad[(pos < 0) | (pos >= 50), :H + KH, :R] = True
    bad = bad.view(S, -1)
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], ref[~bad])


def test_zero_rows_infinities_and_nan():
    """A head of zeros stays zero (eps keeps its root finite) and has the gradient w dz / sqrt(eps); an infinity
    or NaN stays in its own head."""
    log("qk_norm_rope zeros, infinities, NaN")
    B, S, H, D = 1, 3, 4, 64
    qkv, wq, wk, rope = _inputs(B, S, H, H, D, D, torch.float32)
    clean = Q.qk_norm_rope(qkv, wq, wk, rope, B, S, H, D, EPS)
    x = qkv.clone()
    heads = x.view(S, 3 * H, D)
    heads[0, 1], heads[1, 2, 5], heads[2, 5, 7] = 0, float("inf"), float("nan")
    dout = seeded(x.shape, 4, dtype=torch.float32)
    leaf = x.requires_grad_(True)
    out = Q.qk_norm_rope(leaf, wq, wk, rope, B, S, H, D, EPS)
    (dx,) = torch.autograd.grad(out, leaf, dout)
    touched = torch.zeros(S, 3 * H, dtype=torch.bool, device="cuda")
    touched[0, 1] = touched[1, 2] = touched[2, 5] = True
    o, c = out.detach().view(S, 3 * H, D), clean.view(S, 3 * H, D)
    assert torch.equal(o[~touched], c[~touched])
    assert (o[0, 1] == 0).all() and torch.isfinite(dx.view(S, 3 * H, D)[0, 1]).all()
    assert torch.isnan(o[1, 2]).any() and torch.isnan(o[2, 5]).any()
    assert torch.isfinite(dx.view(S, 3 * H, D)[~touched]).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=lambda d: str(d).split(".")[-1])
@pytest.mark.parametrize("size", [1e-16, 1e16])
def test_small_and_large_heads(size, dt):
    """Heads whose squares still fit fp32, though the cube of their norm does not."""
    log(f"qk_norm_rope heads of {size} {dt}")
    B, S, H, D = 1, 5, 3, 64
    qkv, wq, wk, rope = _inputs(B, S, H, H, D, D, dt)
    leaves = [t.requires_grad_(True) for t in (qkv * size, wq, wk)]
    dout = seeded(qkv.shape, 9, dtype=dt)
    out = Q.qk_norm_rope(*leaves, rope, B, S, H, D, 1e-36)
    grads = torch.autograd.grad(out, leaves, dout)
    _verify(out, grads, dout, *leaves, rope, torch.arange(S), H, H, D, False, dt, 1e-36)


def test_empty_batch():
    log("qk_norm_rope empty batch")
    qkv, wq, wk, rope = _inputs(0, 5, 2, 2, 64, 64, torch.bfloat16, length=5)
    leaves = [t.requires_grad_(True) for t in (qkv, wq, wk)]
    out = Q.qk_norm_rope(*leaves, rope, 0, 5, 2, 64, EPS)
    grads = torch.autograd.grad(out, leaves, torch.empty_like(out))
    assert out.shape == (0, 384) and grads[0].shape == (0, 384)
    assert all((g == 0).all() for g in grads[1:])


def test_rows_past_two_to_the_31():
    """More elements than 31 bits count: the last rows are those of a call on them alone."""
    H, D = 16, 128
    tokens = (1 << 31) // (3 * H * D) + 70
    log(f"qk_norm_rope tokens {tokens}")
    tail = seeded((64, 3 * H * D), 1)
    qkv = torch.zeros(tokens, 3 * H * D, device="cuda", dtype=torch.bfloat16)
    qkv[-64:] = tail
    _, wq, wk, rope = _inputs(1, 64, H, H, D, D, torch.bfloat16, length=64)
    pos = torch.arange(tokens, device="cuda") % 64
    leaf = qkv.requires_grad_(True)
    out = Q.qk_norm_rope(leaf, wq, wk, rope, tokens, 1, H, D, EPS, positions=pos)
    small = tail.requires_grad_(True)
    ref = Q.qk_norm_rope(small, wq, wk, rope, 64, 1, H, D, EPS, positions=pos[-64:])
    assert torch.equal(out[-64:], ref)
    dout = torch.zeros_like(out)
    dout[-64:] = seeded(ref.shape, 2)
    (dx,) = torch.autograd.grad(out, leaf, dout)
    (ds,) = torch.autograd.grad(ref, small, dout[-64:].contiguous())
    assert torch.equal(dx[-64:], ds) and not dx[:64].any()


@pytest.mark.parametrize("dt", DTYPES, ids=lambda d: str(d).split(".")[-1])
def test_graph_replay_matches_eager(dt):
    log(f"qk_norm_rope graph replay {dt}")
    B, S, H, D = 2, 100, 4, 72
    qkv, wq, wk, rope = _inputs(B, S, H, H, D, D, dt)
    other = seeded((64, 256), 6)
    _replay_matches(lambda *t: Q.qk_norm_rope(*t, rope, B, S, H, D, EPS), [qkv, wq, wk], seeded(qkv.shape, 5, dtype=dt),
                    lambda: other.float().square().sum(1))


def test_launches_go_to_the_current_stream():
    log("qk_norm_rope on a side stream")
    B, S, H, D = 1, 64, 4, 64
    qkv, wq, wk, rope = _inputs(B, S, H, H, D, D, torch.bfloat16)
    ref = Q.qk_norm_rope(qkv * 2, wq, wk, rope, B, S, H, D, EPS)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = qkv * 2
        out = Q.qk_norm_rope(x, wq, wk, rope, B, S, H, D, EPS)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)


def test_selftest_protocol_and_compile():
    log("selftest_autograd qk_norm_rope + torch.compile(fullgraph)")
    torch.manual_seed(0)
    B, S, H, KH, D = 2, 64, 4, 2, 64
    qkv, wq, wk, rope = _inputs(B, S, H, KH, D, 32, torch.bfloat16)
    for kw in ({}, {"positions": torch.arange(B * S, device="cuda") % 40, "interleaved": True}):
        res = selftest_autograd(lambda *t: Q.qk_norm_rope(*t, rope, B, S, H, D, EPS, kv_heads=KH, **kw),
                                lambda *t: Q.reference(*t, rope, B, S, H, D, EPS, kv_heads=KH, **kw), [qkv, wq, wk],
                                time=False)
        assert res["pass"], res["checks"]
        assert res["compiled"].get("pass"), res["compiled"]


def test_refusals():
    log("qk_norm_rope refusals")
    B, S, H, D = 2, 5, 2, 64
    qkv, wq, wk, rope = _inputs(B, S, H, H, D, D, torch.bfloat16)
    ok = dict(qkv=qkv, q_weight=wq, k_weight=wk, rope=rope, B=B, S=S, H=H, D=D, eps=EPS)
    Q.qk_norm_rope(**ok)
    pos = torch.zeros(B * S, device="cuda", dtype=torch.int64)
    for error, change in [
            (ValueError, dict(qkv=qkv.cpu())), (TypeError, dict(qkv=qkv.double())), (ValueError, dict(qkv=qkv[:9])),
            (ValueError, dict(qkv=qkv[:, 1:])), (ValueError, dict(qkv=qkv[0])), (TypeError, dict(q_weight=wq.float())),
            (ValueError, dict(k_weight=wk[:32])), (TypeError, dict(rope=rope.half())), (ValueError, dict(rope=rope[:4])),
            (ValueError, dict(rope=rope[:, :63])), (ValueError, dict(rope=torch.ones(5, 66, device="cuda"))),
            (ValueError, dict(rope=rope.clone().requires_grad_(True))), (ValueError, dict(D=60)),
            (ValueError, dict(kv_heads=0)), (ValueError, dict(kv_heads=3)), (ValueError, dict(positions=pos[1:])),
            (TypeError, dict(positions=pos.float())), (ValueError, dict(positions=pos.cpu())),
            (RuntimeError, dict(eps=float("nan")))]:
        with pytest.raises(error):
            Q.qk_norm_rope(**{**ok, **change})
