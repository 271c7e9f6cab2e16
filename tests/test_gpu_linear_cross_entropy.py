"""linear_cross_entropy (the loss of an output projection whose logits are not kept) on the GPU against its
definition in 64 bits.

Tolerances, derived. u = 2^-24 is fp32's half step, h = finfo.eps / 2 that of the activation type.
A logit adds K exact products in fp32: off by at most a = K u max_v sum |x||w|. lse and the target's logit each
carry that; the sum of exponentials adds at most 34 + V / 1024 of them one after another; exp and log take
arguments and give results of a few half steps of |lse| and 1. So the loss is off by
  e = 2 a + (64 + V / 1024 + 8 |lse|) u,  and a probability by e of itself.
dl is off by e g p + h |dl| (its rounding; in fp16 also half a step of its subnormals, 2^-25 at a scale where
the largest |g| is at 2^14 or more). A gradient adds V (or rows) products in fp32 and is rounded once."""
import pytest
import torch

import _hip
import krsi_oracle as O
import linear_cross_entropy as L
from _harness import selftest_autograd
from krsi_testutil import log, seeded
from test_gpu_graphs import _replay_matches

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def _inputs(rows, K, V, dt, seed=0, lean=6.0):
    w = (seeded((V, K), seed, dtype=torch.float32) / K ** 0.5).to(dt)
    g = torch.Generator().manual_seed(seed + 1)
    targets = torch.randint(0, V, (rows,), generator=g).cuda()
    x = seeded((rows, K), seed + 2, dtype=torch.float32) + lean * torch.rand(rows, 1, generator=g).cuda() * w[targets].float()
    return x.to(dt), w, targets


def _within(name, got, ref, bound):
    off = (got.double().to(ref.device) - ref).abs()
    log(f"{name}: worst {(off / bound.clamp_min(1e-300)).max().item() if ref.numel() else 0:.3f} of its bound")
    assert got.shape == ref.shape and bool((off <= bound).all()), (name, (off - bound).max().item())


def _verify(out, dx, dw, x, w, targets, dout, ignore=-100, reduction="mean", device="cpu"):
    dt, (rows, K), V = x.dtype, x.shape, w.shape[0]
    r = O.linear_cross_entropy_64(*(t.detach().to(device) for t in (x, w, targets, dout)), ignore, reduction)
    e = 2 * K * STEP * r["terms"] + (64 + V / 1024 + 8 * r["lse"].abs()) * STEP
    loss_bound = e if reduction == "none" else (
        e[targets.to(device) != ignore].sum() * r["share"] + 2 * STEP * r["loss"].abs())
    _within("loss", out.detach(), r["loss"], loss_bound)
    h, least = torch.finfo(dt).eps / 2, 0.0
    if dt == torch.float16:
        least = 2.0 ** -25 * float(r["g"].abs().max()) / 2.0 ** 14
    worst_p = float(e.max())
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0  # half a step of the result's own subnormals
    if dx is not None:
        _within("dx", dx, r["dx"], h * r["dx"].abs() + (h + (V + 2) * STEP) * r["dx_mag"] * (1 + h) + worst_p * r["dx_p"]
                + least * w.detach().to(device).double().abs().sum(0) + sub)
    if dw is not None:
        _within("dw", dw, r["dw"], h * r["dw"].abs() + (h + (rows + 2) * STEP) * r["dw_mag"] * (1 + h)
                + worst_p * r["dw_p"] + least * x.detach().to(device).double().abs().sum(0) + sub)


CASES = [  # rows, K, V
    (1, 64, 1), (1, 64, 2), (3, 64, 7), (17, 128, 129), (130, 64, 257), (300, 256, 5003), (257, 192, 300),
    (1000, 64, 1000), (513, 1152, 2000), (2049, 128, 777), (64, 512, 40001),
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("rows,K,V", CASES)
def test_against_64_bits(rows, K, V, reduction, dt):
    log(f"linear_cross_entropy x[{rows},{K}] w[{V},{K}] {reduction} {dt}")
    x, w, targets = _inputs(rows, K, V, dt)
    targets[3::7] = -100
    dout = seeded((rows,), 5, dtype=torch.float32) if reduction == "none" else torch.tensor(3.0, device="cuda")
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = L.linear_cross_entropy(*leaves, targets, reduction=reduction)
    dx, dw = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    _verify(out, dx, dw, x, w, targets, dout, reduction=reduction)
    assert not dx[3::7].any()
    again = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])  # bitwise reproducible
    other = L.linear_cross_entropy(*leaves, targets.int(), reduction=reduction)
    assert torch.equal(out, other)
    # One gradient alone is bitwise the same.
    assert torch.equal(torch.autograd.grad(out, leaves[0], dout, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(out, leaves[1], dout)[0], dw)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
def test_pieces_of_the_vocabulary(dt):
    """More rows x V than one piece of the backward holds (the oracle on the GPU, in torch's float64)."""
    rows, K, V = 66000, 64, 4100
    log(f"linear_cross_entropy in pieces x[{rows},{K}] w[{V},{K}] {dt}")
    x, w, targets = _inputs(rows, K, V, dt)
    dout = torch.tensor(1024.0, device="cuda")
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = L.linear_cross_entropy(*leaves, targets)
    _verify(out, *torch.autograd.grad(out, leaves, dout), x, w, targets, dout, device="cuda")


def test_rows_in_chunks():
    """More rows than the forward keeps pairs of at a time: the rows' losses are those of the chunks alone."""
    rows, K, V = 4300, 64, 1 << 20
    log(f"linear_cross_entropy in chunks of rows x[{rows},{K}] w[{V},{K}]")
    x, w, targets = _inputs(rows, K, V, torch.bfloat16)
    targets[[5, 4200]] = -100
    with torch.no_grad():
        out = L.linear_cross_entropy(x, w, targets, reduction="none")
        parts = [L.linear_cross_entropy(x[a:b], w, targets[a:b], reduction="none") for a, b in ((0, 4096), (4096, rows))]
        assert torch.equal(out, torch.cat(parts))
        some = torch.arange(0, rows, 173, device="cuda")
        ref = torch.nn.functional.cross_entropy(x[some].double() @ w.double().t(), targets[some], reduction="none")
        assert ((out[some].double() - ref).abs() < 2e-4).all()  # 2 K u 10 + (64 + V / 1024 + 8 * 14) u = 1.5e-4


def test_gradient_scales_exactly():
    """dout times a power of two: the gradients times that power, bitwise (dl's own scale is one too)."""
    log("linear_cross_entropy gradient scale")
    x, w, targets = _inputs(100, 128, 500, torch.bfloat16)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    out = L.linear_cross_entropy(*leaves, targets)
    one = torch.autograd.grad(out, leaves, torch.tensor(1.0, device="cuda"), retain_graph=True)
    for k in (-20, 3, 40):
        got = torch.autograd.grad(out, leaves, torch.tensor(2.0 ** k, device="cuda"), retain_graph=True)
        assert all(torch.equal(a, b * 2.0 ** k) for a, b in zip(got, one))
    zero = torch.autograd.grad(out, leaves, torch.tensor(0.0, device="cuda"))
    assert not any(t.any() for t in zero)


def test_ignored_and_bad_targets():
    """All ignored: mean NaN, sum 0, gradients zero. A target outside [0, V): its loss and dx row NaN, dw NaN."""
    log("linear_cross_entropy ignored and bad targets")
    x, w, targets = _inputs(40, 64, 100, torch.bfloat16)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    none = torch.full_like(targets, 7)
    for reduction in ("mean", "sum"):
        out = L.linear_cross_entropy(*leaves, none, ignore_index=7, reduction=reduction)
        assert bool(torch.isnan(out)) if reduction == "mean" else out.item() == 0
        assert not any(g.any() for g in torch.autograd.grad(out, leaves))
    good = L.linear_cross_entropy(*leaves, targets, reduction="none")
    (dgood,) = torch.autograd.grad(good.sum(), leaves[0])
    for bad in (-1, 100, -100, 1 << 40):
        t = targets.clone()
        t[5] = bad
        out = L.linear_cross_entropy(*leaves, t, ignore_index=-7, reduction="none")
        dx, dw = torch.autograd.grad(out.sum(), leaves)
        rest = torch.arange(40, device="cuda") != 5
        assert torch.isnan(out[5]) and torch.equal(out[rest], good[rest])
        assert torch.isnan(dx[5]).all() and torch.equal(dx[rest], dgood[rest]) and torch.isnan(dw).all()


def test_large_logits_infinities_and_nan():
    """Logits whose exponentials overflow are exact to the bound; NaN or an infinity in a row stays in it."""
    log("linear_cross_entropy large logits, infinities, NaN")
    x, w, targets = _inputs(50, 128, 300, torch.bfloat16)
    big = (x.float() * 500).to(torch.bfloat16)
    leaves = [big.requires_grad_(True), w.requires_grad_(True)]
    out = L.linear_cross_entropy(*leaves, targets, reduction="none")
    dout = seeded((50,), 4, dtype=torch.float32)
    _verify(out, None, None, big, w, targets, dout, reduction="none")
    odd = x.clone()
    odd[3, 5], odd[4, 6] = float("nan"), float("inf")
    leaf = odd.requires_grad_(True)
    out = L.linear_cross_entropy(leaf, w, targets, reduction="none")
    clean = x.detach().requires_grad_(True)
    ref = L.linear_cross_entropy(clean, w, targets, reduction="none")
    rest = torch.ones(50, dtype=torch.bool, device="cuda")
    rest[3:5] = False
    assert torch.isnan(out[3:5]).all() and torch.equal(out[rest], ref[rest])
    # With no weight on those rows: ignored rows have no gradient whatever they hold.
    t = torch.where(rest, targets, -100)
    dx, dw = torch.autograd.grad(L.linear_cross_entropy(leaf, w, t, reduction="sum"), [leaf, w])
    assert not dx[~rest].any() and torch.isfinite(dx).all()


def test_shapes_and_layouts():
    """Leading dimensions; strided and unaligned x, w and targets give what their contiguous copies give."""
    log("linear_cross_entropy shapes and layouts")
    x, w, targets = _inputs(24, 64, 90, torch.bfloat16)
    ref = L.linear_cross_entropy(x, w, targets, reduction="none")
    shaped = L.linear_cross_entropy(x.view(2, 3, 4, 64), w, targets.view(2, 3, 4), reduction="none")
    assert shaped.shape == (2, 3, 4) and torch.equal(shaped.flatten(), ref)
    one = L.linear_cross_entropy(x[0], w, targets[0], reduction="none")
    assert one.shape == () and torch.equal(one, ref[0])
    off = torch.empty(24 * 64 + 1, device="cuda", dtype=x.dtype)[1:].view(24, 64).copy_(x)
    leaf = x.t().contiguous().t().detach().requires_grad_(True)
    ws = torch.stack([w, w], 1)[:, 0]
    for a, b, t in ((leaf, w, targets), (off, w, targets), (x, ws, targets), (x, w, torch.stack([targets] * 2, 1)[:, 1])):
        assert torch.equal(L.linear_cross_entropy(a, b, t, reduction="none"), ref)
    flat = x.detach().requires_grad_(True)
    grads = [torch.autograd.grad(L.linear_cross_entropy(a, w, targets), a)[0] for a in (leaf, flat)]
    assert torch.equal(*grads)


def test_no_rows():
    log("linear_cross_entropy no rows")
    x, w, targets = _inputs(0, 64, 90, torch.float16)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    for reduction in ("mean", "sum", "none"):
        out = L.linear_cross_entropy(*leaves, targets, reduction=reduction)
        dx, dw = torch.autograd.grad(out, leaves, torch.ones_like(out))
        assert dx.shape == (0, 64) and not dw.any()
        assert {"mean": bool(torch.isnan(out).all()), "sum": not out.any(), "none": out.shape == (0,)}[reduction]


@pytest.mark.parametrize("rows,K,V", [(200, 128, 1000), (30, 64, 70)])
def test_graph_replay_matches_eager(rows, K, V):
    log(f"linear_cross_entropy graph replay x[{rows},{K}] w[{V},{K}]")
    x, w, targets = _inputs(rows, K, V, torch.bfloat16)
    other = seeded((64, 256), 6)
    _replay_matches(lambda a, b: L.linear_cross_entropy(a, b, targets), [x, w], torch.tensor(2.0, device="cuda"),
                    lambda: other.float().square().sum(1))


def test_selftest_protocol_and_compile():
    log("selftest_autograd linear_cross_entropy + torch.compile(fullgraph)")
    torch.manual_seed(0)
    x, w, targets = _inputs(200, 128, 1000, torch.bfloat16)
    for reduction in ("none", "mean"):
        res = selftest_autograd(lambda a, b: L.linear_cross_entropy(a, b, targets, reduction=reduction),
                                lambda a, b: L.reference(a, b, targets, reduction=reduction), [x, w], time=False)
        assert res["pass"], res["checks"]
        assert res["compiled"].get("pass"), res["compiled"]


def test_refusals():
    log("linear_cross_entropy refusals")
    x, w, targets = _inputs(8, 64, 20, torch.bfloat16)
    for error, args, kw in [
            (ValueError, (x.cpu(), w, targets), {}), (TypeError, (x.float(), w.float(), targets), {}),
            (TypeError, (x, w.half(), targets), {}), (TypeError, (x, w, targets.float()), {}),
            (ValueError, (x, w[:, :32], targets), {}), (ValueError, (x[:, :32], w[:, :32], targets), {}),
            (ValueError, (x, w, targets[1:]), {}), (ValueError, (x[None], w, targets), {}),
            (ValueError, (x, w[:0], targets), {}), (ValueError, (x, w, targets), {"reduction": "max"})]:
        with pytest.raises(error):
            L.linear_cross_entropy(*args, **kw)


def test_saved_statistics_are_checked():
    log("linear_cross_entropy backward refusals")
    x, w, targets = _inputs(8, 64, 20, torch.bfloat16)
    loss, stats = _hip.linear_cross_entropy_fwd(x, w, targets, -100, "mean")
    for dout, s in ((loss.double(), stats), (loss.expand(8), stats), (loss, stats[1:]), (loss, stats.double())):
        with pytest.raises(ValueError):
            _hip.linear_cross_entropy_bwd(dout, x, w, targets, s, -100, "mean")
