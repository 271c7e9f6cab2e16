"""add_rmsnorm and its 8-bit form on the GPU against the formulas in 64 bits.

Tolerances: with u half a step of the type relative to the value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32) and e a few
roundings in 32 bits (sums over a tree of 16384: 64 * 2^-24 covers it), r is off by u |r|, y by u |y| and the gradients by u
of theirs; e of the sizes of the terms that are added, which may cancel, comes on top.
"""
import pytest
import torch

import _hip
import add_rmsnorm as A
import rmsnorm as R
from krsi_testutil import log, seeded

pytestmark = pytest.mark.gpu
EPS = 1e-6
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E32 = 64 * 2.0 ** -24
ids = lambda d: str(d).split(".")[-1]  # noqa: E731

SHAPES = [(1, 1), (3, 5), (70, 7), (2, 8), (5, 64), (9, 65), (64, 72), (33, 1001), (4, 1024), (7, 1032), (130, 2048),
          (3, 2049), (6, 4096), (5, 4104), (3, 8191), (4, 8192), (2, 8200), (2, 12288), (3, 16381), (3, 16384),
          (2100, 40)]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _close(got, want, bound, what):
    bad = (got.double() - want).abs() > bound + 1e-300
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / (bound + 1e-300)).max()))


def _inputs(rows, n, dt):
    return (seeded((rows, n), 1, dtype=dt), seeded((rows, n), 2, std=2.0, dtype=dt),
            seeded((n,), 3, std=0.1, mean=1.0, dtype=dt))


def _verify(leaves, y, r, grads, dy, dr, dt, eps=EPS):
    x, res, w = (t.detach().double() for t in leaves)
    n, u = x.shape[1], _u(dt)
    # fp16's subnormals: half their step on top of the relative rounding.
    tiny = torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    _close(r, x + res, u * (x + res).abs() + tiny, "r")
    rr = r.detach().double()
    nrm = rr * torch.rsqrt(rr.square().mean(1, keepdim=True) + eps)
    _close(y, nrm * w, (u + E32) * (nrm * w).abs() + tiny, "y")
    if grads is None:
        return
    g = torch.zeros_like(x) if dy is None else dy.double()
    s = torch.zeros_like(x) if dr is None else dr.double()
    rstd = torch.rsqrt(rr.square().mean(1, keepdim=True) + eps)
    dn = g * w
    d = s + rstd * (dn - nrm * (dn * nrm).mean(1, keepdim=True))
    spread = (dn.abs() + nrm.abs() * (dn * nrm).abs().mean(1, keepdim=True)) * rstd
    bound = u * d.abs() + E32 * (spread + s.abs()) + tiny
    _close(grads[0], d, bound, "dx")
    assert torch.equal(grads[0], grads[1])
    terms = (g * nrm).abs().sum(0)
    _close(grads[2], (g * nrm).sum(0), u * (g * nrm).sum(0).abs() + E32 * terms + tiny, "dw")


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_against_64_bits(rows, n, dt):
    log(f"add_rmsnorm [{rows}, {n}] {dt}")
    leaves = [t.requires_grad_(True) for t in _inputs(rows, n, dt)]
    dy, dr = seeded((rows, n), 4, dtype=dt), seeded((rows, n), 5, dtype=dt)
    y, r = A.add_rmsnorm(*leaves, EPS)
    grads = torch.autograd.grad([y, r], leaves, [dy, dr], retain_graph=True)
    _verify(leaves, y, r, grads, dy, dr, dt)
    again = torch.autograd.grad([y, r], leaves, [dy, dr], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    # The norm alone used: no gradient of the stream.
    _verify(leaves, y, r, torch.autograd.grad(y, leaves, dy, retain_graph=True), dy, None, dt)
    only = torch.autograd.grad(r, leaves[:2], dr)
    assert torch.equal(only[0], dr) and torch.equal(only[1], dr)
    with torch.no_grad():
        y2, r2 = A.add_rmsnorm(*leaves, EPS)
    assert torch.equal(y, y2) and torch.equal(r, r2)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,n", [(6, 64), (5, 1001), (9, 4096), (3, 8191)])
def test_as_the_norm_of_the_sum(rows, n, dt):
    """What rmsnorm gives for the sum, which rounds twice where this rounds once: three half steps apart at most."""
    log(f"add_rmsnorm as rmsnorm(x + residual) [{rows}, {n}] {dt}")
    x, res, w = _inputs(rows, n, dt)
    y, r = A.add_rmsnorm(x, res, w, EPS)
    assert torch.equal(r, x + res)
    want = R.rmsnorm(x + res, w, EPS).double()
    _close(y, want, (3 * _u(dt) * (1 + _u(dt)) + E32) * want.abs() + 2 * torch.finfo(dt).tiny * torch.finfo(dt).eps, "y")


def _codes(z):
    """Codes (as their values) and scales of rows in 64 bits: scale as the kernel's, codes before their rounding."""
    scale = (z.abs().amax(1) / 448).clamp(min=2.0 ** -120)
    return z / scale[:, None], scale


def _verify_codes(q, scale, z):
    """z within half a step of e4m3 (2^-4 relative, 2^-10 below its normal range) of the codes' values, and 32-bit
    roundings of z, its scale and its reciprocal."""
    want, s = _codes(z)
    _close(scale, s, E32 * s, "scale")
    err = (q.double() - want).abs()
    bound = torch.maximum(want.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10, device="cuda")) * (1 + 1e-4) + E32 * want.abs()
    assert (err <= bound).all(), float((err / bound).max())
    assert (q.double().abs().amax(1) <= 448).all()


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows,n", SHAPES)
def test_8bit_against_64_bits(rows, n, dt):
    log(f"add_rmsnorm_8bit [{rows}, {n}] {dt}")
    x, res, w = _inputs(rows, n, dt)
    q, scale, r = A.add_rmsnorm_8bit(x, res, w, EPS)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows,)
    assert torch.equal(r, x + res)

    def norm(t):
        t = t.double()
        return t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * w.double()

    _verify_codes(q, scale, norm(r))
    assert (q.double().abs().amax(1) == 448).all()
    q, scale, same = A.add_rmsnorm_8bit(x, None, w, EPS)
    assert same is x
    _verify_codes(q, scale, norm(x))
    q, scale = _hip.quantize_rows(x)
    _verify_codes(q, scale, x.double())


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_quantize_long_rows(dt):
    for rows, n in ((2, 16392), (1, 32768), (2, 40000), (1, 65536), (2, 65543), (1, 200001)):
        log(f"quantize_rows [{rows}, {n}] {dt}")
        x = seeded((rows, n), 1, dtype=dt)
        q, scale = _hip.quantize_rows(x)
        _verify_codes(q, scale, x.double())


def test_8bit_rounding_is_to_nearest_even():
    """Every pair of neighbouring codes: values between them go to the nearer one, a tie to the even code."""
    log("quantize_rows rounding")
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()  # 0 .. 448
    lo, hi = codes[:-1], codes[1:]
    mid = (lo + hi) / 2
    below, above = torch.nextafter(mid, lo), torch.nextafter(mid, hi)
    even = torch.where(torch.arange(126) % 2 == 0, lo, hi)
    x = torch.stack([torch.cat([t, torch.tensor([448.0])]) for t in (lo, hi, below, above, mid)])
    want = torch.stack([torch.cat([t, torch.tensor([448.0])]) for t in (lo, hi, lo, hi, even)])
    for sign in (1, -1):
        q, scale = _hip.quantize_rows((sign * x).cuda())
        assert torch.equal(scale.cpu(), torch.ones(5)) and torch.equal(q.float().cpu(), sign * want)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("n", [40, 1024, 1001, 4096, 20000])
def test_8bit_zero_infinite_nan_rows(n, dt):
    """A row of zeros reads back as zeros; one with an infinity or NaN as NaN throughout; others are untouched."""
    log(f"8 bit: zero, infinite and NaN rows n={n} {dt}")
    x = seeded((6, n), 1, dtype=dt)
    clean = x.clone()
    x[1], x[2, n - 1], x[3, 0], x[4, n // 2] = 0, float("inf"), float("nan"), float("-inf")
    res, w = torch.zeros_like(x), torch.ones(n, device="cuda", dtype=dt)
    calls = [lambda t: _hip.quantize_rows(t)]
    if n <= 16384:
        calls += [lambda t: A.add_rmsnorm_8bit(t, None, w, EPS)[:2], lambda t: A.add_rmsnorm_8bit(t, res, w, EPS)[:2]]
    for call in calls:
        q, s = call(x)
        back, want = q.float() * s[:, None], call(clean)
        assert (back[1] == 0).all() and torch.isnan(back[2:5]).all()
        for i in (0, 5):
            assert torch.equal(q[i].float(), want[0][i].float()) and s[i] == want[1][i]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("size", [1e-16, 1e16])
def test_small_and_large_rows(size, dt):
    """Rows whose squares still fit fp32, though the cube of their reciprocal root does not."""
    log(f"add_rmsnorm rows of {size} {dt}")
    x, res, w = _inputs(5, 200, dt)
    leaves = [(t * size).to(dt).requires_grad_(True) for t in (x, res)] + [w.requires_grad_(True)]
    dy = seeded((5, 200), 4, dtype=dt)
    y, r = A.add_rmsnorm(*leaves, 1e-36)
    _verify(leaves, y, r, torch.autograd.grad(y, leaves, dy), dy, None, dt, 1e-36)


def test_zero_rows_keep_a_finite_gradient():
    log("add_rmsnorm zero rows")
    x = torch.zeros(3, 40, device="cuda", requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    y, r = A.add_rmsnorm(x, torch.zeros_like(x), w, EPS)
    dy = seeded((3, 40), 4, dtype=torch.float32)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    assert not y.any() and not r.any() and not dw.any()
    assert torch.allclose(dx, dy * 1000, rtol=1e-6, atol=0)


def test_gradients_against_differences():
    """Central differences of a sum over both outputs, in fp32 inputs' 64-bit formula steps of 2^-7: off by the third
    derivative's share, below 2^-14 of the terms here, and fp32's roundings over the step."""
    log("add_rmsnorm against differences")
    x, res, w = (t.requires_grad_(True) for t in _inputs(3, 24, torch.float32))
    dy, dr = seeded((3, 24), 4, dtype=torch.float32), seeded((3, 24), 5, dtype=torch.float32)
    y, r = A.add_rmsnorm(x, res, w, EPS)
    grads = torch.autograd.grad([y, r], [x, res, w], [dy, dr])

    def value(x, res, w):
        y, r = A.add_rmsnorm(x, res, w, EPS)
        return float((y.double() * dy.double()).sum() + (r.double() * dr.double()).sum())

    h = 2.0 ** -7
    for which in range(3):
        for at in (0, 11, 23):
            up, down = ([t.detach().clone() for t in (x, res, w)] for _ in range(2))
            up[which].view(-1)[at] += h
            down[which].view(-1)[at] -= h
            slope = (value(*up) - value(*down)) / (2 * h)
            # 144 terms rounded by 2^-24 each, of sizes up to 6, over 2 h; h^2 / 6 times third derivatives below 50.
            assert abs(slope - float(grads[which].view(-1)[at])) < 144 * 6 * 2.0 ** -24 / h + h * h / 6 * 50


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_off_alignment(dt):
    """Tensors that start off any 16-byte boundary, of a length that whole chunks would fit."""
    log(f"add_rmsnorm off alignment {dt}")
    rows, n = 7, 256
    views = []
    for i, t in enumerate((*_inputs(rows, n, dt), seeded((rows, n), 4, dtype=dt), seeded((rows, n), 5, dtype=dt))):
        flat = torch.empty(t.numel() + 8, device="cuda", dtype=dt)
        view = flat[1 + i:1 + i + t.numel()].view(t.shape)
        views.append(view.copy_(t))
    leaves = [t.detach().requires_grad_(True) for t in views[:3]]
    y, r = A.add_rmsnorm(*leaves, EPS)
    grads = torch.autograd.grad([y, r], leaves, views[3:])
    _verify(leaves, y, r, grads, *views[3:], dt)
    q, s, r2 = A.add_rmsnorm_8bit(*(t.detach() for t in leaves), EPS)
    qa, sa, ra = A.add_rmsnorm_8bit(*(t.detach().clone() for t in leaves), EPS)
    assert torch.equal(r2, ra) and torch.allclose(s, sa, rtol=1e-6) and (q.float() - qa.float()).abs().max() <= 32


def test_empty_batch():
    log("add_rmsnorm empty batch")
    x, res = (torch.empty(0, 96, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    w = torch.ones(96, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y, r = A.add_rmsnorm(x, res, w, EPS)
    dx, dres, dw = torch.autograd.grad([y, r], [x, res, w], [torch.empty_like(y), torch.empty_like(r)])
    assert y.shape == r.shape == dx.shape == dres.shape == (0, 96) and not dw.any()
    with torch.no_grad():
        q, s, r = A.add_rmsnorm_8bit(x, res, w, EPS)
    assert q.shape == (0, 96) and s.shape == (0,) and r.shape == (0, 96)


def test_rows_past_two_to_the_31():
    """More elements than 31 bits count: the last rows are those of a call on them alone."""
    n = 4096
    rows = (1 << 31) // n + 70
    log(f"add_rmsnorm rows {rows}")
    tail, tres = seeded((64, n), 1), seeded((64, n), 2)
    w = seeded((n,), 3, std=0.1, mean=1.0).requires_grad_(True)
    x, res = (torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    x[-64:], res[-64:] = tail, tres
    leaf = x.requires_grad_(True)
    y, r = A.add_rmsnorm(leaf, res, w, EPS)
    small = tail.requires_grad_(True)
    ys, rs = A.add_rmsnorm(small, tres, w, EPS)
    assert torch.equal(y[-64:], ys) and torch.equal(r[-64:], rs) and not y[:64].any()
    dy = torch.zeros_like(y)
    dy[-64:] = seeded((64, n), 4)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    (ds,) = torch.autograd.grad(ys, small, dy[-64:].contiguous())
    assert torch.equal(dx[-64:], ds) and not dx[:64].any()
    del dy, dx, y, r
    with torch.no_grad():
        q, s, _ = A.add_rmsnorm_8bit(leaf, res, w, EPS)
        qs, ss, _ = A.add_rmsnorm_8bit(small, tres, w, EPS)
    assert torch.equal(q[-64:].float(), qs.float()) and torch.equal(s[-64:], ss) and not q[:64].float().any()


def test_shared_leaf_and_broadcast():
    """One tensor as layer output and stream at once gets both shares; a broadcast one is refused until copied."""
    log("add_rmsnorm shared leaf, broadcast")
    x, _, w = _inputs(6, 128, torch.float32)
    x.requires_grad_(True)
    dy = seeded((6, 128), 4, dtype=torch.float32)
    y, _ = A.add_rmsnorm(x, x, w, EPS)
    (dx,) = torch.autograd.grad(y, x, dy)
    two = [x.detach().clone().requires_grad_(True) for _ in range(2)]
    y2, _ = A.add_rmsnorm(*two, w, EPS)
    da, db = torch.autograd.grad(y2, two, dy)
    assert torch.equal(y, y2) and torch.equal(dx, da + db)
    row = seeded((1, 128), 7, dtype=torch.float32).requires_grad_(True)
    with pytest.raises(ValueError, match="contiguous"):
        A.add_rmsnorm(x, row.expand(6, 128), w, EPS)
    y3, r3 = A.add_rmsnorm(x, row.expand(6, 128).contiguous(), w, EPS)
    (drow,) = torch.autograd.grad(r3, row, dy)
    assert torch.allclose(drow, dy.sum(0, keepdim=True), rtol=1e-5, atol=1e-6)


def test_accumulated_gradients_do_not_share_memory():
    """x and residual get one gradient tensor from the kernel; their .grad can be changed apart."""
    log("add_rmsnorm .grad of both inputs")
    leaves = [t.requires_grad_(True) for t in _inputs(4, 64, torch.bfloat16)]
    y, r = A.add_rmsnorm(*leaves, EPS)
    torch.autograd.backward([y, r], [torch.ones_like(y), torch.ones_like(r)])
    before = leaves[1].grad.clone()
    leaves[0].grad.zero_()
    assert torch.equal(leaves[1].grad, before) and before.any()


def test_refusals_on_the_gpu():
    log("add_rmsnorm refusals")
    x, res, w = _inputs(4, 64, torch.bfloat16)
    for args, err in [((x, res, w.float()), TypeError), ((x, res.float(), w), TypeError), ((x, res[:3], w), ValueError),
                      ((x, res, w[:63]), ValueError), ((x.t(), res, w), ValueError), ((x, res.t().contiguous().t(), w), ValueError),
                      ((x, res.cpu(), w), ValueError), ((x.double(), res.double(), w.double()), TypeError),
                      ((x[0], res[0], w), ValueError)]:
        with pytest.raises(err):
            A.add_rmsnorm(*args, EPS)
        with pytest.raises(err):
            A.add_rmsnorm_8bit(*args, EPS)
    with pytest.raises(_hip.KrsiError):
        A.add_rmsnorm(x, res, w, float("nan"))
    wide = torch.zeros(1, 16392, device="cuda")
    with pytest.raises(_hip.KrsiError):
        A.add_rmsnorm(wide, wide, wide[0], EPS)
    with pytest.raises(ValueError, match="no gradient"):
        A.add_rmsnorm_8bit(x.requires_grad_(True), res, w, EPS)
    with torch.no_grad():
        A.add_rmsnorm_8bit(x, res, w, EPS)
