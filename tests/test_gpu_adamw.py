"""adamw_step, grad_norm and AdamW on the GPU against the formulas in 64 bits.

Tolerances, e = 2^-24: m and v are two products and a sum in fp32 of values that the 64-bit formula has exactly, 4 e of
their terms' sizes (and 2 e more of the gradient through a clipped one, 4 of its square). The change of w is lr / bc1 * m / (root + eps) with a root
and a reciprocal of 1 unit each and six roundings, 16 e of it, and w's product and sum 3 e |w|; a rounding to the
parameter's type half a step more. An 8-bit state's value is a step of e4m3 off at most (2^-3 relative, 2^-9 of the scale
below the normal range)."""
import math

import pytest
import torch

import _hip
import adamw as W
from krsi_testutil import log, seeded

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ids = lambda d: str(d).split(".")[-1]  # noqa: E731
E = 2.0 ** -24
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SHAPES = [(1,), (7,), (8,), (255,), (256,), (257,), (3, 5, 2), (0,), (33, 129), (8192,), (8193,), (100, 173), (16385,)]


def _lists(shapes, dt, bits=32, masters=False, gdt=None, seed=0, grad_std=1e-2):
    """Parameters, gradients and states of some steps, and the arguments of a call."""
    w = [seeded(s, seed + 3 * i, std=0.5, dtype=torch.float32) for i, s in enumerate(shapes)]
    g = [seeded(s, seed + 100 + i, std=grad_std, dtype=torch.float32).to(gdt or dt) for i, s in enumerate(shapes)]
    m = [seeded(s, seed + 200 + i, std=grad_std / 3, dtype=torch.float32) for i, s in enumerate(shapes)]
    v = [(seeded(s, seed + 300 + i, std=grad_std, dtype=torch.float32).abs() + grad_std / 4).square()
         for i, s in enumerate(shapes)]
    steps = torch.arange(len(shapes), dtype=torch.int32, device="cuda") * 7
    kw = {"params": [t.to(dt) for t in w], "grads": g, "steps": steps}
    if masters:
        kw["masters"] = [t.clone() for t in w]
    if bits == 32:
        kw.update(exp_avgs=m, exp_avg_sqs=v)
    else:
        pairs = [(_to_blocks(a), _to_blocks(b.sqrt())) for a, b in zip(m, v)]
        kw["scales"] = [torch.stack([a[1], b[1]]) for a, b in pairs]
        kw["exp_avgs"], kw["exp_avg_sqs"] = ([p[k][0].view(s) for p, s in zip(pairs, shapes)] for k in (0, 1))
    return kw


def _to_blocks(t):
    flat = torch.nn.functional.pad(t.flatten(), (0, -t.numel() % 256)).view(-1, 256)
    scale = (flat.abs().amax(1) / 448).clamp(min=2.0 ** -120) if flat.numel() else flat.new_zeros(0)
    return (flat / scale[:, None]).to(torch.float8_e4m3fn).flatten()[:t.numel()], scale


def _spread(scale, n):
    return scale.repeat_interleave(256)[:n]


def _copy(kw):
    return {k: [t.clone() for t in v] if isinstance(v, list) else v.clone() for k, v in kw.items()}


def _values(kw, i):
    """m and v of tensor i in 64 bits."""
    m, v = kw["exp_avgs"][i].double().flatten(), kw["exp_avg_sqs"][i].double().flatten()
    if "scales" in kw:
        ms, rs = (_spread(s.double(), m.numel()) for s in kw["scales"][i])
        return m * ms, (v * rs).square()
    return m, v


def _formula(kw, i, share=1.0, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1):
    m0, v0 = _values(kw, i)
    g = kw["grads"][i].double().flatten() * share
    w = kw["masters" if "masters" in kw else "params"][i].double().flatten()
    t = int(kw["steps"][i]) + 1
    m, v = betas[0] * m0 + (1 - betas[0]) * g, betas[1] * v0 + (1 - betas[1]) * g * g
    step = lr / (1 - betas[0] ** t) * m / (v.sqrt() / math.sqrt(1 - betas[1] ** t) + eps)
    size = m0.abs() * betas[0] + (1 - betas[0]) * g.abs()  # of m's terms, which may cancel
    return w * (1 - lr * weight_decay) - step, m, v, size, w, lr / (1 - betas[0] ** t) / (v.sqrt() / math.sqrt(1 - betas[1] ** t) + eps)


def _near(got, want, bound, what):
    bad = ~((got.double().flatten() - want).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((got.double().flatten() - want).abs().max()))


def _verify(before, after, share=1.0, hyper=HYPER):
    for i, p in enumerate(after["params"]):
        if before["grads"][i] is None:
            for k in before:
                if k not in ("grads", "steps"):
                    assert torch.equal(before[k][i].view(torch.uint8), after[k][i].view(torch.uint8)), k
            assert after["steps"][i] == before["steps"][i]
            continue
        assert after["steps"][i] == before["steps"][i] + 1
        w, m, v, size, w0, rate = _formula(before, i, share, **hyper)
        bound = 4 * E * w0.abs() + rate * 32 * E * size + 1e-45
        if "masters" in after:
            _near(after["masters"][i], w, bound, "master")
            assert torch.equal(p, after["masters"][i].to(p.dtype))
        else:
            info = torch.finfo(p.dtype)
            half = 0 if p.dtype == torch.float32 else info.eps / 2
            _near(p, w, bound * 2 + half * w.abs() * (1 + E) + (info.tiny * info.eps if half else 0), "param")
        if "scales" not in after:
            _near(after["exp_avgs"][i], m, 8 * E * size + 1e-45, "m")
            _near(after["exp_avg_sqs"][i], v, 14 * E * v + 1e-45, "v")
            continue
        n = m.numel()
        for got, want, scale in ((after["exp_avgs"][i], m, after["scales"][i][0]),
                                 (after["exp_avg_sqs"][i], v.sqrt(), after["scales"][i][1])):
            flat = torch.nn.functional.pad(want, (0, -n % 256)).view(-1, 256)
            top = flat.abs().amax(1) / 448 if n else flat.new_zeros(0)
            # m's terms may cancel; over a block the largest term is within a few times the largest m here.
            assert torch.allclose(scale.double(), top.clamp(min=2.0 ** -120), rtol=64 * E, atol=0)
            s = _spread(scale.double(), n)
            q = got.double().flatten()
            x = (want / s).clamp(-448, 448) if n else want
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
            # up or down by less than a step (of the size above where x is just below a power of two)
            assert ((q - x).abs() < step * (1 + 1e-3) + 1e-12).all()
            assert (q.abs() <= 448).all()
        r = after["exp_avg_sqs"][i].double().flatten()
        assert (r[v > 0] > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt,masters,gdt", [(torch.bfloat16, True, None), (torch.bfloat16, False, None),
                                            (torch.bfloat16, True, torch.float32), (torch.bfloat16, False, torch.float32),
                                            (torch.float16, True, None), (torch.float16, False, None),
                                            (torch.float16, True, torch.float32), (torch.float16, False, torch.float32),
                                            (torch.float32, False, None)])
def test_against_64_bits(dt, masters, gdt, bits):
    log(f"adamw {dt} masters {masters} grads {gdt} bits {bits}")
    kw = _lists(SHAPES, dt, bits, masters, gdt)
    kw["grads"][4] = None
    before = {k: list(v) if k == "grads" else _copy({k: v})[k] for k, v in kw.items()}
    assert W.adamw_step(**kw, **HYPER) is None
    _verify(before, kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_launches(bits):
    """More tensors than a launch holds, some empty, some without a gradient."""
    log(f"adamw 150 tensors, {bits} bits")
    shapes = [((37 * i) % 700,) for i in range(150)]
    kw = _lists(shapes, torch.float32, bits)
    for i in range(0, 150, 11):
        kw["grads"][i] = None
    before = {k: list(v) if k == "grads" else _copy({k: v})[k] for k, v in kw.items()}
    W.adamw_step(**kw, **HYPER)
    _verify(before, kw)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_off_alignment_and_neighbours(dt, bits):
    """Tensors packed into one buffer at any offset: the same values as apart, and what lies between them stays."""
    log(f"adamw packed {dt} {bits} bits")
    apart = _lists(SHAPES, dt, bits, masters=dt != torch.float32)
    packed, guards = {"steps": apart["steps"].clone()}, []
    for k, ts in apart.items():
        if k == "steps":
            continue
        flat = torch.zeros(sum(t.numel() + 3 for t in ts) + 1, device="cuda", dtype=torch.float32).to(ts[0].dtype)
        at, views = 1, []
        for t in ts:
            views.append(flat[at:at + t.numel()].view(t.shape).copy_(t))
            at += t.numel() + 3
        packed[k] = views
        gap = torch.ones_like(flat, dtype=torch.bool)
        at = 1
        for t in ts:
            gap[at:at + t.numel()] = False
            at += t.numel() + 3
        guards.append((flat, gap))
    W.adamw_step(**apart, **HYPER, seed=5)
    W.adamw_step(**packed, **HYPER, seed=5)
    for k in apart:
        if k != "steps":
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(apart[k], packed[k])), k
    for flat, gap in guards:
        assert not flat.float()[gap].any()


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_grad_norm(dt):
    """At most 20 fp32 additions and a square on a term's way (nine squares a lane's sum, three sums of eight, a wave, a
    workgroup), then fp64: 21 times 2^-24 of the sum, half of it through the root and one rounding more; 64 is above it."""
    log(f"grad_norm {dt}")
    grads = [seeded(s, i, dtype=dt) for i, s in enumerate(SHAPES + [(65536,), (65537,), (3, 70001)])]
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    norm = W.grad_norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32 and abs(float(norm) - want) < 64 * E * want
    assert torch.equal(norm, W.grad_norm(grads)) and torch.equal(norm, W.grad_norm([None, *grads]))
    odd = torch.empty(70001 + 1, device="cuda", dtype=dt)[1:].copy_(grads[-1].flatten()[:70001])
    assert abs(float(W.grad_norm([odd])) - float(odd.double().norm())) < 64 * E * float(odd.double().norm())
    assert float(W.grad_norm([torch.empty(0, device="cuda", dtype=dt)])) == 0
    assert torch.allclose(W.grad_norm([g.t().contiguous().t() if g.dim() == 2 else g for g in grads]), norm, rtol=64 * E)


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping(bits):
    log(f"adamw clipping {bits} bits")
    for max_norm in (0.05, 1e6, 0.0):
        kw = _lists(SHAPES, torch.bfloat16, bits, masters=True)
        before = _copy(kw)
        norm = W.adamw_step(**kw, **HYPER, max_norm=max_norm)
        total = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
        assert abs(float(norm) - total) < 64 * E * total
        _verify(before, kw, min(1.0, max_norm / (float(norm) + 1e-6)))
        again = _copy(before)  # the norm given
        assert W.adamw_step(**again, **HYPER, max_norm=max_norm, norm=norm) is norm
        for k in kw:
            same = zip(kw[k], again[k]) if k != "steps" else [(kw[k], again[k])]
            assert all(torch.equal(a.float(), b.float()) for a, b in same)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_norm_that_is_not_finite_changes_nothing(bad):
    log(f"adamw norm {bad}")
    for bits in (32, 8):
        kw = _lists(SHAPES, torch.bfloat16, bits, masters=True)
        kw["grads"][5][0] = bad
        before = _copy(kw)
        assert not torch.isfinite(W.adamw_step(**kw, **HYPER, max_norm=1.0))
        for k in kw:
            same = zip(kw[k], before[k]) if k != "steps" else [(kw[k], before[k])]
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in same), k


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradient_that_is_not_finite_stays_with_its_block(bad):
    """Without a norm: its own element in 32 bits; in 8 bits its parameter, and the states of its 256 elements."""
    log(f"adamw gradient {bad}")
    for bits in (32, 8):
        kw = _lists([(1000,), (300,)], torch.float32, bits)
        clean = _copy(kw)
        kw["grads"][0][300] = bad
        W.adamw_step(**kw, **HYPER)
        W.adamw_step(**clean, **HYPER)
        keep = torch.ones(1000, dtype=torch.bool, device="cuda")
        keep[300] = False
        assert torch.equal(kw["params"][0][keep], clean["params"][0][keep])
        assert torch.equal(kw["params"][1], clean["params"][1])
        if bits == 8:
            keep[256:512] = False
            spread = torch.isnan(kw["exp_avgs"][0].float() * _spread(kw["scales"][0][0], 1000))
            assert spread[256:512].all() and not spread[:256].any() and not spread[512:].any()
        for k in ("exp_avgs", "exp_avg_sqs"):
            assert torch.equal(kw[k][0].float()[keep], clean[k][0].float()[keep])


def test_8bit_rounding_is_right_on_average():
    """The mean of the stored m, and of the stored root's square, over many seeds: off by at most five standard errors
    of a rounding up or down (half a step each), and the two states' roundings of an element are not tied."""
    log("adamw 8-bit rounding on average")
    n, seeds = 512, 400
    g = seeded((n,), 1, std=1.0, dtype=torch.float32)
    g[:20] *= 1e-4  # below the normal range of the codes
    base = _lists([(n,)], torch.float32, 8)
    base["grads"] = [g]
    w, m, v, *_ = _formula(base, 0, **HYPER)
    got_m, got_v = [], []
    for seed in range(seeds):
        kw = _copy(base)
        W.adamw_step(**kw, **HYPER, seed=seed)
        a, b = _values(kw, 0)
        got_m.append(a)
        got_v.append(b)
    s = _spread(kw["scales"][0][0].double(), n)
    step_m = torch.exp2(torch.floor(torch.log2((m / s).abs().clamp(2.0 ** -6, 447))) - 3) * s
    a, b = torch.stack(got_m), torch.stack(got_v)
    assert ((a.mean(0) - m).abs() <= 5 * step_m / 2 / math.sqrt(seeds) + 1e-9).all()
    rs = _spread(kw["scales"][0][1].double(), n)
    r = v.sqrt() / rs
    step_r = torch.exp2(torch.floor(torch.log2(r.clamp(2.0 ** -6, 447))) - 3)
    k = torch.floor(r / step_r)
    gap = (2 * k + 1) * (step_r * rs) ** 2  # between the two squares
    known = k >= 1  # a root below the least code is kept above zero: larger on purpose
    err = (b.mean(0) - v).abs() / (gap / 2 / math.sqrt(seeds))
    assert known.sum() > 480 and (err[known] <= 5 + 1e-3).all(), float(err[known].max())
    up = torch.stack([((x > y).double() - (x > y).double().mean(0)).flatten() for x, y in ((a, m), (b, v))])
    assert abs(float(torch.corrcoef(up)[0, 1])) < 0.02


def test_8bit_average_of_squares_moves():
    """v under gradients of another size: rounded to nearest it would stand still. After 2000 steps the mean over 4096
    elements is at 1 - 0.999^2000 of its way; the random walk of an element (a third of v) averages to half a percent."""
    log("adamw 8-bit v moves")
    kw = _lists([(4096,)], torch.float32, 8)
    kw["grads"] = [torch.full((4096,), 3e-2, device="cuda")]
    v0 = _values(kw, 0)[1].mean()
    for _ in range(2000):
        W.adamw_step(**kw, lr=0.0)
    share = 0.999 ** 2000
    assert abs(float(_values(kw, 0)[1].mean()) / float(v0 * share + (1 - share) * 9e-4) - 1) < 0.05


def test_stored_rounding_repeats_and_depends_on_the_seed():
    log("adamw seeds")
    runs = []
    for seed in (3, 3, 4, 2 ** 32 + 3, -1):
        kw = _lists([(5000,), (5000,)], torch.float32, 8, seed=0)
        kw["steps"].fill_(5)
        for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "scales"):
            kw[k][1] = kw[k][0].clone()
        W.adamw_step(**kw, **HYPER, seed=seed)
        runs.append(kw["exp_avgs"])
    same = lambda a, b: (a.float() == b.float()).float().mean().item()  # noqa: E731
    assert same(runs[0][0], runs[1][0]) == 1 and same(runs[0][0], runs[3][0]) == 1
    assert 0.3 < same(runs[0][0], runs[2][0]) < 0.9 and 0.3 < same(runs[0][0], runs[0][1]) < 0.9


def test_rate_on_the_device_and_captured_steps():
    """A captured step counts on, follows a rate that is changed between replays, and equals eager steps."""
    log("adamw captured")
    for bits in (32, 8):
        kw = _lists(SHAPES, torch.bfloat16, bits, masters=True)
        eager = _copy(kw)
        lr = torch.tensor(1e-2, device="cuda")
        call = lambda k, rate: W.adamw_step(**k, lr=rate, max_norm=0.5, seed=9)  # noqa: E731
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(kw, lr)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = call(kw, lr)
        call(eager, 1e-2)
        for i in range(5):
            lr.fill_(1e-2 / (i + 1))
            kw["grads"][8].mul_(0.5)
            eager["grads"][8].mul_(0.5)
            graph.replay()
            other = call(eager, float(lr))
            torch.cuda.synchronize()
            assert torch.equal(norm, other)
            for k in kw:
                same = zip(kw[k], eager[k]) if k != "steps" else [(kw[k], eager[k])]
                assert all(torch.equal(a.float(), b.float()) for a, b in same), (i, k)
        del graph


def test_another_stream():
    log("adamw on a side stream")
    kw = _lists(SHAPES, torch.float32, 32)
    want = _copy(kw)
    W.adamw_step(**want, **HYPER, max_norm=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        W.adamw_step(**kw, **HYPER, max_norm=0.1)
    side.synchronize()
    assert all(torch.equal(a, b) for k in ("params", "exp_avgs", "exp_avg_sqs") for a, b in zip(kw[k], want[k]))


def test_native_matches_python_path():
    log("adamw native against Python path")
    n = _hip.native()
    assert n is not _hip._NoNative
    for bits, dt, masters in ((32, torch.bfloat16, True), (8, torch.float16, False), (32, torch.float32, False)):
        for max_norm in (None, 0.1):
            a = _lists(SHAPES, dt, bits, masters)
            a["grads"][2] = None
            b = {k: list(v) if k == "grads" else _copy({k: v})[k] for k, v in a.items()}
            order = lambda k: (k["params"], k["grads"], k["exp_avgs"], k["exp_avg_sqs"], k["steps"], 1e-2, 0.9, 0.999, 1e-8,  # noqa: E731
                               0.1, k.get("masters"), k.get("scales"), max_norm, None, 3)
            got, want = n.adamw_step(*order(a)), _hip.adamw_step(*order(b))
            assert isinstance(got, tuple) and (got[0] is None) == (want is None)
            assert want is None or torch.equal(got[0], want)
            for k in ("params", "exp_avgs", "exp_avg_sqs", "masters", "scales"):
                assert all(torch.equal(x.float(), y.float()) for x, y in zip(a.get(k, []), b.get(k, [])))
            assert torch.equal(a["steps"], b["steps"])
    kw = _lists([(8, 8)], torch.float32, 32)
    args = [kw["params"], kw["grads"], kw["exp_avgs"], kw["exp_avg_sqs"], kw["steps"], 1e-2, 0.9, 0.999, 1e-8, 0.1, None,
            None, None, None, 0]
    t = kw["grads"][0]
    for i, bad in [(0, [t.cpu()]), (0, []), (1, [t[:4]]), (1, [t.t()]), (1, [t.double()]), (1, []), (2, [t.half()]), (3, [t[:7]]),
                   (4, kw["steps"].long()), (5, 1), (5, kw["steps"]), (6, 0), (10, [t]), (11, [t]), (13, t), (14, -1),
                   (0, tuple(kw["params"]))]:
        if i == 10:
            continue  # masters of fp32 parameters: the C entry refuses them, and the Python path says why
        assert n.adamw_step(*[bad if k == i else v for k, v in enumerate(args)]) is None, i
    assert int(kw["steps"][0]) == 0
    assert n.grad_norm([]) is None and n.grad_norm([None]) is None and n.grad_norm([t, t.half()]) is None
    assert n.grad_norm([t.cpu()]) is None and n.grad_norm((t,)) is None


def test_refusals():
    log("adamw refusals")

    def call(err, match=None, hyper=HYPER, **change):
        kw = _lists([(8, 4), (300,)], torch.bfloat16, 8, masters=True)
        kw.update(change)
        with pytest.raises(err, match=match):
            W.adamw_step(**kw, **hyper)
        assert "steps" in change or not (kw["steps"] - _lists([(8, 4), (300,)], torch.bfloat16)["steps"]).any()

    kw = _lists([(8, 4), (300,)], torch.bfloat16, 8, masters=True)
    p, s = kw["params"], kw["scales"]
    call(ValueError, "twice", params=[p[0], p[0]], grads=[kw["grads"][0]] * 2, exp_avgs=[kw["exp_avgs"][0]] * 2,
         exp_avg_sqs=[kw["exp_avg_sqs"][0]] * 2, masters=[kw["masters"][0]] * 2, scales=[s[0]] * 2)
    call(ValueError, "twice", exp_avgs=[kw["exp_avgs"][1][:32].view(8, 4), kw["exp_avgs"][1]])
    call(ValueError, "twice", scales=[s[1].flatten()[:2].view(2, 1), s[1]])
    call(ValueError, "twice", exp_avgs=kw["exp_avgs"], exp_avg_sqs=kw["exp_avgs"])
    call(ValueError, "contiguous", params=[p[0].t().contiguous().t(), p[1]])
    call(TypeError, "exp_avg 0", exp_avgs=[t.float() for t in kw["exp_avgs"]])
    call(ValueError, "scales 1", scales=[s[0], s[1][:, :1].contiguous()])
    call(ValueError, "scales 1", scales=[s[0], s[1].t().contiguous().t()])
    call(ValueError, "grads", grads=kw["grads"][:1])
    call(ValueError, "gradient 0", grads=[kw["grads"][0][:4], kw["grads"][1]])
    call(TypeError, "one dtype", grads=[kw["grads"][0], kw["grads"][1].float()])
    call(TypeError, "gradients", grads=[g.half() for g in kw["grads"]])
    call(TypeError, "master 0", masters=p)
    call(ValueError, "steps", steps=kw["steps"].long())
    call(ValueError, "steps", steps=kw["steps"][:1])
    call(ValueError, "GPU", grads=[g.cpu() for g in kw["grads"]])
    call(ValueError, "lr", hyper={**HYPER, "lr": torch.tensor([1.0, 2.0], device="cuda")})
    call(ValueError, "lr", hyper={**HYPER, "lr": torch.tensor(1.0, device="cuda", dtype=torch.float64)})
    call(ValueError, "norm without", hyper={**HYPER, "norm": torch.tensor(1.0, device="cuda")})
    with pytest.raises(TypeError, match="16-bit"):
        f = _lists([(8,)], torch.float32)
        W.adamw_step(**f, **HYPER, masters=[f["params"][0].clone()])


def test_saved_tensors_count_as_changed():
    log("adamw versions")
    p = torch.ones(4, device="cuda", requires_grad=True)
    out = (p * p).sum()
    kw = {"exp_avgs": [torch.zeros(4, device="cuda")], "exp_avg_sqs": [torch.zeros(4, device="cuda")]}
    for call in (W.adamw_step, lambda *a, **k: W.adamw_step(tuple(a[0]), *a[1:], **k)):  # native, Python path
        call([p], [torch.ones(4, device="cuda")], **kw, steps=torch.zeros(1, device="cuda", dtype=torch.int32), lr=0.1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.backward()
        out = (p * p).sum()
    out.backward()


# ----------------------------------------------------------------- the class
def _model(dt=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(dt).cuda()) for s in ((64, 48), (48,), (7, 3))]


def _set_grads(params, seed):
    for i, p in enumerate(params):
        p.grad = seeded(tuple(p.shape), seed + i, std=0.1, dtype=p.dtype)


def test_class_against_torch():
    """32-bit states of fp32 parameters: torch's own AdamW, which forms the same in fp32 in another order (ten steps, each
    off by a few units of the change)."""
    log("AdamW against torch.optim.AdamW")
    a, b = _model(torch.float32), _model(torch.float32)
    own = W.AdamW([{"params": a[:2]}, {"params": a[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=1e-3)
    ref = torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=1e-3, foreach=False)
    for step in range(10):
        for ps in (a, b):
            _set_grads(ps, 10 * step)
            if step < 4:
                ps[1].grad = None  # joins later: its own count
        own.step()
        ref.step()
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 10 * 40 * E * 1e-2 + 20 * E * q.abs().max()
    assert [int(own.state[p]["step"]) for p in a] == [10, 6, 10]


@pytest.mark.parametrize("bits", [32, 8])
def test_class_states_through_a_checkpoint(bits):
    log(f"AdamW state_dict {bits} bits")
    a = _model()
    opt = W.AdamW(a, lr=1e-2, state_bits=bits, max_norm=1.0, seed=3)
    for step in range(3):
        _set_grads(a, step)
        opt.step()
    saved = torch.utils._pytree.tree_map(lambda t: t.cpu() if isinstance(t, torch.Tensor) else t, opt.state_dict())
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    other = W.AdamW(b, lr=1e-2, state_bits=bits, max_norm=1.0, seed=3)
    other.load_state_dict(saved)
    for p, q in zip(a, b):
        for k, t in opt.state[p].items():
            assert other.state[q][k].dtype == t.dtype and torch.equal(other.state[q][k].float(), t.float())
    for step in range(3, 5):
        _set_grads(a, step)
        _set_grads(b, step)
        opt.step()
        other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(ValueError, match="bits"):
        W.AdamW(_model(), state_bits=40 - bits).load_state_dict(saved)
    import copy
    import io

    file = io.BytesIO()
    torch.save(opt, file)  # plain pickle does not load a float8 tensor of this torch
    file.seek(0)
    for clone in (copy.deepcopy(opt), torch.load(file, weights_only=False)):
        assert clone.state_bits == bits and clone.max_norm == 1.0
        ps = clone.param_groups[0]["params"]
        _set_grads(ps, 77)
        clone.step()
        _set_grads(b, 77)
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, b))


def test_class_captured_after_its_first_step(monkeypatch):
    log("AdamW captured")
    a, b = _model(), _model()
    opts = [W.AdamW(ps, lr=1e-2, state_bits=8, max_norm=1.0) for ps in (a, b)]
    _set_grads(a, 1)
    _set_grads(b, 1)
    with monkeypatch.context() as m:  # as within a capture, which is not begun: a failed one would outlast the test
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="first step"):
            opts[0].step()
    for o in opts:
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for i in range(4):
        for p, q in zip(a, b):
            p.grad.copy_(seeded(tuple(p.shape), 50 + i, std=0.1))
            q.grad.copy_(p.grad)
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), i
    assert int(opts[0].state[a[0]]["step"]) == 5


def test_class_mixed_types_scheduler_and_closure():
    log("AdamW mixed types")
    ps = _model(torch.bfloat16) + _model(torch.float32, 1) + [torch.nn.Parameter(torch.zeros(0, device="cuda"))]
    opt = W.AdamW(ps, lr=1e-2, max_norm=0.5)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda e: 0.5 ** e)

    def closure():
        opt.zero_grad()
        _set_grads(ps, 5)
        return torch.tensor(3.0)

    before = [p.detach().clone() for p in ps]
    assert opt.step(closure) == 3.0
    sched.step()
    opt.step(closure)
    assert all(not torch.equal(p, q) for p, q in zip(ps[:-1], before))
    assert "master" in opt.state[ps[0]] and "master" not in opt.state[ps[3]]
    with pytest.raises(ValueError, match="state_bits"):
        W.AdamW(ps, state_bits=16)
    with pytest.raises(ValueError, match="betas"):
        W.AdamW(ps, betas=(1.0, 0.9))
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(5, device="cuda"))], "lr": 0.1})
    opt.param_groups[1]["params"][0].grad = torch.ones(5, device="cuda")
    opt.step()
    assert int(opt.state[opt.param_groups[1]["params"][0]]["step"]) == 1 and int(opt.state[ps[0]]["step"]) == 3


def test_class_masters_of_some_parameters():
    """States loaded without a master beside new ones that have one, in one group: each parameter is stepped by its own kind."""
    log("AdamW, masters of some parameters")
    a = _model()
    opt = W.AdamW(a, lr=1e-2, masters=False)
    _set_grads(a, 0)
    opt.step()
    saved = opt.state_dict()
    for missing in (0, 2):  # the one without a state first, and last
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        other = W.AdamW(b, lr=1e-2)
        other.load_state_dict({**saved, "state": {i: s for i, s in saved["state"].items() if i != missing}})
        before = [p.detach().clone() for p in b]
        _set_grads(b, 5)
        other.step()
        assert ["master" in other.state[p] for p in b] == [i == missing for i in range(3)]
        assert all(not torch.equal(p, q) for p, q in zip(b, before))
        master = other.state[b[missing]]["master"]
        assert torch.equal(master.to(torch.bfloat16), b[missing]) and not torch.equal(master, b[missing].float())
        assert [int(other.state[p]["step"]) for p in b] == [1 if i == missing else 2 for i in range(3)]


def test_class_refused_states_change_nothing():
    log("AdamW, refused states")
    a, b = _model(), _model()
    opt, other = W.AdamW(a, lr=1e-2, state_bits=8), W.AdamW(b, lr=3e-3)
    for ps, o in ((a, opt), (b, other)):
        _set_grads(ps, 0)
        o.step()
    before = {p: {k: t.clone() for k, t in other.state[p].items()} for p in b}
    with pytest.raises(ValueError, match="bits"):
        other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["lr"] == 3e-3
    for p in b:
        assert other.state[p].keys() == before[p].keys()
        assert all(t.dtype == before[p][k].dtype and torch.equal(t, before[p][k]) for k, t in other.state[p].items())
    _set_grads(b, 1)
    other.step()
    assert [int(other.state[p]["step"]) for p in b] == [2, 2, 2]


def test_class_captured_right_after_loading():
    """The first step after a load, captured: its replays count on and equal eager steps."""
    log("AdamW captured after a load")
    a, b = _model(), _model()
    opt = W.AdamW(a, lr=1e-2, state_bits=8, max_norm=1.0)
    other = W.AdamW(b, lr=1e-2, state_bits=8, max_norm=1.0)
    for step in range(2):
        _set_grads(a, step)
        opt.step()
    for p, q in zip(a, b):
        q.data.copy_(p)
        q.grad = p.grad.clone()
    other.load_state_dict(opt.state_dict())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.step()
    for i in range(4):
        for p, q in zip(a, b):
            p.grad.copy_(seeded(tuple(p.shape), 50 + i, std=0.1))
            q.grad.copy_(p.grad)
        graph.replay()
        opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), i
        assert [int(other.state[q]["step"]) for q in b] == [3 + i] * 3
    del graph


@pytest.mark.parametrize("bits", [32, 8])
def test_class_goes_on_from_changed_parameters(bits):
    """bf16 parameters that are loaded, clamped, or changed between replays of a captured step: the next step starts there,
    and what was not changed keeps its master."""
    log(f"AdamW, changed parameters, {bits} bits")
    ps = _model()
    opt = W.AdamW(ps, lr=1e-3, weight_decay=0.0, state_bits=bits)
    for step in range(3):
        _set_grads(ps, step)
        opt.step()
    for group in opt.param_groups:
        group["lr"] = 0.0
    masters = [opt.state[p]["master"].clone() for p in ps]
    assert all(torch.equal(m.to(p.dtype), p) and not torch.equal(m, p.float()) for m, p in zip(masters, ps))
    want = [p.detach().clone() for p in ps]
    with torch.no_grad():
        for p, w in zip(ps, want):
            p.clamp_(-0.05, 0.05)
            w.clamp_(-0.05, 0.05)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(3):
        for p, w, m in zip(ps, want, masters):
            m.copy_(torch.where(m.to(p.dtype) == w, m, w.float()))
            assert torch.equal(p, w) and torch.equal(opt.state[p]["master"], m), i
        for p, w in zip(ps, want):
            p.data.flatten()[i] = w.flatten()[i] = 3.0 + i
        opt.masters_from_parameters()
        graph.replay()
        torch.cuda.synchronize()
    del graph


@pytest.mark.parametrize("path", ["native", "python"])
def test_tensors_without_a_gradient_do_not_count_as_changed(path):
    """A graph that saved a parameter which the step does not touch still runs; one that is stepped counts in all of its
    tensors."""
    log(f"adamw versions without a gradient, {path}")
    kw = _lists([(8,), (300,), (0,), (16,)], torch.bfloat16, 8, masters=True)
    kw["grads"][1] = kw["grads"][3] = None
    lists = ("params", "exp_avgs", "exp_avg_sqs", "masters", "scales")
    before = {k: [t._version for t in kw[k]] for k in lists}
    saved = [p.requires_grad_(True) for p in kw["params"]]
    outs = [(p * p).sum() for p in saved]
    if path == "python":
        kw["params"] = tuple(kw["params"])  # which the native path hands back
    with torch.no_grad():
        W.adamw_step(**kw, **HYPER)
    for k in lists:
        assert [t._version - v for t, v in zip(kw[k], before[k])] == [1, 0, 1, 0], k
    outs[1].backward()
    outs[3].backward()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        outs[0].backward()


def test_class_leaves_unused_parameters_to_their_graphs():
    """Two networks in one optimizer: a step of one does not disturb a retained graph of the other."""
    log("AdamW, a graph of an unused parameter")
    ps = _model(torch.float32)
    opt = W.AdamW(ps, lr=1e-2)
    _set_grads(ps, 0)
    opt.step()
    out = (ps[1] * ps[1]).sum()
    ps[1].grad = None
    opt.step()
    out.backward()
    assert torch.equal(ps[1].grad, 2 * ps[1])


@pytest.mark.parametrize("bits", [32, 8])
def test_an_error_left_by_an_earlier_call_is_not_the_steps(bits):
    """A HIP call that failed before leaves its error for whoever asks next: the step is made once all the same."""
    import ctypes

    log(f"adamw after another call's error, {bits} bits")
    hip = ctypes.CDLL("libamdhip64.so.7")
    for clip in ({}, {"max_norm": 0.1}):
        kw = _lists(SHAPES, torch.bfloat16, bits, masters=True)
        want = _copy(kw)
        W.adamw_step(**want, **HYPER, **clip)
        torch.cuda.synchronize()
        assert hip.hipSetDevice(1 << 20) != 0  # no such device: nothing is done, and the error stays
        W.adamw_step(**kw, **HYPER, **clip)
        torch.cuda.synchronize()
        for k in kw:
            same = zip(kw[k], want[k]) if k != "steps" else [(kw[k], want[k])]
            assert all(torch.equal(a.float(), b.float()) for a, b in same), k


@pytest.mark.parametrize("bits", [32, 8])
def test_class_under_another_default_dtype(bits):
    log(f"AdamW, default dtype bf16, {bits} bits")
    a, b = _model(), _model()
    opts = [W.AdamW(ps, lr=1e-2, state_bits=bits, max_norm=1.0) for ps in (a, b)]
    for step in range(2):
        _set_grads(a, step)
        _set_grads(b, step)
        opts[0].step()
        torch.set_default_dtype(torch.bfloat16)
        try:
            opts[1].step()
        finally:
            torch.set_default_dtype(torch.float32)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def _tiny_gradients(n, lo, hi, seed):
    g = torch.Generator().manual_seed(seed)
    size = torch.exp(math.log(lo) + math.log(hi / lo) * torch.rand(n, generator=g, dtype=torch.float64))
    return (size * (1 - 2 * torch.randint(0, 2, (n,), generator=g))).float().cuda()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-25, 1e-20])
def test_first_step_of_tiny_gradients(bits, eps):
    """v below fp32's normal range. A first step is lr g / (|g| + eps), but for v's own rounding: (1 - b2) g^2 is two
    products, each off by half of 2^-149 at most (the first times 1 - b2), less than 2^-149 together, which is half as much of the
    root relative to v; and 32 roundings at most of 2^-24."""
    log(f"adamw tiny gradients, {bits} bits, eps {eps}")
    n = 4096
    g = _tiny_gradients(n, 3e-20, 1e-15, 5)
    m, v = [torch.zeros(n, device="cuda")], [torch.zeros(n, device="cuda")]
    kw = {}
    if bits == 8:
        m, v = [m[0].to(torch.float8_e4m3fn)], [v[0].to(torch.float8_e4m3fn)]
        kw["scales"] = [torch.zeros(2, n // 256, device="cuda")]
    p = [torch.zeros(n, device="cuda")]
    steps = torch.zeros(1, device="cuda", dtype=torch.int32)
    W.adamw_step(p, [g], m, v, steps, lr=1e-2, eps=eps, weight_decay=0.0, **kw)
    assert int((1e-3 * g.double().square() < 2.0 ** -126).sum()) > 1000  # below the normal range
    d = g.double()
    want = -1e-2 * d / (d.abs() + eps)
    loss = 2.0 ** -149 / (1e-3 * d.square())
    _near(p[0], want, want.abs() * (loss + 32 * E), "param")
    if bits == 32:
        _near(v[0], 1e-3 * d.square(), 8 * E * d.square() * 1e-3 + 2.0 ** -149, "v")


@pytest.mark.parametrize("eps", [0.0, 1e-25])
def test_steps_from_tiny_averages(eps):
    """The stored v as it is: from the least subnormal number to beyond the range where the root is scaled."""
    log(f"adamw tiny averages, eps {eps}")
    v0 = torch.exp2(torch.arange(-149, -30, device="cuda", dtype=torch.float64).repeat_interleave(16)
                    + torch.arange(16, device="cuda", dtype=torch.float64).repeat(119) / 16).float()
    m0 = seeded((v0.numel(),), 3, dtype=torch.float32) * v0.double().sqrt().float()
    p, m, v = [torch.zeros_like(v0)], [m0.clone()], [v0.clone()]
    steps = torch.full((1,), 99, device="cuda", dtype=torch.int32)
    W.adamw_step(p, [torch.zeros_like(v0)], m, v, steps, lr=1e-2, eps=eps, weight_decay=0.0)
    root = v[0].double().sqrt() / math.sqrt(1 - 0.999 ** 100)  # of v as it was stored
    live = v[0] > 0
    assert int(live.sum()) >= v0.numel() - 16
    want = -1e-2 / (1 - 0.9 ** 100) * m[0].double() / (root + eps)
    _near(p[0][live], want[live], 32 * E * want[live].abs() + 2.0 ** -149, "param")


def test_8bit_roots_of_tiny_averages():
    """An 8-bit root that small is kept: its square is (1 - b2) g^2 to the codes' rounding."""
    log("adamw 8-bit tiny roots")
    g = torch.full((512,), 1e-20, device="cuda")
    m = torch.zeros(512, device="cuda").to(torch.float8_e4m3fn)
    kw = dict(params=[torch.zeros(512, device="cuda")], grads=[g], exp_avgs=[m.clone()], exp_avg_sqs=[m.clone()],
              scales=[torch.zeros(2, 2, device="cuda")], steps=torch.zeros(1, device="cuda", dtype=torch.int32))
    W.adamw_step(**kw, lr=0.0)
    v = _values(kw, 0)[1]
    want = 1e-3 * float(g[0].double()) ** 2
    # The scale is the largest root over 448, all roots are the largest; v is off by 2^-149 at most, the scale by roundings.
    _near(v, torch.full_like(v, want), 2.0 ** -149 + 32 * E * want, "v")
