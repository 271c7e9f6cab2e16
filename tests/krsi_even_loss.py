"""Inputs of linear_cross_entropy whose gradients show one rounding alone: that of the target's entry of dl.

Every logit of a row is the same (w is constant over the vocabulary where x is not zero), so p = 1 / V with V a power
of two, and weights g_n are powers of two: every entry of dl but the target's is exact in 16 bits, every product
and partial sum of both gradients is a small multiple of one power of two, exact in fp32. The target's entry,
g (1 / V - 1), rounds to -g: its rounding takes g / V. The columns are chosen so that the gradients are small beside what
that loss times w or x is:
  columns 0 .. 63     w = 2^-9 in each row, x_n = 2^13 / g_n but 0 in column (rank of n) mod 64:
                      dx is 0, dw is -2^13 / 64 but in one column.
  columns 64 .. 127   x = 0, w_v = 1 but 0 in column v mod 64: dx is -g_n / 64 but in one column; dw is 0.
With u = 2^-24 (fp32), h = finfo.eps / 2: p is off by e of itself, e = (2 K sum|x||w| + 64 + V / 1024 + 8 |lse|) u as the
forward's logits and exponentials have it; below h / 2, so that the other entries round to 1 / V. dl of the
target is off by (e / V + u) g, what comes back and its addition by u each, the result by its own rounding:
  |error| <= h |result| + (e / V + 4 u) g |w_t|   (dw: |x_n|), and 2^-25 for fp16's subnormals,
of which the second term is V e + 4 V u < 1/4 of what the rounding takes."""
import torch

V, K, STEP = 8192, 128, 2.0 ** -24


def inputs(dt, ignored=0, unweighted=0, seed=0, device="cuda"):
    """x, w, targets, dout (per row), rank: of each row that counts its number, else -1. Every vocabulary entry is the
    target of one row that counts; rows of weight 0 that name some of them come after, ignored rows before and after."""
    g = torch.Generator().manual_seed(seed)
    before = min(ignored, 37)
    rank = torch.cat([torch.full((before,), -1), torch.arange(V), torch.full((unweighted + ignored - before,), -1)])
    order = torch.randperm(V, generator=g)
    targets = torch.full((len(rank),), -100)
    targets[before:before + V] = order
    zero = slice(before + V, before + V + unweighted)
    targets[zero] = order[torch.randperm(V, generator=g)[:unweighted]]
    weight = 2.0 ** torch.randint(10, 14, (len(rank),), generator=g)
    x = torch.zeros(len(rank), K)
    x[:, :64] = (rank[:, None] % 64 != torch.arange(64)) * (2.0 ** 13 / weight)[:, None]
    w = torch.cat([torch.full((V, 64), 2.0 ** -9), (torch.arange(V)[:, None] % 64 != torch.arange(64)).float()], 1)
    dout = weight.clone()
    dout[zero] = 0.0
    return x.to(dt).to(device), w.to(dt).to(device), targets.to(device), dout.to(device), rank.to(device)


def bounds(r, x, w, targets, rank):
    """Of the oracle's result r for such inputs: what dx and dw may be off by (see above)."""
    h = torch.finfo(x.dtype).eps / 2
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    e = ((2 * K * r["terms"] + 64 + V / 1024 + 8 * r["lse"].abs()) * STEP).max().item()
    assert e < h / 2 and e + 4 * V * STEP < 0.25
    off = (e / V + 4 * STEP) * r["g"].abs()[:, None]
    counts = rank >= 0
    at = torch.where(targets >= 0, targets, 0)
    dw = h * r["dw"].abs() + sub
    dw[at[counts]] += off[counts] * x[counts].double().abs()
    return h * r["dx"].abs() + sub + off * w[at].double().abs(), dw


def emulated(x, w, targets, dout, fault=None):
    """dx and dw as the kernels form them, rounded to x's type, from float64; with a fault planted in what comes back
    of the target's rounding."""
    dt = x.dtype
    xd, wd = x.double(), w.double()
    g = torch.where(targets >= 0, dout.double(), 0.0)
    at = torch.where(targets >= 0, targets, 0)
    n = torch.arange(len(at))
    d = torch.softmax(xd @ wd.t(), 1) * g[:, None]
    d[n, at] -= g
    dl = d.to(dt).double()
    rest = (d - dl)[n, at]
    last = torch.full((len(w),), -1)
    names = g != 0 if fault != "rows without weight" else targets >= 0
    last.scatter_reduce_(0, at[names], n[names], "amax")
    if fault == "none":
        rest = torch.zeros_like(rest)
    elif fault == "sign":
        rest = -rest
    elif fault == "another row's":
        rest = rest.roll(1)
    to_w, to_x = (at, last) if fault != "another entry" else ((at + 1) % len(w), torch.where(last > 0, last - 1, last))
    dx = dl @ wd + rest[:, None] * wd[to_w]
    dw = dl.t() @ xd + torch.where(last >= 0, rest[last], 0.0)[:, None] * xd[to_x]
    return dx.to(dt), dw.to(dt)


def within(got, ref, bound):
    return bool(((got.double() - ref).abs() <= bound).all())
