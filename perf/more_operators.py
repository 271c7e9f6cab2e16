"""The operators of a training step and of a served layer beside those of perf/operators.py, case by case, in their
plain form and through the library: the norm of a residual stream with the addition before it (its output in the
activations' type, or in 8 bits with a scale per row), the projection of 8-bit rows by an 8-bit weight, and the
AdamW step over all of a model's tensors (states in 32 bits, or in 8 with scales).

`own` chooses: False, elementary torch operations in 32 bits, rounded once; True, the public functions
of kernel-rsi_amd/library. `listed()` has the named cases, `draw()` further ones of the same ranges,
`exact()` the operators' definitions in 64 bits.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
TOP = 448.0            # the largest value of e4m3
LEAST = 2.0 ** -120    # a scale is no smaller: its reciprocal and its products stay normal
EPS = 1e-6
# The optimizer's: rate, decay of the averages, the divisor's floor, decay of the weights, seed of the 8-bit roundings.
LR, BETA1, BETA2, ADAM_EPS, DECAY, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 7
BLOCK = 256            # values that share a scale of an 8-bit state


def listed() -> list[dict]:
    return [
        # One step of generation: the newest token of 32 sequences, its norm in 8 bits for the projection that follows.
        {"name": "norm8_decode_32x4096_bf16", "op": "norm", "mode": "8bit", "dtype": "bf16", "rows": 32, "n": 4096},
        # Prefill in 8 bits, a number of tokens that no tile divides, fp16.
        {"name": "norm8_prefill_8191x8192_fp16", "op": "norm", "mode": "8bit", "dtype": "fp16", "rows": 8191, "n": 8192},
        # Training in 32 bits with an odd width.
        {"name": "norm_train_2042x1001_fp32", "op": "norm", "mode": "train", "dtype": "fp32", "rows": 2042, "n": 1001},
        # A large training layer.
        {"name": "norm_train_32768x4096_bf16", "op": "norm", "mode": "train", "dtype": "bf16", "rows": 32768, "n": 4096},
        # One step of generation of a single sequence: bound by the weight.
        {"name": "linear8_decode_1_k4096_f8192", "op": "linear", "dtype": "bf16", "rows": 1, "k": 4096, "f": 8192,
         "given": "8bit"},
        # 48 sequences, an odd number of outputs (fp16).
        {"name": "linear8_decode_48_k4112_f5633", "op": "linear", "dtype": "fp16", "rows": 48, "k": 4112, "f": 5633,
         "given": "8bit"},
        # A layer between kernels that give 16 bits: the rows are brought to 8 within the call.
        {"name": "linear8_rows1000_k1024_f5632_from_bf16", "op": "linear", "dtype": "bf16", "rows": 1000, "k": 1024,
         "f": 5632, "given": "16bit"},
        # A large prefill.
        {"name": "linear8_prefill_8192_k8192_f8192", "op": "linear", "dtype": "bf16", "rows": 8192, "k": 8192, "f": 8192,
         "given": "8bit"},
        # Many small tensors off any alignment, as in a small model whose parameters are packed: launches and latency.
        {"name": "adamw_145_small_tensors_fp32", "op": "adamw", "dtype": "fp32", "masters": False, "bits": 32, "clip": True,
         "layers": 24, "width": 69, "ffn": 200, "vocab": 1000},
        # A model of bf16 weights with fp32 masters, gradients clipped to a norm.
        {"name": "adamw_302M_masters_clip_bf16", "op": "adamw", "dtype": "bf16", "masters": True, "bits": 32, "clip": True,
         "layers": 1, "width": 4096, "ffn": 8192, "vocab": 32128},
        # The same with states in 8 bits.
        {"name": "adamw_302M_8bit_masters_bf16", "op": "adamw", "dtype": "bf16", "masters": True, "bits": 8, "clip": False,
         "layers": 1, "width": 4096, "ffn": 8192, "vocab": 32128},
        # States in 8 bits of a small model without masters, blocks that end inside rows and tensors that end inside blocks.
        {"name": "adamw_19M_8bit_fp32", "op": "adamw", "dtype": "fp32", "masters": False, "bits": 8, "clip": True,
         "layers": 4, "width": 505, "ffn": 1408, "vocab": 8000},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "linear", "adamw"])
    if op == "norm":
        n = _log_int(rng, 64, 16384)
        n = n if rng.random() < 0.3 else (n + 7) // 8 * 8
        return {"op": op, "mode": rng.choice(["8bit", "8bit", "train", "train", "eval"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "rows": _log_int(rng, 1, min(32768, (1 << 26) // n)),
                "n": n}
    if op == "linear":
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "rows": _log_int(rng, 1, 8192),
                "k": 16 * _log_int(rng, 8, 512), "f": _log_int(rng, 64, 8192), "given": rng.choice(["8bit", "8bit", "16bit"])}
    dtype, width = rng.choice(["bf16", "bf16", "fp16", "fp32"]), _log_int(rng, 64, 4096)
    ffn, vocab = _log_int(rng, width, 4 * width), _log_int(rng, 256, 32768)
    room = ((1 << 28) - vocab * width) // (4 * width * width + 3 * width * ffn)
    return {"op": op, "dtype": dtype, "masters": dtype != "fp32" and rng.random() < 0.7, "bits": rng.choice([8, 32]),
            "clip": rng.random() < 0.5, "layers": _log_int(rng, 1, max(1, min(24, room))), "width": width, "ffn": ffn,
            "vocab": vocab}


# ------------------------------------------------------------------ inputs
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(std).add_(mean).to(dtype)


def _stream(gen, rows: int, n: int, dtype):
    """Activations of a residual stream: rows of different sizes, a few columns far larger than the others."""
    t = torch.randn(rows, n, generator=gen, device="cuda")
    t *= torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    t[:, torch.randint(0, n, (max(1, n // 500),), generator=gen, device="cuda")] *= 12
    return t.to(dtype)


def _rows_to_8bit(t):
    """Codes and scales of the rows of an fp32 tensor: the largest value of a row becomes the largest code."""
    scale = (t.abs().amax(1) * (1 / TOP)).clamp_(min=LEAST)
    return (t * (1 / scale)[:, None]).to(E4M3), scale


def _shapes(case: dict) -> list[tuple]:
    """A model's tensors: the table, then of each layer its two norms and four projections."""
    w, f = case["width"], case["ffn"]
    return [(case["vocab"], w)] + case["layers"] * [(w,), (3 * w, w), (w, w), (w,), (2 * f, w), (w, f)]


def _views(flat, shapes) -> list:
    return [t.view(s) for t, s in zip(flat.split([math.prod(s) for s in shapes]), shapes)]


def _blocks(shapes) -> list[int]:
    return [-(-math.prod(s) // BLOCK) for s in shapes]


def _prepare_adamw(case: dict, gen, dt) -> dict:
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    flat = {"masters": _randn(gen, (sum(sizes),), torch.float32, 0.02)}
    flat["params"] = flat["masters"].to(dt)
    flat["grads"] = torch.empty_like(flat["params"])
    rms = [10 ** (-2 - 2 * x) for x in torch.rand(len(sizes), generator=gen, device="cuda").tolist()]
    grads = [x.copy_(_randn(gen, (n,), torch.float32, r)) for x, n, r in zip(flat["grads"].split(sizes), sizes, rms)]
    # Averages as some hundred steps leave them: m a fraction of the gradient's size, v near its square.
    m = torch.cat([0.3 * r * torch.randn(n, generator=gen, device="cuda") for n, r in zip(sizes, rms)])
    v = torch.cat([(r * (0.5 + torch.rand(n, generator=gen, device="cuda"))) ** 2 for n, r in zip(sizes, rms)])
    del grads
    if not case["masters"]:
        del flat["masters"]
    st = {"steps": torch.full((len(sizes),), 400, dtype=torch.int32, device="cuda")}
    if case["bits"] == 32:
        flat["m"], flat["v"] = m, v
    else:
        v.sqrt_()
        codes, scales = [], []
        for t in (m, v):
            parts = [torch.nn.functional.pad(x, (0, -len(x) % BLOCK)).view(-1, BLOCK) for x in t.split(sizes)]
            found = [_rows_to_8bit(x) for x in parts]
            codes.append(torch.cat([q.flatten()[:n] for (q, _), n in zip(found, sizes)]))
            scales.append([s for _, s in found])
        flat["m"], flat["v"] = codes
        flat["scales"] = torch.cat([x for pair in zip(*scales) for x in pair])
        st["scales"] = [t.view(2, b) for t, b in zip(flat["scales"].split([2 * b for b in _blocks(shapes)]), _blocks(shapes))]
    st["flat"] = flat
    st.update({k: _views(t, shapes) for k, t in flat.items() if k != "scales"})
    return st


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "adamw":
        return {**st, **_prepare_adamw(case, gen, dt)}
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        st["x"], st["residual"] = _randn(gen, (rows, n), dt), _stream(gen, rows, n, dt)
        st["w"] = _randn(gen, (n,), dt, 0.1, 1.0)
        if case["mode"] == "train":
            st["douts"] = [_randn(gen, (rows, n), dt), _randn(gen, (rows, n), dt)]
            st["leaves"] = [st[c].requires_grad_(True) for c in ("x", "residual", "w")]
        return st
    rows, k, f = case["rows"], case["k"], case["f"]
    st["w"], st["w_scale"] = _rows_to_8bit(_randn(gen, (f, k), torch.float32, k ** -0.5))
    x = _stream(gen, rows, k, torch.float32)
    if case["given"] == "8bit":
        st["x"], st["x_scale"] = _rows_to_8bit(x)
    else:
        st["x"] = x.to(dt)
    return st


# ------------------------------------------------------------------ one pass
def _library():
    path = str(Path(__file__).resolve().parents[1] / "kernel-rsi_amd" / "library")
    if path not in sys.path:
        sys.path.insert(0, path)
    import adamw
    import add_rmsnorm
    import linear_8bit
    return adamw, add_rmsnorm, linear_8bit


def _adamw_outputs(st: dict, norm) -> dict:
    out = {k: t for k, t in st["flat"].items() if k != "grads"}
    out["steps"] = st["steps"]
    return out if norm is None else {**out, "norm": norm}


def _own(st: dict):
    adamw, add_rmsnorm, linear_8bit = _library()
    c = st["case"]
    if c["op"] == "adamw":
        norm = adamw.adamw_step(st["params"], st["grads"], st["m"], st["v"], st["steps"], lr=LR, betas=(BETA1, BETA2),
                                eps=ADAM_EPS, weight_decay=DECAY, masters=st.get("masters"), scales=st.get("scales"),
                                max_norm=1.0 if c["clip"] else None, seed=SEED)
        return _adamw_outputs(st, norm)
    if c["op"] == "linear":
        with torch.no_grad():
            return {"out": linear_8bit.linear_8bit(st["x"], st["w"], st["w_scale"], x_scale=st.get("x_scale"),
                                                   out_dtype=DTYPES[c["dtype"]])}
    if c["mode"] == "train":
        y, r = add_rmsnorm.add_rmsnorm(st["x"], st["residual"], st["w"], EPS)
        return {"y": y.detach(), "r": r.detach(), "grads": list(torch.autograd.grad([y, r], st["leaves"], st["douts"]))}
    with torch.no_grad():
        if c["mode"] == "8bit":
            q, scale, r = add_rmsnorm.add_rmsnorm_8bit(st["x"], st["residual"], st["w"], EPS)
            return {"q": q, "scale": scale, "r": r}
        y, r = add_rmsnorm.add_rmsnorm(st["x"], st["residual"], st["w"], EPS)
        return {"y": y, "r": r}


def _plain_norm(st: dict) -> dict:
    c, dt = st["case"], st["x"].dtype
    x, res, w = (st[k].detach().float() for k in ("x", "residual", "w"))
    r = (x + res).to(dt)  # the stream that goes on, which the norm reads
    rf = r.float()
    rstd = 1 / torch.sqrt((rf * rf).mean(1, keepdim=True) + EPS)
    y = w * (rf * rstd)
    if c["mode"] == "8bit":
        q, scale = _rows_to_8bit(y)
        return {"q": q, "scale": scale, "r": r}
    out = {"y": y.to(dt), "r": r}
    if c["mode"] == "train":
        gy, gr = (g.float() for g in st["douts"])
        dn = gy * w
        d = (gr + (rstd * dn - rf * (rstd * rstd * rstd) * (dn * rf).mean(1, keepdim=True))).to(dt)
        out["grads"] = [d, d, (gy * rf * rstd).sum(0).to(dt)]
    return out


def _plain_linear(st: dict) -> dict:
    x, w = st["x"], st["w"].float()
    q, scale = (x, st["x_scale"]) if "x_scale" in st else _rows_to_8bit(x.float())
    return {"out": ((q.float() @ w.t()) * scale[:, None] * st["w_scale"]).to(DTYPES[st["case"]["dtype"]])}


def _mixed(h):
    """32 mixed bits of each whole number (held in 64 bits)."""
    h = h & 0xFFFFFFFF
    h = ((h ^ (h >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _uniform(step, sizes: list[int]):
    """Two uniform numbers of 16 bits for each element of the tensors' blocks in a step."""
    key = _mixed(torch.full((len(sizes),), SEED, dtype=torch.int64, device="cuda"))
    # The last word: an element's number over 2^32.
    for word in (step, torch.arange(len(sizes), device="cuda"), 0):
        key = _mixed(key * 3 + word * 0x9E3779B1 + 1)
    blocks = [-(-n // BLOCK) for n in sizes]
    first = torch.cat([torch.arange(n, device="cuda") for n in blocks])[:, None] * BLOCK
    key = torch.cat([k.expand(n) for k, n in zip(key, blocks)])[:, None]
    h = _mixed((first + torch.arange(BLOCK, device="cuda")) * 0x9E3779B1 + key)
    return [u.float() / 65536 for u in (h & 0xFFFF, h >> 16)]


def _grid(t):
    """The spacing of e4m3 at the size of each value."""
    return torch.exp2(torch.frexp(t).exponent.sub(1).clamp(-6, 8).float() - 3)


def _requantized(m, root, uniform):
    """m and the root of v of blocks [blocks, BLOCK] as codes and scales, rounded up or down at random so that the
    codes' values (of the root: their squares) are right on average; a root above zero stays above it."""
    ms, rs = ((t.abs().amax(1, keepdim=True) * (1 / TOP)).clamp(min=LEAST) for t in (m, root))
    a, b = m * (1 / ms), root * (1 / rs)
    ga, gb = _grid(a), _grid(b)
    ka = torch.floor(a / ga + uniform[0])
    t = b / gb
    low = torch.floor(t)
    kb = low + ((t - low) * (t + low) > uniform[1] * (2 * low + 1))
    kb = torch.where((low == 0) & (t > 0), 1.0, kb)
    return (ka * ga).clamp(-TOP, TOP).to(E4M3), (kb * gb).clamp(max=TOP).to(E4M3), ms, rs


def _adamw_of(w, g, m, v, factors):
    """The new weights and averages of fp32 ones; v's root with them."""
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(v)
    return w * (1 - LR * DECAY) - factors[0] * m / (root * factors[1] + ADAM_EPS), m, v, root


def _in_blocks(flat, sizes: list[int]):
    """The tensors of a flat buffer, each filled up to whole blocks: [blocks, BLOCK]."""
    return torch.cat([torch.nn.functional.pad(t, (0, -n % BLOCK)) for t, n in zip(flat.split(sizes), sizes)]).view(-1, BLOCK)


def _plain_adamw_8bit(st: dict, g, step, factors):
    """The new weights; the states' codes and scales are written."""
    flat, sizes = st["flat"], [t.numel() for t in st["params"]]
    blocks = [-(-n // BLOCK) for n in sizes]
    out_of = lambda t: torch.cat([x.flatten()[:n] for x, n in zip(t.split(blocks), sizes)])  # noqa: E731
    ms, rs = (torch.cat([s[k] for s in st["scales"]])[:, None] for k in (0, 1))
    m, root = _in_blocks(flat["m"], sizes).float() * ms, _in_blocks(flat["v"], sizes).float() * rs
    w = flat["masters"] if "masters" in flat else flat["params"].float()
    w, m, _, root = _adamw_of(_in_blocks(w, sizes), _in_blocks(g, sizes), m, root * root, factors)
    qm, qr, ms, rs = _requantized(m, root, _uniform(step, sizes))
    flat["m"].copy_(out_of(qm))
    flat["v"].copy_(out_of(qr))
    flat["scales"].copy_(torch.cat([x.flatten() for pair in zip(ms.split(blocks), rs.split(blocks)) for x in pair]))
    return out_of(w)


def _plain_adamw(st: dict) -> dict:
    c, flat = st["case"], st["flat"]
    g = flat["grads"].float()
    norm, share = None, 1.0
    if c["clip"]:
        norm = torch.sqrt((g * g).sum())
        share = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    st["steps"] += 1
    step = st["steps"][0].to(torch.int64)
    # Powers near 1, in 64 bits.
    factors = [(LR / (1 - BETA1 ** step.double())).float(), (1 / torch.sqrt(1 - BETA2 ** step.double())).float()]
    if c["bits"] == 8:
        w = _plain_adamw_8bit(st, g * share, step, factors)
    else:
        w, m, v, _ = _adamw_of(flat["masters"] if "masters" in flat else flat["params"].float(), g * share, flat["m"],
                               flat["v"], factors)
        flat["m"].copy_(m)
        flat["v"].copy_(v)
    flat["params"].copy_(w)
    if "masters" in flat:
        flat["masters"].copy_(w)
    return _adamw_outputs(st, norm)


def run(st: dict) -> dict:
    if own:
        return _own(st)
    return {"norm": _plain_norm, "linear": _plain_linear, "adamw": _plain_adamw}[st["case"]["op"]](st)


# ---------------------------------------------------------------- what counts
def work(case: dict) -> dict:
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        each = rows * n
        # x, residual -> r and y or its codes; and dy, dr, r -> the one gradient of x and residual, dw.
        nbytes = 2 * e * each + e * n + e * each + (each + 4 * rows if case["mode"] == "8bit" else e * each)
        return ({"bytes": nbytes + 4 * e * each + 2 * e * n, "flops": 19 * each} if case["mode"] == "train" else
                {"bytes": nbytes, "flops": 7 * each})
    if case["op"] == "linear":
        rows, k, f = case["rows"], case["k"], case["f"]
        x = rows * k + 4 * rows if case["given"] == "8bit" else e * rows * k
        return {"bytes": x + f * k + 4 * f + e * rows * f, "flops": 2 * rows * k * f}
    shapes = _shapes(case)
    total = sum(math.prod(s) for s in shapes)
    # Gradients, the weights (and masters) read once and written once, both averages both ways.
    nbytes = total * (e + (8 + e if case["masters"] else 2 * e) + (16 if case["bits"] == 32 else 4))
    nbytes += 8 * len(shapes) + (16 * sum(_blocks(shapes)) if case["bits"] == 8 else 0)
    return {"bytes": nbytes, "flops": total * (16 if case["bits"] == 32 else 40)}


# ------------------------------------------------------------------ in 64 bits
def _exact_norm(st: dict) -> dict:
    c, dt = st["case"], st["x"].dtype
    x, res, w = (st[k].detach().double() for k in ("x", "residual", "w"))
    total = x + res
    r = total.to(dt).double().requires_grad_(c["mode"] == "train")
    w.requires_grad_(c["mode"] == "train")
    y = r * (r.square().sum(1, keepdim=True) / c["n"] + EPS).rsqrt()
    y = y * w
    if c["mode"] == "8bit":
        scale = (torch.linalg.vector_norm(y, math.inf, dim=1) / TOP).clamp_(min=LEAST)
        return {"q": y / scale[:, None], "scale": scale, "r": total}
    if c["mode"] == "eval":
        return {"y": y, "r": total}
    dr, dw = torch.autograd.grad(y, [r, w], st["douts"][0].double())
    d = dr + st["douts"][1].double()
    return {"y": y.detach(), "r": total, "grads": [d, d, dw]}


def _exact_linear(st: dict) -> dict:
    x, w = st["x"].double(), st["w"].double() * st["w_scale"].double()[:, None]
    if "x_scale" in st:
        x = x * st["x_scale"].double()[:, None]
    else:  # the 8-bit values that the definition rounds the rows to, whose rounding borders are those of 32 bits
        q, scale = _rows_to_8bit(st["x"].float())
        x = q.double() * scale.double()[:, None]
    return {"out": torch.nn.functional.linear(x, w)}


def _exact_adamw(st: dict) -> dict:
    c, flat = st["case"], st["flat"]
    sizes = [t.numel() for t in st["params"]]
    g = flat["grads"].double()
    norm = torch.linalg.vector_norm(g)
    if c["clip"]:
        g /= torch.clamp(norm + 1e-6, min=1.0)
    m, v = flat["m"].double(), flat["v"].double()
    if c["bits"] == 8:
        ms, rs = (torch.cat([s[k].double().repeat_interleave(BLOCK)[:n] for s, n in zip(st["scales"], sizes)])
                  for k in (0, 1))
        m *= ms
        v = (v * rs).square_()
    m += (1 - BETA1) * (g - m)
    v += (1 - BETA2) * (g.square_() - v)
    t = int(st["steps"][0]) + 1
    w = flat["masters" if "masters" in flat else "params"].double()
    w = w - LR * DECAY * w - LR * (m / (1 - math.pow(BETA1, t))) / ((v / (1 - math.pow(BETA2, t))).sqrt() + ADAM_EPS)
    out = {k: w for k in ("masters", "params") if k in flat}
    out["steps"] = st["steps"] + 1
    if c["clip"]:
        out["norm"] = norm
    if c["bits"] == 32:
        return {**out, "m": m, "v": v}
    tops = [torch.nn.functional.pad(x.abs(), (0, -len(x) % BLOCK)).view(-1, BLOCK).amax(1) / TOP
            for pair in zip(m.split(sizes), v.sqrt().split(sizes)) for x in pair]
    return {**out, "m": None, "v": None, "scales": torch.cat(tops).clamp_(min=LEAST)}  # codes are rounded at random


def exact(case: dict, seed: int):
    return {"norm": _exact_norm, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](prepare(case, seed))
