"""The operators of a language model's training step around the layers, case by case, in their plain
form and through the library: the token embedding, the norm and rotation of query and key heads, and
the cross entropy of the output projection.

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
EPS = 1e-6
IGNORE = -100


def listed() -> list[dict]:
    return [
        # One step of generation: the newest token of 32 sequences at positions of their own.
        {"name": "qk_decode_b32_h32_kv16_d128_bf16", "op": "qk_norm_rope", "train": False, "dtype": "bf16", "b": 32,
         "s": 1, "h": 32, "kv": 16, "d": 128, "rot": 128, "interleaved": False, "positions": True},
        # Prefill of a model whose heads rotate half of their columns, in adjacent pairs, with few key heads.
        {"name": "qk_prefill_b1_s8191_h32_kv8_d128_fp16", "op": "qk_norm_rope", "train": False, "dtype": "fp16", "b": 1,
         "s": 8191, "h": 32, "kv": 8, "d": 128, "rot": 64, "interleaved": True, "positions": False},
        # Training with heads of 72 columns over a length that no tile divides.
        {"name": "qk_train_b2_s1021_h16_d72_bf16", "op": "qk_norm_rope", "train": True, "dtype": "bf16", "b": 2,
         "s": 1021, "h": 16, "kv": 16, "d": 72, "rot": 72, "interleaved": False, "positions": False},
        # A large training layer: 16384 tokens of 16 heads.
        {"name": "qk_train_b4_s4096_h16_d128_bf16", "op": "qk_norm_rope", "train": True, "dtype": "bf16", "b": 4,
         "s": 4096, "h": 16, "kv": 16, "d": 128, "rot": 128, "interleaved": False, "positions": False},
        # The embedding of one step of generation.
        {"name": "embed_decode_64_v32128_d4096_bf16", "op": "embedding", "train": False, "dtype": "bf16", "n": 64,
         "v": 32128, "d": 4096, "padded": False},
        # A mid-sized model's embedding in training, padded sequences.
        {"name": "embed_train_8191_v32128_d1024_bf16", "op": "embedding", "train": True, "dtype": "bf16", "n": 8191,
         "v": 32128, "d": 1024, "padded": True},
        # Full precision, an odd vocabulary and rows that no vector load divides.
        {"name": "embed_train_4099_v50257_d1001_fp32", "op": "embedding", "train": True, "dtype": "fp32", "n": 4099,
         "v": 50257, "d": 1001, "padded": False},
        # A large model's embedding in training.
        {"name": "embed_train_32768_v131072_d4096_bf16", "op": "embedding", "train": True, "dtype": "bf16", "n": 32768,
         "v": 131072, "d": 4096, "padded": False},
        # Scoring one short text: the loss of every token, no gradient.
        {"name": "loss_score_300_v32128_k1152_bf16", "op": "loss", "train": False, "dtype": "bf16", "n": 300,
         "v": 32128, "k": 1152, "reduction": "none"},
        # The loss of a mid-sized model's training step.
        {"name": "loss_train_2048_v32128_k1024_bf16", "op": "loss", "train": True, "dtype": "bf16", "n": 2048,
         "v": 32128, "k": 1024, "reduction": "mean"},
        # fp16 with a scaled loss, odd vocabulary and row count.
        {"name": "loss_train_4099_v50257_k2048_fp16", "op": "loss", "train": True, "dtype": "fp16", "n": 4099,
         "v": 50257, "k": 2048, "reduction": "mean"},
        # The loss of a large model's training step.
        {"name": "loss_train_8192_v131072_k4096_bf16", "op": "loss", "train": True, "dtype": "bf16", "n": 8192,
         "v": 131072, "k": 4096, "reduction": "mean"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["qk_norm_rope", "embedding", "loss"])
    train = rng.random() < 0.7
    if op == "qk_norm_rope":
        d = rng.choice([32, 40, 64, 72, 80, 96, 128, 128])
        h, b = _log_int(rng, 2, 32), _log_int(rng, 1, 32)
        kv = rng.choice([k for k in range(1, h + 1) if h % k == 0])
        s = 1 if not train and rng.random() < 0.5 else _log_int(rng, 2, max(2, (1 << 27) // (b * h * d * 8)))
        return {"op": op, "train": train, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "b": b, "s": s, "h": h,
                "kv": kv, "d": d, "rot": rng.choice([d, d, d // 2 // 2 * 2]), "interleaved": rng.random() < 0.3,
                "positions": s == 1 or rng.random() < 0.3}
    if op == "embedding":
        d = _log_int(rng, 64, 4096)
        d = d if rng.random() < 0.25 else d // 8 * 8
        return {"op": op, "train": train, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "n": _log_int(rng, 1, 16384), "v": _log_int(rng, 256, 65536), "d": d, "padded": rng.random() < 0.3}
    n, v, k = _log_int(rng, 1, 8192), _log_int(rng, 1000, 131072), _log_int(rng, 1, 64) * 64
    return {"op": op, "train": train, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "n": n, "v": v, "k": k,
            "reduction": rng.choice(["mean", "sum", "none"])}


# ------------------------------------------------------------------ inputs
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(std).add_(mean).to(dtype)


def _zipf(gen, n: int, v: int):
    """Token ids whose frequency falls as 1 / (id + 1), as ids sorted by frequency have it."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "qk_norm_rope":
        b, s, h, kv, d, rot = (case[c] for c in ("b", "s", "h", "kv", "d", "rot"))
        st["qkv"] = _randn(gen, (b * s, (h + 2 * kv) * d), dt)
        st["wq"], st["wk"] = _randn(gen, (d,), dt, 0.1, 1.0), _randn(gen, (d,), dt, 0.1, 1.0)
        length = max(s, 16384) if case["positions"] else s
        angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            10000.0, torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / -rot)
        st["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        st["positions"] = (torch.randint(0, length, (b * s,), generator=gen, device="cuda")
                           if case["positions"] else None)
        shape, leaves = st["qkv"].shape, ("qkv", "wq", "wk")
    elif case["op"] == "embedding":
        n, v, d = case["n"], case["v"], case["d"]
        st["tokens"] = _zipf(gen, n, v)
        if case["padded"]:  # a third of the positions holds the padding token 0
            st["tokens"][torch.rand(n, generator=gen, device="cuda") < 1 / 3] = 0
        st["table"] = _randn(gen, (v, d), dt, d ** -0.5)
        shape, leaves = (n, d), ("table",)
    else:
        n, v, k = case["n"], case["v"], case["k"]
        st["w"] = _randn(gen, (v, k), dt, k ** -0.5)
        st["targets"] = _zipf(gen, n, v)
        # Hidden states that lean to their token, some much and some little: losses from near 0 to log v.
        lean = 12 * torch.rand(n, 1, generator=gen, device="cuda")
        st["x"] = (torch.randn(n, k, generator=gen, device="cuda") + lean * st["w"][st["targets"]].float()).to(dt)
        st["targets"][torch.rand(n, generator=gen, device="cuda") < 0.1] = IGNORE  # of a prompt: no loss
        st["targets"][0] = 0
        shape, leaves = () if case["reduction"] != "none" else (n,), ("x", "w")
    if case["train"]:
        if case["op"] == "loss":
            # The loss's gradient: 1, in fp16 a loss scale, per token a weight.
            st["dout"] = torch.full(shape, 1024.0 if case["dtype"] == "fp16" else 1.0, device="cuda")
            if shape:
                st["dout"] *= torch.rand(shape, generator=gen, device="cuda") / case["n"]
        else:
            st["dout"] = _randn(gen, shape, dt)
        st["leaves"] = [st[c].requires_grad_(True) for c in leaves]
    return st


# ------------------------------------------------------------------ one pass
def _library():
    path = str(Path(__file__).resolve().parents[1] / "kernel-rsi_amd" / "library")
    if path not in sys.path:
        sys.path.insert(0, path)
    import embedding
    import linear_cross_entropy
    import qk_norm_rope
    return embedding, linear_cross_entropy, qk_norm_rope


def _own_forward(st: dict):
    embedding, linear_cross_entropy, qk_norm_rope = _library()
    c = st["case"]
    if c["op"] == "qk_norm_rope":
        return qk_norm_rope.qk_norm_rope(st["qkv"], st["wq"], st["wk"], st["rope"], c["b"], c["s"], c["h"], c["d"], EPS,
                                         kv_heads=c["kv"], positions=st["positions"], interleaved=c["interleaved"])
    if c["op"] == "embedding":
        return embedding.embedding(st["tokens"], st["table"], c["d"] ** 0.5, padding_idx=0 if c["padded"] else None)
    return linear_cross_entropy.linear_cross_entropy(st["x"], st["w"], st["targets"], ignore_index=IGNORE,
                                                     reduction=c["reduction"])


def _pairs(t, rot: int, interleaved: bool):
    """The two columns of each rotated pair, and the columns that do not rotate."""
    r = t[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    return a, b, t[..., rot:]


def _joined(a, b, rest, interleaved: bool):
    r = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([r, rest], -1)


def _plain_qk(st: dict) -> dict:
    c = st["case"]
    h, kv, d, rot, inter = c["h"], c["kv"], c["d"], c["rot"], c["interleaved"]
    tokens = c["b"] * c["s"]
    pos = torch.arange(tokens, device="cuda") % c["s"] if st["positions"] is None else st["positions"]
    cos, sin = st["rope"][pos][:, None].chunk(2, -1)
    x = st["qkv"].detach().float().view(tokens, h + 2 * kv, d)
    q, v = x[:, :h + kv], x[:, h + kv:]
    w = torch.cat([st["wq"].detach().float().expand(h, d), st["wk"].detach().float().expand(kv, d)])
    r = 1 / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS)
    a, b, rest = _pairs(w * q * r, rot, inter)
    y = torch.cat([_joined(a * cos - b * sin, b * cos + a * sin, rest, inter), v], 1)
    out = {"out": y.view(tokens, -1).to(st["qkv"].dtype)}
    if c["train"]:
        g = st["dout"].float().view(tokens, h + 2 * kv, d)
        a, b, rest = _pairs(g[:, :h + kv], rot, inter)
        dz = _joined(a * cos + b * sin, b * cos - a * sin, rest, inter)
        dw = (dz * q * r).sum(0)
        dn = dz * w
        dx = r * dn - q * (r * r * r) * (dn * q).mean(-1, keepdim=True)
        dqkv = torch.cat([dx, g[:, h + kv:]], 1).view(tokens, -1)
        out["grads"] = [t.to(st["qkv"].dtype) for t in (dqkv, dw[:h].sum(0), dw[h:].sum(0))]
    return out


def _plain_embedding(st: dict) -> dict:
    c, table = st["case"], st["table"].detach()
    scale = c["d"] ** 0.5
    out = {"out": (table[st["tokens"]].float() * scale).to(table.dtype)}
    if c["train"]:
        sums = torch.zeros(c["v"], c["d"], device="cuda").index_add_(0, st["tokens"], st["dout"].float())
        if c["padded"]:
            sums[0] = 0
        out["grads"] = [(sums * scale).to(table.dtype)]
    return out


def _plain_loss(st: dict) -> dict:
    c, targets = st["case"], st["targets"]
    x, w = st["x"].detach().float(), st["w"].detach().float()
    kept = targets != IGNORE
    at = torch.where(kept, targets, 0)[:, None]
    logits = x @ w.t()
    top = logits.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    loss = torch.where(kept, (lse - logits.gather(1, at))[:, 0], 0.0)
    share = 1 / kept.sum() if c["reduction"] == "mean" else 1.0
    out = {"out": loss if c["reduction"] == "none" else loss.sum() * share}
    if c["train"]:
        g = torch.where(kept, st["dout"] * share, 0.0)[:, None]
        p = torch.exp(logits - lse)
        p.scatter_add_(1, at, torch.full_like(g, -1.0))
        p *= g
        out["grads"] = [(p @ w).to(st["x"].dtype), (p.t() @ x).to(st["w"].dtype)]
    return out


def run(st: dict) -> dict:
    if not own:
        return {"qk_norm_rope": _plain_qk, "embedding": _plain_embedding, "loss": _plain_loss}[st["case"]["op"]](st)
    if not st["case"]["train"]:
        with torch.no_grad():
            return {"out": _own_forward(st)}
    out = _own_forward(st)
    grads = torch.autograd.grad(out, st["leaves"], st["dout"])
    return {"out": out.detach(), "grads": list(grads)}


# ---------------------------------------------------------------- what counts
def work(case: dict) -> dict:
    e, train = DTYPES[case["dtype"]].itemsize, case["train"]
    if case["op"] == "qk_norm_rope":
        tokens, d = case["b"] * case["s"], case["d"]
        normed, every = tokens * (case["h"] + case["kv"]) * d, tokens * (case["h"] + 2 * case["kv"]) * d
        table = 4 * case["rot"] * (tokens if case["positions"] else case["s"])
        # qkv -> y; and dy, q, k -> dqkv. The rotation table each way.
        nbytes = 2 * e * every + table + (e * (2 * every + normed) + table if train else 0)
        return {"bytes": nbytes, "flops": normed * (8 + (16 if train else 0))}
    if case["op"] == "embedding":
        n, v, d = case["n"], case["v"], case["d"]
        # Rows that the tokens name -> out; and dout -> every row of the gradient.
        nbytes = 8 * n + e * d * (min(n, v) + n) + (8 * n + e * d * (n + v) if train else 0)
        return {"bytes": nbytes, "flops": n * d * (3 if train else 1)}
    n, v, k = case["n"], case["v"], case["k"]
    nbytes = e * (n * k + v * k) + 12 * n + (2 * e * (n * k + v * k) if train else 0)
    return {"bytes": nbytes, "flops": 2 * n * v * k * (3 if train else 1)}


# ------------------------------------------------------------------ in 64 bits
def _exact_qk(st: dict):
    """Each pair as a complex number, turned by one of modulus 1."""
    c = st["case"]
    tokens, h, kv, d, rot = c["b"] * c["s"], c["h"], c["kv"], c["d"], c["rot"]
    x, wq, wk = (st[n].detach().double().requires_grad_(c["train"]) for n in ("qkv", "wq", "wk"))
    pos = st["positions"] if c["positions"] else torch.arange(c["s"], device="cuda").repeat(c["b"])
    table = st["rope"].double().index_select(0, pos)
    turn = torch.complex(table[:, :rot // 2], table[:, rot // 2:]).unsqueeze(1)

    def head(t, w):
        t = t.reshape(tokens, -1, d)
        t = t * (t.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * w
        shape = (rot // 2, 2) if c["interleaved"] else (2, rot // 2)
        p = t[..., :rot].unflatten(-1, shape)
        p = p if c["interleaved"] else p.transpose(-1, -2)
        p = torch.view_as_real(torch.complex(p[..., 0], p[..., 1]) * turn)
        p = (p if c["interleaved"] else p.transpose(-1, -2)).flatten(-2)
        return torch.cat([p, t[..., rot:]], -1).flatten(1)

    out = torch.cat([head(x[:, :h * d], wq), head(x[:, h * d:(h + kv) * d], wk), x[:, (h + kv) * d:]], 1)
    return out, [x, wq, wk]


def _exact_embedding(st: dict):
    c = st["case"]
    table = st["table"].detach().double().requires_grad_(c["train"])
    out = torch.nn.functional.embedding(st["tokens"], table, padding_idx=0 if c["padded"] else None)
    return out * math.sqrt(c["d"]), [table]


def _exact_loss(st: dict):
    c = st["case"]
    x, w = (st[n].detach().double().requires_grad_(c["train"]) for n in ("x", "w"))
    loss = torch.nn.functional.cross_entropy(x @ w.t(), st["targets"], ignore_index=IGNORE, reduction=c["reduction"])
    return loss, [x, w]


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    out, leaves = {"qk_norm_rope": _exact_qk, "embedding": _exact_embedding, "loss": _exact_loss}[case["op"]](st)
    if not case["train"]:
        return {"out": out}
    return {"out": out.detach(), "grads": list(torch.autograd.grad(out, leaves, st["dout"].double()))}
