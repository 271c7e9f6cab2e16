"""The operators together, as a program uses them. Training: a language model whose residual stream goes through
add_rmsnorm, its loss by linear_cross_entropy, its gradients applied by AdamW, eager and as one captured step. Serving:
the trained layer's weights in 8 bits, its norm, projections and MLP on 8-bit rows, for a whole text and for single
tokens."""
import pytest
import torch

import adamw as W
import add_rmsnorm as N
import embedding as E
import geglu as G
import linear_8bit as L8
import linear_cross_entropy as L
import qk_norm_rope as Q
import relpos_attention as A
import rmsnorm as R
from krsi_testutil import assert_parity, log, seeded

pytestmark = pytest.mark.gpu

B, S, H, D, F, V, LAYERS, EPS = 2, 33, 2, 64, 192, 211, 2, 1e-6
M = H * D


class Library:
    embedding, norm, add_norm, qk = staticmethod(E.embedding), staticmethod(R.rmsnorm), staticmethod(N.add_rmsnorm), staticmethod(Q.qk_norm_rope)
    attention, mlp, loss = staticmethod(A.relpos_attention), staticmethod(G.geglu_linear), staticmethod(L.linear_cross_entropy)


class Reference:
    embedding, norm, add_norm, qk = staticmethod(E.reference), staticmethod(R.reference), staticmethod(N.reference), staticmethod(Q.reference)
    attention, mlp, loss = staticmethod(A.reference), staticmethod(G.reference_linear), staticmethod(L.reference)


def parameters(dt=torch.bfloat16):
    def mat(n, k, seed):
        return (seeded((n, k), seed, dtype=torch.float32) / k ** 0.5).to(dt)

    def gain(seed, n=M):
        return seeded((n,), seed, 0.1, 1.0, dtype=dt)

    p = {"table": mat(V, M, 1), "first": gain(2)}
    for i in range(LAYERS):
        s = 10 * (i + 1)
        p |= {f"qkv{i}": mat(3 * M, M, s + 1), f"q{i}": gain(s + 2, D), f"k{i}": gain(s + 3, D), f"out{i}": mat(M, M, s + 4),
              f"norm_m{i}": gain(s + 5), f"up{i}": mat(2 * F, M, s + 6), f"down{i}": mat(M, F, s + 7), f"next{i}": gain(s)}
    return p


def loss_of(ops, p, tokens, targets, rope):
    b, s = tokens.shape
    linear = torch.nn.functional.linear
    pd = torch.where(torch.arange(2 * s - 1, device="cuda") < s, 0.0, float("-inf")).expand(H, -1).contiguous()
    x = ops.embedding(tokens, p["table"], M ** 0.5).reshape(b * s, M)
    y = ops.norm(x, p["first"], EPS)
    for i in range(LAYERS):
        qkv = ops.qk(linear(y, p[f"qkv{i}"]), p[f"q{i}"], p[f"k{i}"], rope, b, s, H, D, EPS)
        y, x = ops.add_norm(linear(ops.attention(qkv, pd, b, s, H, D, D ** -0.5), p[f"out{i}"]), x, p[f"norm_m{i}"], EPS)
        y, x = ops.add_norm(linear(ops.mlp(y, p[f"up{i}"]), p[f"down{i}"]), x, p[f"next{i}"], EPS)
    return ops.loss(y, p["table"], targets)


def batch(seed=0):
    tokens = torch.randint(0, V, (B, S + 1), generator=torch.Generator().manual_seed(seed)).cuda()
    targets = tokens[:, 1:].clone()
    targets[:, :3] = -100
    return tokens[:, :-1].contiguous(), targets.reshape(-1)


def leaves_of(p, dt=None):
    return {k: v.detach().to(dt or v.dtype, copy=True).requires_grad_(True) for k, v in p.items()}


def test_training_step_against_the_reference():
    log(f"training step with add_rmsnorm B{B} S{S} H{H} D{D} F{F} V{V}")
    p, (tokens, targets), rope = parameters(), batch(), Q.rope_table(S, D)
    runs = []
    for ops, dt in ((Reference, torch.float32), (Reference, None), (Library, None)):
        leaves = leaves_of(p, dt)
        loss = loss_of(ops, leaves, tokens, targets, rope)
        runs.append([loss.detach().view(1), *torch.autograd.grad(loss, list(leaves.values()))])
    assert_parity(["loss", *p], *runs, row_slack=float("inf"))


def _train(p, opt, grads, tokens, targets, rope):
    """One step, gradients into the same tensors."""
    loss = loss_of(Library, p, tokens, targets, rope)
    for g, new in zip(grads, torch.autograd.grad(loss, list(p.values()))):
        g.copy_(new)
    opt.step()
    return loss


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_equals_eager_training(bits):
    """Loss, gradients and the step of all parameters in one graph, replayed on other tokens; between the replays the
    eager program makes the same step on its own copies."""
    log(f"captured training {bits} bits")
    rope = Q.rope_table(S, D)
    tokens, targets = batch()
    sides = []
    for _ in range(2):
        p = leaves_of(parameters())
        for t in p.values():
            t.grad = torch.zeros_like(t)
        opt = W.AdamW(list(p.values()), lr=1e-3, state_bits=bits, max_norm=1.0)
        sides.append((p, opt, [t.grad for t in p.values()]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sides:  # the first step of each makes its states
            _train(*s, tokens, targets, rope)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = _train(*sides[0], tokens, targets, rope)
    for i in range(4):
        new_tokens, new_targets = batch(i + 1)
        tokens.copy_(new_tokens)
        targets.copy_(new_targets)
        graph.replay()
        want = _train(*sides[1], tokens, targets, rope)
        torch.cuda.synchronize()
        assert torch.equal(loss, want), i
        for k in sides[0][0]:
            assert torch.equal(sides[0][0][k], sides[1][0][k]), (i, k)
    assert int(sides[0][1].state[sides[0][0]["table"]]["step"]) == 5


def test_step_applies_the_gradients_of_the_library():
    """The parameters after one step are those of the formula on the masters, rounded."""
    log("AdamW after the library's backward")
    p, (tokens, targets), rope = leaves_of(parameters()), batch(), Q.rope_table(S, D)
    opt = W.AdamW(list(p.values()), lr=1e-2, weight_decay=0.1)
    loss_of(Library, p, tokens, targets, rope).backward()
    before = {k: t.detach().double() for k, t in p.items()}
    opt.step()
    for k, t in p.items():
        g = t.grad.double()
        want = before[k] * (1 - 1e-2 * 0.1) - 1e-2 * g / (g.abs() + 1e-8)  # at the first step m / sqrt(v) is g / |g|
        master = opt.state[t]["master"]
        # 16 roundings of the step (its size 1e-2 at most) and 4 of the weight; where g is near eps, of their quotient.
        assert ((master.double() - want).abs() <= 16 * 2.0 ** -24 * 1e-2 + 4 * 2.0 ** -24 * before[k].abs()).all(), k
        assert torch.equal(t.detach(), master.to(t.dtype)), k


def _verify_linear(out, x, w, q, s, wq, ws):
    """The 8-bit projection against that of x and w: each code is off by 2^-4 of its value, or 2^-10 of the scale below the
    normal range, so an output by (2^-4 + 2^-4 + 2^-8) of its terms' sizes and what the small ones add; 2^-9 for bf16."""
    a, b = x.double().abs() + s.double()[:, None] * 2.0 ** -6, w.double().abs() + ws.double()[:, None] * 2.0 ** -6
    bound = (2 * 2.0 ** -4 + 2.0 ** -8 + 2.0 ** -8) * (a @ b.t())
    assert ((out.double() - x.double() @ w.double().t()).abs() <= bound).all()
    exact = (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()
    err = (out.double() - exact).norm() / exact.norm()
    # A bf16 rounding (2^-9 at most, 2^-9.8 in the mean) and the matrix instruction's cut, 1e-4.
    assert err < 2.0 ** -9 + 2e-4, float(err)


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_served_layer_in_8_bits(rows):
    """norm and addition, projection, GEGLU, projection: every 8-bit product against that of what it stands for."""
    log(f"served layer rows={rows}")
    p = parameters()
    up, down = (L8.quantize_rows(p[k]) for k in ("up0", "down0"))
    x, res = seeded((rows, M), 5), seeded((rows, M), 6)
    with torch.no_grad():
        q, s, r = N.add_rmsnorm_8bit(x, res, p["norm_m0"], EPS)
        u = L8.linear_8bit(q, *up, x_scale=s)
        h = G.geglu(u)
        out = L8.linear_8bit(h, *down)
    y, stream = N.add_rmsnorm(x, res, p["norm_m0"], EPS)
    assert torch.equal(r, stream)
    # y is the norm rounded to bf16, the codes are of the norm itself: 2^-8 of a term more, within the bound's slack of 2^-8.
    _verify_linear(u, y, p["up0"], q, s, *up)
    hq, hs = L8.quantize_rows(h)
    _verify_linear(out, h, p["down0"], hq, hs, *down)


def test_single_tokens_give_the_rows_of_the_whole_text():
    """One token at a time through the 8-bit layer: the rows that the text at once gives, within the products' other order
    of sums (each kernel adds in its own: 2^-8 of a bf16 output is a step)."""
    log("single tokens in 8 bits")
    p = parameters()
    qkv = L8.quantize_rows(p["qkv0"])
    x, res = seeded((150, M), 5), seeded((150, M), 6)
    with torch.no_grad():
        q, s, r = N.add_rmsnorm_8bit(x, res, p["norm_m0"], EPS)
        whole = L8.linear_8bit(q, *qkv, x_scale=s, out_dtype=torch.float32)
        for t in (0, 77, 149):
            q1, s1, r1 = N.add_rmsnorm_8bit(x[t:t + 1], res[t:t + 1], p["norm_m0"], EPS)
            assert torch.equal(q1.float(), q[t:t + 1].float()) and torch.equal(s1, s[t:t + 1]) and torch.equal(r1, r[t:t + 1])
            one = L8.linear_8bit(q1, *qkv, x_scale=s1, out_dtype=torch.float32)
            size = (q1.double().abs() @ qkv[0].double().abs().t()) * s1.double()[:, None] * qkv[1].double()
            # Groups of eight products are the same in both; sums across them are fp32's.
            assert ((one - whole[t:t + 1]).double().abs() <= 2 * (M / 8 + 16) * 2.0 ** -24 * size).all()
