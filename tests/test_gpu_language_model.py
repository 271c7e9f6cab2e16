"""A language model's training step on the library's kernels alone: embedding, then layers of rmsnorm, the fused
projection, qk_norm_rope, causal relpos_attention, rmsnorm and geglu_linear, then rmsnorm and
linear_cross_entropy with the embedding's table as its weight. Loss and every parameter's gradient against the
same model from each operator's reference() in fp32, with its bf16 run as the yardstick (the acceptance rule of the
library's self-tests); under a captured graph; and generation token by token against the whole sequence."""
import pytest
import torch

import embedding as E
import geglu as G
import linear_cross_entropy as L
import qk_norm_rope as Q
import relpos_attention as A
import rmsnorm as R
from krsi_testutil import assert_parity, log, seeded

pytestmark = pytest.mark.gpu

B, S, H, D, F, V, LAYERS, EPS = 3, 50, 3, 64, 384, 517, 2, 1e-6
M = H * D


class Library:
    embedding, norm, qk = staticmethod(E.embedding), staticmethod(R.rmsnorm), staticmethod(Q.qk_norm_rope)
    attention, mlp, loss = staticmethod(A.relpos_attention), staticmethod(G.geglu_linear), staticmethod(L.linear_cross_entropy)


class Reference:
    embedding, norm, qk = staticmethod(E.reference), staticmethod(R.reference), staticmethod(Q.reference)
    attention, mlp, loss = staticmethod(A.reference), staticmethod(G.reference_linear), staticmethod(L.reference)


def parameters(dt=torch.bfloat16):
    def mat(n, k, seed):
        return (seeded((n, k), seed, dtype=torch.float32) / k ** 0.5).to(dt)

    p = {"table": mat(V, M, 1), "norm": seeded((M,), 2, 0.1, 1.0, dtype=dt)}
    for i in range(LAYERS):
        s = 10 * (i + 1)
        p |= {f"norm_a{i}": seeded((M,), s, 0.1, 1.0, dtype=dt), f"qkv{i}": mat(3 * M, M, s + 1),
              f"q{i}": seeded((D,), s + 2, 0.1, 1.0, dtype=dt), f"k{i}": seeded((D,), s + 3, 0.1, 1.0, dtype=dt),
              f"out{i}": mat(M, M, s + 4), f"norm_m{i}": seeded((M,), s + 5, 0.1, 1.0, dtype=dt),
              f"up{i}": mat(2 * F, M, s + 6), f"down{i}": mat(M, F, s + 7)}
    return p


def causal(S):
    """The bias table of a decoder: 0 up to the query's own position, -inf after it."""
    return torch.where(torch.arange(2 * S - 1, device="cuda") < S, 0.0, float("-inf")).expand(H, -1).contiguous()


def hidden(ops, p, tokens, rope):
    b, s = tokens.shape
    linear, pd = torch.nn.functional.linear, causal(s)
    x = ops.embedding(tokens, p["table"], M ** 0.5).reshape(b * s, M)
    for i in range(LAYERS):
        qkv = linear(ops.norm(x, p[f"norm_a{i}"], EPS), p[f"qkv{i}"])
        qkv = ops.qk(qkv, p[f"q{i}"], p[f"k{i}"], rope, b, s, H, D, EPS)
        x = x + linear(ops.attention(qkv, pd, b, s, H, D, D ** -0.5), p[f"out{i}"])
        x = x + linear(ops.mlp(ops.norm(x, p[f"norm_m{i}"], EPS), p[f"up{i}"]), p[f"down{i}"])
    return ops.norm(x, p["norm"], EPS)


def batch():
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, V, (B, S + 1), generator=g).cuda()
    targets = tokens[:, 1:].clone()
    targets[:, :5] = -100  # a prompt
    targets[1, 30:] = -100  # a shorter sequence
    return tokens[:, :-1].contiguous(), targets.reshape(-1)


def step(ops, p, tokens, targets, rope):
    leaves = list(p.values())
    loss = ops.loss(hidden(ops, p, tokens, rope), p["table"], targets)
    return loss, torch.autograd.grad(loss, leaves)


def leaves_of(p, dt=None):
    return {k: v.detach().to(dt or v.dtype).requires_grad_(True) for k, v in p.items()}


def test_training_step():
    log(f"language model step B{B} S{S} H{H} D{D} F{F} V{V} layers {LAYERS}")
    p, (tokens, targets), rope = parameters(), batch(), Q.rope_table(S, D)
    runs = [step(ops, leaves_of(p, dt), tokens, targets, rope)
            for ops, dt in ((Reference, torch.float32), (Reference, None), (Library, None))]
    ref, orig, cand = ([loss.detach().view(1), *grads] for loss, grads in runs)
    assert_parity(["loss", *p], ref, orig, cand, row_slack=float("inf"))


def test_captured_step_replays_to_the_eager_one():
    """Replayed with other tokens in the same buffers, an eager step between the replays."""
    log("language model step in a graph")
    p, (tokens, targets), rope = leaves_of(parameters()), batch(), Q.rope_table(S, D)
    mine = leaves_of(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(Library, mine, tokens, targets, rope)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step(Library, mine, tokens, targets, rope)
    for i in range(3):
        tokens.copy_((tokens * 3 + i) % V)
        targets.copy_(torch.where(targets == -100, -100, (targets + 7 * i) % V))
        graph.replay()
        torch.cuda.synchronize()
        want, wants = step(Library, p, tokens, targets, rope)
        assert torch.equal(loss, want) and all(torch.equal(a, b) for a, b in zip(grads, wants)), i


def test_steps_on_two_streams_at_once():
    """Steps of two batches, each on its own stream, none waiting for the other: bitwise those made one after another."""
    log("language model steps on two streams")
    p, (tokens, targets), rope = parameters(), batch(), Q.rope_table(S, D)
    batches = [(tokens, targets), (tokens.flip(1).contiguous(), targets.flip(0).contiguous())]
    want = [step(Library, leaves_of(p), t, u, rope) for t, u in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    mine = [leaves_of(p) for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(Library, mine[i], *batches[i], rope))
    torch.cuda.synchronize()
    for (loss, grads), runs in zip(want, got):
        for other, others in runs:
            assert torch.equal(loss, other) and all(torch.equal(a, b) for a, b in zip(grads, others))


def test_single_tokens_at_their_positions():
    """One token of each sequence (S = 1) with its position: the rows that the whole sequences give, bitwise."""
    log("embedding and qk_norm_rope of single tokens")
    p, (tokens, _), rope = parameters(), batch(), Q.rope_table(S, D)
    at = torch.tensor([49, 0, 17], device="cuda")
    x = E.embedding(tokens, p["table"], M ** 0.5)
    one = E.embedding(tokens[torch.arange(B, device="cuda"), at], p["table"], M ** 0.5)
    assert torch.equal(one, x[torch.arange(B, device="cuda"), at])
    qkv = seeded((B * S, 3 * M), 3)
    whole = Q.qk_norm_rope(qkv, p["q0"], p["k0"], rope, B, S, H, D, EPS).view(B, S, -1)
    rows = qkv.view(B, S, -1)[torch.arange(B, device="cuda"), at]
    single = Q.qk_norm_rope(rows, p["q0"], p["k0"], rope, B, 1, H, D, EPS, positions=at)
    assert torch.equal(single, whole[torch.arange(B, device="cuda"), at])
