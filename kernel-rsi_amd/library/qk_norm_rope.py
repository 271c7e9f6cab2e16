"""RMS norm of every query and key head with the position rotation in the same pass, on gfx950 (MI355X)
HIP kernels, forward and backward: qk_norm_rope(qkv, q_weight, k_weight, rope, B, S, H, D, eps).

qkv [B*S, (H + 2*kv_heads)*D] is the fused projection output as relpos_attention takes it: token t holds
its H query heads, then its key heads, then its value heads, D columns each. The result has the same
layout, contiguous: every query and key head x is z = w * x / sqrt(mean(x^2) + eps), with w = q_weight or
k_weight [D], then its first R columns are rotated in pairs (a, b) by the token's angles,
(a cos - b sin, b cos + a sin); value heads are copied. So it stands between the projection and
relpos_attention (kv_heads = H there).
  rope       [P, R] fp32, R even, R <= D: row p holds the R/2 cosines, then the R/2 sines, of position p.
             rope_table() builds it. No gradient flows to it.
  positions  None: token t is at position t % S (P >= S). Or one int32 or int64 per token, as one step
             of generation (S = 1) has them. One outside [0, P) makes its token's rotated columns NaN.
  interleaved  False: pair i is columns (i, i + R/2); True: columns (2i, 2i + 1).
fp32 arithmetic from the load to the store, rounded once. The weights' gradients are summed in fp32 in a
fixed order, so they are bitwise reproducible. qkv may be wider than its heads and its rows may lie apart
(any alignment); without unit column stride it is copied first. D any multiple of 8 up to 128; bf16, fp16
or fp32. Usable under torch.compile(fullgraph=True).
"""
import sys
from pathlib import Path

import torch
from torch.autograd.function import once_differentiable

sys.path.insert(0, str(Path(__file__).resolve().parent))
import _hip  # noqa: E402
from _compat import compiling  # noqa: E402


def _ops():
    import _ops as ops  # noqa: PLC0415 - registers the krsi:: ops on first use
    return ops


class QKNormRope(torch.autograd.Function):
    """Eager path of calls the native one hands back: launches the kernels directly."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, rope, positions, *dims):
        out = _hip.qk_norm_rope_fwd(qkv, q_weight, k_weight, rope, positions, *dims)
        ctx.save_for_backward(qkv, q_weight, k_weight, rope, positions)
        ctx.dims = dims
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return (*_hip.qk_norm_rope_bwd(dout, *ctx.saved_tensors, *ctx.dims), *[None] * 9)


def rope_table(length, dim, theta=10000.0, device="cuda"):
    """[length, dim] fp32 for qk_norm_rope: the cosines, then the sines, of p * theta^(-2i/dim) for position p and
    i < dim/2. The angles are formed in 64 bits, where those of far positions keep their fraction of a turn."""
    if length < 1 or dim < 2 or dim % 2:
        raise ValueError(f"rope_table needs length >= 1 and an even dim >= 2, got {length} and {dim}")
    turn = theta ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * turn
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _in_place_layout(qkv, cols):
    """qkv itself when the kernels can read it where it is, else a copy of its heads' columns
    (differentiable, so the gradient reaches qkv)."""
    if qkv.dim() != 2 or qkv.shape[1] < cols:
        return qkv  # rejected with its shape by the kernel wrapper
    if qkv.stride(1) == 1 and (qkv.shape[0] <= 1 or qkv.stride(0) >= cols):
        return qkv
    return qkv[:, :cols].clone(memory_format=torch.contiguous_format)


def qk_norm_rope(qkv, q_weight, k_weight, rope, B, S, H, D, eps, *, kv_heads=None, positions=None, interleaved=False):
    """qkv with its query and key heads normalised and rotated (see the module)."""
    kv = H if kv_heads is None else kv_heads
    if not compiling():
        out = _hip.native().qk_norm_rope(qkv, q_weight, k_weight, rope, positions, B, S, H, kv, D, eps, int(interleaved))
        if out is not None:
            return out
    if rope.requires_grad:
        raise ValueError("rope is a constant of qk_norm_rope: it gets no gradient, but requires one")
    qkv = _in_place_layout(qkv, (H + 2 * kv) * D)
    args = (qkv, q_weight, k_weight, rope, positions, B, S, H, kv, D, eps, bool(interleaved))
    if compiling():
        return _ops().qk_norm_rope_fwd_op(*args)
    return QKNormRope.apply(*args)


def reference(qkv, q_weight, k_weight, rope, B, S, H, D, eps, *, kv_heads=None, positions=None, interleaved=False):
    kv = H if kv_heads is None else kv_heads
    pos = torch.arange(B * S, device=qkv.device) % S if positions is None else positions.reshape(-1).long()
    R = rope.shape[1]
    cos, sin = rope[pos][:, None].chunk(2, -1)
    x = qkv[:, :(H + 2 * kv) * D].reshape(B * S, H + 2 * kv, D)
    heads = []
    for part, w in ((x[:, :H], q_weight), (x[:, H:H + kv], k_weight)):
        f = part.float()
        z = w * (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + eps)).to(qkv.dtype)
        r = z[..., :R].float()
        a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, -1)
        a, b = a * cos - b * sin, b * cos + a * sin
        r = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        heads.append(torch.cat([r.to(qkv.dtype), z[..., R:]], -1))
    return torch.cat([*heads, x[:, H + kv:]], 1).reshape(B * S, -1)


def selftest():
    from _harness import selftest_autograd  # noqa: PLC0415

    B, S, H, D = 4, 512, 16, 128
    qkv = torch.randn(B * S, 3 * H * D, device="cuda", dtype=torch.bfloat16)
    wq, wk = ((1 + 0.1 * torch.randn(D, device="cuda")).to(torch.bfloat16) for _ in range(2))
    rope = rope_table(S, D)
    return selftest_autograd(lambda *t: qk_norm_rope(*t, rope, B, S, H, D, 1e-6),
                             lambda *t: reference(*t, rope, B, S, H, D, 1e-6), [qkv, wq, wk])


if __name__ == "__main__":
    print(selftest())
