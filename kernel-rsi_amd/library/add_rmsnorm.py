"""The addition of a layer's output to the residual stream with the RMS norm of the sum in one pass, on gfx950
(MI355X) HIP kernels: add_rmsnorm(x2d, residual, w, eps) -> (y, r), forward and backward, and
add_rmsnorm_8bit(x2d, residual, w, eps) -> (q, scale, r), whose norm comes in 8 bits for linear_8bit.

x2d (a layer's output) and residual (the stream so far) are [rows, N], contiguous, and w is [N], of one type (bf16,
fp16 or fp32); N up to 16384. r = x2d + residual, rounded once, is the stream that goes on; y is the norm of r, in
fp32 and rounded once (rmsnorm(r, w, eps) rounds the normalised row as well). Both outputs carry gradients: those of y and
of r reach x2d and residual as one tensor in a single pass, rounded once, and w's gradient is summed in fp32 in a fixed
order (bitwise reproducible).

In 8 bits: the norm in fp32, its rounding to the activations' type left out, becomes float8_e4m3fn codes q [rows, N]
with an fp32 scale per row, which makes the row's largest value 448, the type's largest: the norm is about
q * scale[:, None]. residual=None: the norm of x2d alone, and r is x2d. A row that holds an infinity or NaN reads back
as NaN throughout. There is no gradient: it is refused where one would be recorded.
Usable under torch.compile(fullgraph=True).
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


class AddRMSNorm(torch.autograd.Function):
    """Eager path of calls the native one hands back: launches the kernels directly."""

    @staticmethod
    def forward(ctx, x2d, residual, w, eps):
        y, r, rstd = _hip.add_rmsnorm_fwd(x2d, residual, w, eps)
        ctx.save_for_backward(r, w, rstd)
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr):
        r, w, rstd = ctx.saved_tensors
        if dy is None:  # the stream alone was used
            return dr, dr, None, None
        dx, dw = _hip.add_rmsnorm_bwd(dy, None if dr is None else dr.contiguous(), r, w, rstd)
        return dx, dx, dw, None


def add_rmsnorm(x2d, residual, w, eps):
    """(norm of r, r) for r = x2d + residual (see the module)."""
    if compiling():
        return _ops().add_rmsnorm_fwd_op(x2d, residual, w, eps)[:2]
    out = _hip.native().add_rmsnorm(x2d, residual, w, eps)
    return AddRMSNorm.apply(x2d, residual, w, eps) if out is None else out


def add_rmsnorm_8bit(x2d, residual, w, eps):
    """(q, scale, r): the norm of r = x2d + residual in 8 bits (see the module)."""
    _hip.refuse_recording("add_rmsnorm_8bit", x2d, residual, w)
    if compiling():
        if residual is None:
            return (*_ops().rmsnorm_8bit_op(x2d, w, eps), x2d)
        return _ops().add_rmsnorm_8bit_op(x2d, residual, w, eps)
    out = _hip.native().add_rmsnorm_8bit(x2d, residual, w, eps)
    q, scale, r = _hip.add_rmsnorm_8bit(x2d, residual, w, eps) if out is None else out
    return q, scale, x2d if residual is None else r


def reference(x2d, residual, w, eps):
    r = x2d + residual
    var = r.float().pow(2).mean(-1, keepdim=True)
    return w * (r.float() * torch.rsqrt(var + eps)).to(r.dtype), r


def selftest():
    from _harness import selftest_autograd  # noqa: PLC0415

    x, res = (torch.randn(4096, 1024, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w = (1 + 0.1 * torch.randn(1024, device="cuda")).to(torch.bfloat16)
    # Both outputs side by side, as one: the protocol takes a function of one output.
    return selftest_autograd(lambda *t: torch.cat(add_rmsnorm(*t, 1e-6), 1), lambda *t: torch.cat(reference(*t, 1e-6), 1),
                             [x, res, w])


if __name__ == "__main__":
    print(selftest())
