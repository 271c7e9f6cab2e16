"""Softmax cross entropy of an output projection without its logits, on gfx950 (MI355X) HIP kernels,
forward and backward: linear_cross_entropy(x, w, targets).

x [..., K] hidden states, w [V, K] the projection's weight (nn.Linear or a tied embedding), targets [...] int32
or int64. The loss of a row is log(sum_v exp(l_v)) - l_target for l = x w^T, formed in one pass over the
vocabulary: the logits are fp32 in registers and are never written. The backward computes them again in
pieces of the vocabulary; each piece's gradient is rounded to x's dtype (times a power of two, so that fp16
keeps small probabilities; rows of reduction="none" whose weight is 2^-k of the largest keep them down to 2^(k - 28)) and
multiplied into dx, which is carried in fp32, and dw; they are off by 1.1 to 1.3 times what their own rounding takes. The
backward allocates a piece, 512 MB or 8192 bytes a row where that is more, and fp32 sums: of dx, 4 rows K bytes for each part
of its sum, where there are several pieces or parts, and likewise of dw's piece. The logits themselves would take 4 bytes for
each row and vocabulary entry.
The loss is fp32: its mean over the targets that are not ignore_index (NaN if there are none), their sum,
or with reduction="none" the loss of each (0 where ignored, whatever its row of x holds). A row that is ignored, or whose
loss has gradient 0, gets none, whatever it holds; dw, which adds that row times zero, needs it finite. A target outside
[0, V) that is not ignore_index makes the loss, and the gradients, NaN. bf16 or fp16, K a multiple of 64. Usable under
torch.compile(fullgraph=True).
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


class LinearCrossEntropy(torch.autograd.Function):
    """Eager path of calls the native one hands back: launches the kernels directly."""

    @staticmethod
    def forward(ctx, x, w, targets, ignore_index, reduction):
        loss, stats = _hip.linear_cross_entropy_fwd(x, w, targets, ignore_index, reduction)
        ctx.save_for_backward(x, w, targets, stats)
        ctx.args = (ignore_index, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return (*_hip.linear_cross_entropy_bwd(dout, *ctx.saved_tensors, *ctx.args, *ctx.needs_input_grad[:2]), None,
                None, None)


def linear_cross_entropy(x, w, targets, *, ignore_index=-100, reduction="mean"):
    """cross_entropy(x @ w.T, targets) (see the module)."""
    shape = targets.shape
    if x.dim() != 2 or targets.dim() != 1:
        if x.shape[:-1] != shape or x.dim() < 1:
            raise ValueError(f"x {tuple(x.shape)} does not hold a row for each of targets {tuple(shape)}")
        x, targets = x.reshape(-1, x.shape[-1]), targets.reshape(-1)
    if compiling():
        loss = _ops().linear_cross_entropy_fwd_op(x, w, targets, ignore_index, reduction)[0]
    else:
        loss = _hip.native().linear_cross_entropy(x, w, targets, ignore_index, _hip.REDUCTIONS.get(reduction))
        if loss is None:
            loss = LinearCrossEntropy.apply(x, w, targets, ignore_index, reduction)
    return loss.view(shape) if loss.dim() and loss.shape != shape else loss


def reference(x, w, targets, *, ignore_index=-100, reduction="mean"):
    logits = torch.nn.functional.linear(x, w).reshape(-1, w.shape[0]).float()
    loss = torch.nn.functional.cross_entropy(logits, targets.reshape(-1).long(), ignore_index=ignore_index,
                                             reduction=reduction)
    return loss.view(targets.shape) if reduction == "none" else loss


def selftest():
    from _harness import selftest_autograd  # noqa: PLC0415

    x = torch.randn(2048, 1024, device="cuda", dtype=torch.bfloat16)
    w = (torch.randn(32128, 1024, device="cuda") / 32).to(torch.bfloat16)
    targets = torch.randint(0, 32128, (2048,), device="cuda")
    return selftest_autograd(lambda x, w: linear_cross_entropy(x, w, targets, reduction="none"),
                             lambda x, w: reference(x, w, targets, reduction="none"), [x, w])


if __name__ == "__main__":
    print(selftest())
