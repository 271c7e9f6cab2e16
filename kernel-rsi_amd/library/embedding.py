"""Token embedding with scaling, on gfx950 (MI355X) HIP kernels, forward and backward:
embedding(tokens, table, scale=1.0).

tokens (int32 or int64, any shape) name rows of table [V, D]; the result [*tokens.shape, D] holds
scale * table[token], rounded once. The gradient of table sums the output gradient's rows of each token in
fp32, over positions that one kernel has sorted by token: no float atomics, so it is bitwise reproducible.
Every row of it is written, zero where no token names it. A token outside [0, V) gives a row of NaN and
adds to no gradient. padding_idx: a row whose gradient stays zero (negative: counted from V).
bf16, fp16 or fp32, V up to 2^24, up to 2^25 tokens. Usable under torch.compile(fullgraph=True).
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


class Embedding(torch.autograd.Function):
    """Eager path of calls the native one hands back: launches the kernels directly."""

    @staticmethod
    def forward(ctx, tokens, table, scale, padding_idx):
        out = _hip.embedding_fwd(tokens, table, scale)
        ctx.save_for_backward(tokens)
        ctx.args = (table.shape[0], scale, padding_idx)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (tokens,) = ctx.saved_tensors
        return None, _hip.embedding_bwd(dout, tokens, *ctx.args), None, None


def embedding(tokens, table, scale=1.0, *, padding_idx=None):
    """scale * table[tokens] (see the module)."""
    pad = -1
    if padding_idx is not None:
        V = table.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx={padding_idx} is not a row of the table's {V}")
        pad = padding_idx % V
    if compiling():
        return _ops().embedding_fwd_op(tokens, table, float(scale), pad)
    out = _hip.native().embedding(tokens, table, float(scale), pad)
    return Embedding.apply(tokens, table, float(scale), pad) if out is None else out


def reference(tokens, table, scale=1.0, *, padding_idx=None):
    return torch.nn.functional.embedding(tokens, table, padding_idx=padding_idx) * scale


def selftest():
    from _harness import selftest_autograd  # noqa: PLC0415

    tokens = torch.randint(0, 32128, (4096,), device="cuda")
    table = torch.randn(32128, 1024, device="cuda", dtype=torch.bfloat16)
    # torch's own gradient of an embedding sorts by library calls that must not be captured: a replay of them faulted.
    return selftest_autograd(lambda t: embedding(tokens, t, 32.0), lambda t: reference(tokens, t, 32.0), [table],
                             graph=False)


if __name__ == "__main__":
    print(selftest())
