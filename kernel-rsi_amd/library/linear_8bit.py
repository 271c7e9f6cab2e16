"""Projection in 8 bits on gfx950 (MI355X) HIP kernels, for serving: linear_8bit(x, w, w_scale) = x @ w.T, with
quantize_rows(x2d) -> (q, scale), which brings a weight, once, and other rows to 8 bits.

w is [F, K] float8_e4m3fn (the layout of nn.Linear's weight) with an fp32 scale per row, as quantize_rows(weight) gives
them. x [rows, K] is float8_e4m3fn with its rows' scales, x_scale, as add_rmsnorm_8bit and quantize_rows give them; or it is
bf16, fp16 or fp32 without, and brought to 8 bits first, row by row. The codes' products are summed in fp32 on the matrix
cores, which cut each eight neighbouring ones at 2^-13 of the largest (1e-4 of an output of random rows); the sum is
scaled by both and rounded once to out_dtype (None: x's type, bf16 for codes).

quantize_rows: the scale makes a row's largest value 448, the type's largest, and codes are rounded to nearest even; a
code is off by 2^-4 of its value at most, or 2^-10 of the scale below 2^-6 of it. A row that holds an infinity or NaN reads back
as NaN throughout. K a multiple of 16, any rows and F. There is no gradient: it is refused where one would be
recorded. Usable under torch.compile(fullgraph=True).
"""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent))
import _hip  # noqa: E402
from _compat import compiling  # noqa: E402


def _ops():
    import _ops as ops  # noqa: PLC0415 - registers the krsi:: ops on first use
    return ops


def quantize_rows(x2d):
    """(q, scale) of the rows of x2d [rows, N] (see the module)."""
    _hip.refuse_recording("quantize_rows", x2d)
    if compiling():
        return _ops().quantize_rows_op(x2d)
    out = _hip.native().quantize_rows(x2d)
    return _hip.quantize_rows(x2d) if out is None else out


def linear_8bit(x, w, w_scale, *, x_scale=None, out_dtype=None):
    """x @ w.T in 8 bits (see the module)."""
    _hip.refuse_recording("linear_8bit", x, w, w_scale, x_scale)
    if x.dtype == _hip.E4M3:
        if x_scale is None:
            raise ValueError("x in 8 bits comes with x_scale, the scales of its rows")
        out_dtype = out_dtype or torch.bfloat16
    elif x_scale is not None:
        raise ValueError(f"x_scale is for x in 8 bits, which {x.dtype} is not")
    out_dtype = out_dtype or x.dtype
    if compiling():
        if x_scale is None:
            x, x_scale = _ops().quantize_rows_op(x)
        return _ops().linear_8bit_op(x, w, w_scale, x_scale, out_dtype)
    out = _hip.native().linear_8bit(x, w, w_scale, x_scale, _hip.DTYPE_CODES.get(out_dtype))
    if out is not None:
        return out
    if x_scale is None:
        x, x_scale = _hip.quantize_rows(x)
    return _hip.linear_8bit(x, w, w_scale, x_scale, out_dtype)


def reference(x, w, w_scale, *, x_scale=None, out_dtype=None):
    out_dtype = out_dtype or (torch.bfloat16 if x.dtype == _hip.E4M3 else x.dtype)
    if x_scale is None:
        f = x.float()
        x_scale = (f.abs().amax(1) / 448).clamp(min=2.0 ** -120)
        x = (f / x_scale[:, None]).to(_hip.E4M3)
    return ((x.float() @ w.float().t()) * x_scale[:, None] * w_scale).to(out_dtype)


def selftest():
    from _harness import compare, significance, time_ab, versions  # noqa: PLC0415

    x = torch.randn(2048, 4096, device="cuda", dtype=torch.bfloat16)
    w, w_scale = quantize_rows(torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16) / 64)
    ref32 = reference(x, w, w_scale, out_dtype=torch.float32)
    orig = reference(x, w, w_scale)
    checks = compare(ref32, orig, linear_8bit(x, w, w_scale))
    variants = {"reference": [lambda: reference(x, w, w_scale)], "kernel": [lambda: linear_8bit(x, w, w_scale)]}
    try:
        torch._dynamo.reset()
        fn_c, ref_c = torch.compile(linear_8bit, fullgraph=True), torch.compile(reference)
        compiled = {"pass": compare(ref32, orig, fn_c(x, w, w_scale))["pass"]}
        variants["compiled_reference"] = [lambda: ref_c(x, w, w_scale)]
        variants["compiled_kernel"] = [lambda: fn_c(x, w, w_scale)]
    except Exception as e:  # noqa: BLE001 - reported, not raised
        compiled = {"pass": False, "error": f"{type(e).__name__}: {str(e).splitlines()[0][:200]}"}
    t = time_ab(variants, rounds=3)
    us = {name: round(v["device_ms"] * 1e3, 1) for name, v in t.items()}

    def speed(base, cand):
        return {"speedup": round(us[base] / us[cand], 2), "significance": significance(t[base], t[cand])}

    if "compiled_kernel" in t:
        compiled.update(kernel_us=us["compiled_kernel"], reference_us=us["compiled_reference"],
                        **speed("compiled_reference", "compiled_kernel"))
    return {"pass": checks["pass"] and compiled.get("pass", False), "checks": checks, **versions(),
            "reference_us": us["reference"], "kernel_us": us["kernel"], **speed("reference", "kernel"),
            "compiled": compiled}


if __name__ == "__main__":
    print(selftest())
