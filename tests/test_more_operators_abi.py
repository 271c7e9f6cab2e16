"""The C entries of add_rmsnorm, linear_8bit and adamw without a GPU: every refusal comes before a launch (FAKE
pointers, nothing on the device is dereferenced), workspaces cover what the kernels use, and the Python functions
refuse CPU tensors and arguments that do not fit."""
import ctypes

import pytest
import torch

import _hip
import adamw as W
import add_rmsnorm as A
import linear_8bit as L

NULL, FAKE = None, 0x10000
NULLP, SHAPE, ALIGN, WS, UNSUP, SCALE = 1, 2, 3, 4, 5, 7
NAN, INF = float("nan"), float("inf")


def test_add_rmsnorm_arguments():
    lib = _hip.lib()
    ok = dict(x=FAKE, residual=FAKE, w=FAKE, y=FAKE, r=FAKE, rstd=FAKE, rows=4, n=64, eps=1e-6, dt=0)

    def fwd(**kw):
        return lib.krsi_add_rmsnorm_fwd(*{**ok, **kw}.values(), NULL)

    sizes = [(dict(dt=3), UNSUP), (dict(dt=-1), UNSUP), (dict(rows=-1), SHAPE), (dict(n=0), SHAPE), (dict(n=16385), SHAPE),
             (dict(rows=1 << 26), SHAPE), (dict(rows=1 << 22, n=16384), SHAPE)]
    assert fwd(rows=0, x=NULL, y=NULL) == 0  # no rows: no-op
    for kw, rc in sizes + [(dict(eps=NAN), SCALE), (dict(eps=INF), SCALE)]:
        assert fwd(**kw) == rc, kw
    for name in ("x", "residual", "w", "y", "r"):
        assert fwd(**{name: NULL}) == NULLP, name
    ok8 = dict(x=FAKE, residual=FAKE, w=FAKE, q=FAKE, scale=FAKE, r=FAKE, rows=4, n=64, eps=1e-6, dt=0)

    def fwd8(**kw):
        return lib.krsi_add_rmsnorm_8bit(*{**ok8, **kw}.values(), NULL)

    assert fwd8(rows=0, x=NULL) == 0
    for kw, rc in sizes + [(dict(eps=NAN), SCALE), (dict(residual=NULL), NULLP), (dict(r=NULL), NULLP), (dict(q=NULL), NULLP),
                           (dict(scale=NULL), NULLP), (dict(x=NULL), NULLP), (dict(w=NULL), NULLP)]:
        assert fwd8(**kw) == rc, kw
    quant = lambda x=FAKE, q=FAKE, s=FAKE, rows=4, n=64, dt=0: lib.krsi_quantize_rows(x, q, s, rows, n, dt, NULL)  # noqa: E731
    assert quant(rows=0, x=NULL) == 0
    assert (quant(x=NULL), quant(q=NULL), quant(s=NULL)) == (NULLP,) * 3
    assert (quant(rows=-1), quant(n=0), quant(n=(1 << 20) + 1), quant(rows=1 << 26)) == (SHAPE,) * 4 and quant(dt=5) == UNSUP
    size = lib.krsi_add_rmsnorm_bwd_workspace_bytes
    # A partial row of fp32 for each workgroup: as many as there are groups of rows, 512 at most.
    assert size(100000, 4096) >= 512 * 4096 * 4 and size(1, 4096) >= 4096 * 4
    assert size(0, 64) == size(5, 0) == size(5, 16385) == 0
    okb = dict(dy=FAKE, dr=FAKE, r=FAKE, w=FAKE, rstd=FAKE, dx=FAKE, dw=FAKE, ws=FAKE, nb=1 << 24, rows=4, n=64, dt=0)

    def bwd(**kw):
        return lib.krsi_add_rmsnorm_bwd(*{**okb, **kw}.values(), NULL)

    for kw, rc in sizes + [(dict(ws=NULL), WS), (dict(nb=size(4, 64) - 1), WS), (dict(ws=FAKE + 8), ALIGN),
                           (dict(rows=0, dw=NULL), NULLP)]:
        assert bwd(**kw) == rc, kw
    for name in ("dy", "r", "w", "rstd", "dx", "dw"):
        assert bwd(**{name: NULL}) == NULLP, name


def test_linear_8bit_arguments():
    ok = dict(x=FAKE, w=FAKE, xs=FAKE, ws=FAKE, out=FAKE, work=NULL, nb=0, rows=4, k=64, f=32, dt=0)

    def call(**kw):
        return _hip.lib().krsi_linear_8bit(*{**ok, **kw}.values(), NULL)

    assert call(rows=0, x=NULL, out=NULL) == 0
    for kw, rc in [(dict(dt=3), UNSUP), (dict(k=40), UNSUP), (dict(k=(1 << 20) + 16), UNSUP), (dict(rows=(1 << 23) + 1), UNSUP),
                   (dict(f=(1 << 23) + 1), UNSUP), (dict(rows=1 << 22, f=1 << 22), UNSUP), (dict(rows=-1), SHAPE),
                   (dict(k=0), SHAPE), (dict(f=0), SHAPE), (dict(x=FAKE + 8), ALIGN), (dict(w=FAKE + 1), ALIGN)]:
        assert call(**kw) == rc, kw
    for name in ("x", "w", "xs", "ws", "out"):
        assert call(**{name: NULL}) == NULLP, name
    # Few outputs of a long sum: parts of it, two at least, in fp32.
    size, long = _hip.lib().krsi_linear_8bit_workspace_bytes, dict(rows=200, k=8192, f=512)
    need = size(*long.values())
    assert need >= 2 * 200 * 512 * 4 and size(8192, 8192, 8192) == 0 and size(0, 64, 64) == size(4, 40, 4) == size(-1, 64, 4) == 0
    assert call(**long) == WS and call(**long, work=FAKE, nb=need - 1) == WS and call(**long, work=FAKE + 4, nb=need) == ALIGN


def _array(*ptrs):
    return (ctypes.c_void_p * len(ptrs))(*ptrs)


def _sizes(*n):
    return (ctypes.c_int64 * len(n))(*n)


def test_adamw_arguments():
    lib = _hip.lib()
    two, apart = _sizes(10, 300), _array(FAKE, FAKE + 4096)
    size = lib.krsi_adamw_workspace_bytes
    m, v = _array(FAKE + 8192, FAKE + 12288), _array(FAKE + 16384, FAKE + 20480)
    ok = dict(params=apart, grads=apart, m=m, v=v, masters=NULL, scales=NULL, sizes=two, count=2, steps=FAKE, lr_at=NULL,
              lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, norm=NULL, given=0, max_norm=0.0, seed=0, bits=32, dt=0, gdt=0,
              ws=FAKE, nb=1 << 20)

    def call(**kw):
        return lib.krsi_adamw_step(*{**ok, **kw}.values(), NULL)

    assert call(count=0, params=NULL, sizes=NULL) == 0
    for kw, rc in [(dict(dt=3), UNSUP), (dict(gdt=1), UNSUP), (dict(dt=2, gdt=0), UNSUP), (dict(dt=2, gdt=2, masters=apart), UNSUP),
                   (dict(bits=16), UNSUP), (dict(bits=8), UNSUP), (dict(scales=apart), UNSUP), (dict(count=-1), SHAPE),
                   (dict(count=(1 << 20) + 1), SHAPE), (dict(sizes=_sizes(-1, 3)), SHAPE), (dict(sizes=_sizes(1 << 36, 3)), SHAPE),
                   (dict(sizes=_sizes(1 << 35, 1 << 35)), SHAPE), (dict(lr=NAN), SCALE), (dict(lr=INF), SCALE),
                   (dict(eps=-1.0), SCALE), (dict(eps=NAN), SCALE), (dict(wd=INF), SCALE), (dict(b1=1.0), SCALE),
                   (dict(b2=-0.1), SCALE), (dict(b1=NAN), SCALE), (dict(norm=FAKE, max_norm=-1.0), SCALE),
                   (dict(norm=FAKE, max_norm=NAN), SCALE), (dict(given=2), SCALE), (dict(ws=NULL), WS), (dict(nb=16), WS),
                   (dict(ws=FAKE + 4), ALIGN), (dict(params=_array(FAKE, FAKE)), SHAPE),
                   (dict(params=_array(FAKE + 16, FAKE)), SHAPE), (dict(m=apart), SHAPE), (dict(v=m), SHAPE),
                   (dict(m=_array(FAKE + 8192, FAKE + 8200)), SHAPE), (dict(masters=v), SHAPE),
                   (dict(scales=_array(FAKE + 30000, FAKE + 30004), bits=8), SHAPE), (dict(params=_array(FAKE, NULL)), NULLP),
                   (dict(m=_array(NULL, FAKE)), NULLP), (dict(v=_array(FAKE, NULL)), NULLP),
                   (dict(masters=_array(FAKE, NULL)), NULLP), (dict(scales=_array(FAKE, NULL), bits=8), NULLP)]:
        assert call(**kw) == rc, kw
    for name in ("params", "grads", "m", "v", "sizes", "steps"):
        assert call(**{name: NULL}) == NULLP, name
    # 32 bytes of factors per tensor and a part of the norm for each 16384 elements of one.
    assert size(two, 2) >= 2 * 32 + 2 * 4 and size(_sizes(1 << 20), 1) >= 32 + 64 * 4
    assert size(_sizes(-1), 1) == 0 and size(NULL, 1) == 0 and size(NULL, 0) > 0
    nsize = lib.krsi_grad_norm_workspace_bytes
    norm = dict(grads=apart, sizes=two, count=2, norm=FAKE, ws=FAKE, nb=1 << 20, dt=0)

    def norm_of(**kw):
        return lib.krsi_grad_norm(*{**norm, **kw}.values(), NULL)

    for kw, rc in [(dict(dt=7), UNSUP), (dict(count=-1), SHAPE), (dict(sizes=_sizes(-1, 1)), SHAPE), (dict(sizes=NULL), NULLP),
                   (dict(grads=NULL), NULLP), (dict(norm=NULL), NULLP), (dict(ws=NULL), WS), (dict(nb=nsize(two, 2) - 1), WS),
                   (dict(ws=FAKE + 2), ALIGN)]:
        assert norm_of(**kw) == rc, kw


def test_python_functions_refuse_before_a_launch():
    x, w = torch.zeros(4, 64), torch.ones(64)
    q = x.to(torch.float8_e4m3fn)
    for fn in (A.add_rmsnorm, A.add_rmsnorm_8bit):
        with pytest.raises(ValueError, match="GPU"):
            fn(x, x, w, 1e-6)
    with pytest.raises(ValueError, match="GPU"):
        L.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        L.linear_8bit(q, q, torch.ones(4), x_scale=torch.ones(4))
    with pytest.raises(ValueError, match="x_scale"):
        L.linear_8bit(q, q, torch.ones(4))
    with pytest.raises(ValueError, match="x_scale"):
        L.linear_8bit(x, q, torch.ones(4), x_scale=torch.ones(4))
    for fn, args in ((A.add_rmsnorm_8bit, (x.clone().requires_grad_(True), x, w, 1e-6)),
                     (L.quantize_rows, (x.clone().requires_grad_(True),)),
                     (L.linear_8bit, (x.clone().requires_grad_(True), q, torch.ones(4)))):
        with pytest.raises(ValueError, match="no gradient"):
            fn(*args)
    steps = torch.zeros(1, dtype=torch.int32)
    ok = dict(lr=1e-3)
    with pytest.raises(ValueError, match="GPU"):
        W.adamw_step([x], [x], [x], [x], steps, **ok)
    with pytest.raises(ValueError, match="parameter"):
        W.adamw_step([], [], [], [], steps, **ok)
    with pytest.raises(ValueError, match="GPU"):
        W.grad_norm([x])
    with pytest.raises(ValueError, match="gradient"):
        W.grad_norm([None])
    for kw, match in [(dict(lr=-1.0), "lr"), (dict(lr=NAN), "lr"), (dict(lr=1e-3, betas=(0.9, 1.0)), "betas"),
                      (dict(lr=1e-3, betas=(NAN, 0.9)), "betas"), (dict(lr=1e-3, eps=-1e-8), "eps"),
                      (dict(lr=1e-3, weight_decay=INF), "weight_decay"), (dict(lr=1e-3, max_norm=-1.0), "max_norm"),
                      (dict(lr=1e-3, max_norm=NAN), "max_norm"), (dict(lr=1e-3, norm=x.sum()), "norm without")]:
        with pytest.raises(ValueError, match=match):
            W.adamw_step([x], [x], [x], [x], steps, **kw)
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    with pytest.raises(ValueError, match="GPU"):
        W.AdamW([p]).step()


@pytest.mark.parametrize("eps", [2.0 ** -127, 1e-40, 1e-46])
def test_adamw_eps_below_the_normal_range(eps):
    """Its reciprocal overflows in fp32 (or it is zero there): 0 / eps, the step of an element that has never had a gradient,
    would be NaN."""
    x, steps = torch.zeros(4, 64), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="eps"):
        W.adamw_step([x], [x], [x], [x], steps, lr=1e-3, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        W.AdamW([torch.nn.Parameter(x)], eps=eps)
    for good in (0.0, 2.0 ** -126):
        with pytest.raises(ValueError, match="GPU"):
            W.adamw_step([x], [x], [x], [x], steps, lr=1e-3, eps=good)
    at = _array(FAKE)
    lib, sizes = _hip.lib(), _sizes(64)

    def call(eps, ws):
        return lib.krsi_adamw_step(at, at, _array(FAKE + 4096), _array(FAKE + 8192), NULL, NULL, sizes, 1, FAKE, NULL, 1e-3, 0.9,
                                   0.999, eps, 0.01, NULL, 0, 0.0, 0, 32, 2, 2, ws, 1 << 20, NULL)

    assert call(2.0 ** -126, NULL) == call(0.0, NULL) == WS
    assert call(eps, FAKE) == SCALE if eps > 2.0 ** -150 else call(eps, NULL) == WS
