"""The C entries of qk_norm_rope, embedding and linear_cross_entropy without a GPU: every refusal comes before a
launch (FAKE pointers, nothing is dereferenced), workspaces cover what the kernels use, and the Python functions
refuse CPU tensors and arguments that do not fit."""
import pytest
import torch

import _hip
import embedding as E
import linear_cross_entropy as L
import qk_norm_rope as Q

NULL, FAKE = None, 0x10000
NULLP, SHAPE, ALIGN, WS, UNSUP, SCALE = 1, 2, 3, 4, 5, 7


def test_qk_norm_rope_arguments():
    lib = _hip.lib()
    ok = dict(qkv=FAKE, ld=384, wq=FAKE, wk=FAKE, rope=FAKE, pos=NULL, out=FAKE, tokens=8, S=4, H=2, KH=2, D=64, R=64,
              rows=4, pb=0, eps=1e-6, inter=0, dt=0)

    def fwd(**kw):
        return lib.krsi_qk_norm_rope_fwd(*{**ok, **kw}.values(), NULL)

    assert fwd(tokens=0, qkv=NULL, out=NULL) == 0  # no tokens: no-op
    for kw, rc in [(dict(qkv=NULL), NULLP), (dict(wq=NULL), NULLP), (dict(wk=NULL), NULLP), (dict(rope=NULL), NULLP),
                   (dict(out=NULL), NULLP), (dict(dt=3), UNSUP), (dict(dt=-1), UNSUP), (dict(inter=2), UNSUP),
                   (dict(D=60), UNSUP), (dict(D=136, ld=1000), UNSUP), (dict(D=0), UNSUP), (dict(ld=383), SHAPE),
                   (dict(tokens=-1), SHAPE), (dict(tokens=1 << 31), SHAPE), (dict(S=0), SHAPE), (dict(H=0), SHAPE),
                   (dict(KH=0), SHAPE), (dict(R=0), SHAPE), (dict(R=63), SHAPE), (dict(R=66), SHAPE), (dict(rows=0), SHAPE),
                   (dict(rows=3), SHAPE), (dict(pos=FAKE, pb=2), SHAPE),
                   (dict(tokens=(1 << 31) - 1, S=1, H=65535, KH=1, ld=1 << 23), SHAPE), (dict(eps=float("nan")), SCALE),
                   (dict(eps=float("inf")), SCALE)]:
        assert fwd(**kw) == rc, kw
    nbytes = lib.krsi_qk_norm_rope_bwd_workspace_bytes(64)
    assert nbytes >= 1024 * 2 * 64 * 4 and lib.krsi_qk_norm_rope_bwd_workspace_bytes(0) == 0
    okb = dict(dout=FAKE, qkv=FAKE, ld=384, wq=FAKE, wk=FAKE, rope=FAKE, pos=NULL, dqkv=FAKE, ldd=384, dwq=FAKE, dwk=FAKE,
               ws=FAKE, nb=nbytes, tokens=8, S=4, H=2, KH=2, D=64, R=64, rows=4, pb=0, eps=1e-6, inter=0, dt=0)

    def bwd(**kw):
        return lib.krsi_qk_norm_rope_bwd(*{**okb, **kw}.values(), NULL)

    for kw, rc in [(dict(dout=NULL), NULLP), (dict(dqkv=NULL), NULLP), (dict(dwq=NULL), NULLP), (dict(dwk=NULL), NULLP),
                   (dict(ldd=383), SHAPE), (dict(ws=NULL), WS), (dict(nb=nbytes - 1), WS), (dict(ws=FAKE + 4), ALIGN),
                   (dict(tokens=0, dwk=NULL), NULLP)]:
        assert bwd(**kw) == rc, kw


def test_embedding_arguments():
    lib = _hip.lib()
    ok = dict(tokens=FAKE, tb=8, table=FAKE, out=FAKE, n=4, V=10, D=8, scale=1.0, dt=0)

    def fwd(**kw):
        return lib.krsi_embedding_fwd(*{**ok, **kw}.values(), NULL)

    assert fwd(n=0, tokens=NULL, table=NULL, out=NULL) == 0
    bad = [(dict(tb=2), UNSUP), (dict(dt=3), UNSUP), (dict(n=-1), SHAPE), (dict(n=(1 << 25) + 1), SHAPE), (dict(V=0), SHAPE),
           (dict(V=(1 << 24) + 1), SHAPE), (dict(D=0), SHAPE), (dict(D=(1 << 20) + 1), SHAPE),
           (dict(scale=float("nan")), SCALE), (dict(scale=float("-inf")), SCALE)]
    for kw, rc in bad + [(dict(tokens=NULL), NULLP), (dict(table=NULL), NULLP), (dict(out=NULL), NULLP)]:
        assert fwd(**kw) == rc, kw
    size = lib.krsi_embedding_bwd_workspace_bytes
    # Positions, tokens, a start and a count per row, and two fp32 rows per piece of 16 (32 from 8193 tokens on).
    assert size(1000, 50, 24) >= 2 * 1000 * 4 + 2 * 50 * 4 + 63 * 2 * 24 * 4 and size(9000, 50, 24) >= 282 * 2 * 24 * 4
    assert size(0, 50, 24) > 0 and size(-1, 50, 24) == 0 and size(5, 0, 24) == 0
    okb = dict(dout=FAKE, tokens=FAKE, tb=8, dtable=FAKE, ws=FAKE, nb=1 << 30, n=4, V=10, D=8, pad=-1, scale=1.0, dt=0)

    def bwd(**kw):
        return lib.krsi_embedding_bwd(*{**okb, **kw}.values(), NULL)

    for kw, rc in bad + [(dict(dout=NULL), NULLP), (dict(tokens=NULL), NULLP), (dict(dtable=NULL), NULLP),
                         (dict(ws=NULL), WS), (dict(nb=16), WS), (dict(ws=FAKE + 8), ALIGN)]:
        assert bwd(**kw) == rc, kw


def test_linear_cross_entropy_arguments():
    lib = _hip.lib()
    size_f, size_b = lib.krsi_linear_cross_entropy_fwd_workspace_bytes, lib.krsi_linear_cross_entropy_bwd_workspace_bytes
    rows, k, v = 100, 128, 1000
    ok = dict(x=FAKE, w=FAKE, t=FAKE, tb=8, loss=FAKE, stats=FAKE, ws=FAKE, nb=size_f(rows, k, v), rows=rows, k=k, v=v,
              ignore=-100, red=1, dt=0)

    def fwd(**kw):
        return lib.krsi_linear_cross_entropy_fwd(*{**ok, **kw}.values(), NULL)

    bad = [(dict(dt=2), UNSUP), (dict(tb=1), UNSUP), (dict(red=3), UNSUP), (dict(red=-1), UNSUP), (dict(rows=-1), SHAPE),
           (dict(k=0), SHAPE), (dict(v=0), SHAPE), (dict(k=100), UNSUP), (dict(k=1 << 21), UNSUP),
           (dict(v=(1 << 23) + 1), UNSUP), (dict(rows=(1 << 23) + 1), UNSUP), (dict(rows=1 << 20, v=1 << 20), UNSUP),
           (dict(x=NULL), NULLP), (dict(w=NULL), NULLP), (dict(t=NULL), NULLP), (dict(stats=NULL), NULLP),
           (dict(x=FAKE + 2), ALIGN), (dict(w=FAKE + 8), ALIGN), (dict(ws=NULL), WS), (dict(nb=16), WS),
           (dict(ws=FAKE + 8), ALIGN)]
    for kw, rc in bad + [(dict(loss=NULL), NULLP)]:
        assert fwd(**kw) == rc, kw
    assert fwd(rows=0, red=0, x=NULL, t=NULL, loss=NULL) == 0 and fwd(rows=0, loss=NULL) == NULLP
    okb = dict(dout=FAKE, x=FAKE, w=FAKE, t=FAKE, tb=8, stats=FAKE, dx=FAKE, dw=FAKE, ws=FAKE, nb=size_b(rows, k, v),
               rows=rows, k=k, v=v, ignore=-100, red=1, dt=0)

    def bwd(**kw):
        return lib.krsi_linear_cross_entropy_bwd(*{**okb, **kw}.values(), NULL)

    for kw, rc in bad + [(dict(dout=NULL), NULLP), (dict(dx=NULL, dw=NULL), NULLP)]:
        assert bwd(**kw) == rc, kw
    assert bwd(rows=0, dw=NULL, x=NULL, dout=NULL) == 0
    # The forward keeps a pair of floats per row and 64 logits; the backward a piece of about 512 MB of 16-bit
    # gradients of logits at most, whatever rows x v is, and fp32 parts of dx.
    assert size_f(8192, 4096, 131072) >= 8192 * 131072 // 64 * 8
    assert 8192 * 32768 * 2 <= size_b(8192, 4096, 131072) < (512 << 20) + 4 * 8192 * 4096 * 4 + (4 << 20)
    assert size_b(100, 128, 1000) >= 100 * 1024 * 2 and size_f(0, 64, 64) == 0 and size_b(5, 100, 64) == 0
    for shape in ((1, 64, 1 << 23), (1 << 23, 64, 1), (1 << 20, 64, 300), (3, 1 << 20, 5), (70000, 64, 4000)):
        assert 0 < size_f(*shape) < 1 << 30 and 0 < size_b(*shape) < 40 << 30
    assert size_f(1 << 20, 4096, 131072) < 1 << 30  # rows whose pairs do not fit at once go in chunks


def test_python_functions_refuse_before_a_launch():
    x, tokens = torch.zeros(4, 192, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    w = torch.ones(64, dtype=torch.bfloat16)
    rope = Q.rope_table(4, 64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        Q.qk_norm_rope(x, w, w, rope, 1, 4, 1, 64, 1e-6)
    with pytest.raises(ValueError, match="constant"):
        Q.qk_norm_rope(x, w, w, rope.requires_grad_(True), 1, 4, 1, 64, 1e-6)
    with pytest.raises(ValueError, match="GPU"):
        E.embedding(tokens, x)
    with pytest.raises(ValueError, match="padding_idx"):
        E.embedding(tokens, x, padding_idx=4)
    with pytest.raises(ValueError, match="GPU"):
        L.linear_cross_entropy(x, x, tokens)
    with pytest.raises(ValueError, match="targets"):
        L.linear_cross_entropy(x.view(2, 2, 192), x, tokens)
    for bad in ((0, 8), (4, 7), (4, 0)):
        with pytest.raises(ValueError, match="rope_table"):
            Q.rope_table(*bad, device="cpu")


def test_rope_table_far_positions():
    """cos and sin of angles whose fp32 product would be off by whole fractions of a turn, to fp32's rounding."""
    import math

    t = Q.rope_table(1 << 17, 8, theta=500000.0, device="cpu")
    for p in (0, 1, 99999, (1 << 17) - 1):
        for i in range(4):
            angle = p * 500000.0 ** (-2 * i / 8)
            assert abs(t[p, i].item() - math.cos(angle)) < 1e-7 and abs(t[p, 4 + i].item() - math.sin(angle)) < 1e-7
