"""Argument checks of the calls around 8-bit rows and of the log probabilities: status
codes before any launch (CPU only; the pointers are never dereferenced)."""
import ctypes as C

import pytest

P = C.c_void_p


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def _a8(hip, rows=32, in_f=512):
    return hip.A8Rows(0x1000, 0x2000, rows, in_f)


def _weights(hip, out_f=256, in_f=512):
    w = hip.W4A16Weights()
    w.qweight, w.scale, w.zeros = 0x1000, 0x2000, 0x3000
    w.out_f, w.in_f, w.group_size, w.num_groups = out_f, in_f, 128, in_f // 128
    return w


def test_alloc_refusals(hip):
    L = hip.lib()
    assert L.qw4_a8_alloc(None, 4, 128) == hip.QW4_ERR_NULL
    for rows, in_f in ((0, 128), (-1, 128), (4, 0), (4, 100), (4, -128)):
        assert L.qw4_a8_alloc(C.byref(hip.A8Rows()), rows, in_f) == hip.QW4_ERR_SHAPE
    assert L.qw4_a8_free(None) == hip.QW4_ERR_NULL
    assert L.qw4_a8_free(C.byref(hip.A8Rows())) == hip.QW4_OK


def _bad_rows(hip):
    """(8-bit rows, status) of structs that no call takes."""
    out = []
    for field, value, st in (("q", None, hip.QW4_ERR_NULL), ("scale", None, hip.QW4_ERR_NULL),
                             ("in_f", 0, hip.QW4_ERR_SHAPE), ("in_f", 500, hip.QW4_ERR_SHAPE),
                             ("max_rows", 0, hip.QW4_ERR_SHAPE), ("q", 0x1008, hip.QW4_ERR_ALIGN),
                             ("scale", 0x2002, hip.QW4_ERR_ALIGN)):
        a = _a8(hip)
        setattr(a, field, value)
        out.append((a, st))
    return out


def test_quantize_refusals(hip):
    L = hip.lib()

    def call(a=_a8(hip), x=0x10000, ld=512, T=4):
        return L.qw4_a8_quantize(C.byref(a) if a else None, P(x), ld, T, None)

    assert call(T=-1) == hip.QW4_ERR_M
    assert call(a=None) == hip.QW4_ERR_NULL
    assert call(x=None) == hip.QW4_ERR_NULL
    assert call(ld=504) == hip.QW4_ERR_SHAPE      # rows that overlap
    assert call(ld=516) == hip.QW4_ERR_SHAPE      # rows off 16 bytes
    assert call(x=0x10008) == hip.QW4_ERR_ALIGN
    assert call(T=33) == hip.QW4_ERR_SCRATCH
    for a, st in _bad_rows(hip):
        assert call(a=a) == st
    assert call(T=0, x=None) == hip.QW4_OK


def test_rmsnorm_refusals(hip):
    L = hip.lib()

    def call(a=_a8(hip), o=0x10000, h=0x20000, r=0x30000, w=0x40000, T=4):
        return L.qw4_a8_rmsnorm(C.byref(a) if a else None, P(o), P(h), P(r), P(w), T, 1e-6, None)

    assert call(T=-1) == hip.QW4_ERR_M
    assert call(T=33) == hip.QW4_ERR_SCRATCH
    for name in ("a", "o", "h", "w"):
        assert call(**{name: None}) == hip.QW4_ERR_NULL
    for name in ("o", "h", "r", "w"):
        assert call(**{name: 0x50008}) == hip.QW4_ERR_ALIGN
    for a, st in _bad_rows(hip):
        assert call(a=a) == st
    assert call(T=0, o=None, h=None, w=None) == hip.QW4_OK


def test_dequant_refusals(hip):
    L = hip.lib()

    def call(a=_a8(hip), dst=0x10000, row0=0, n=4):
        return L.qw4_a8_dequant_rows(P(dst), C.byref(a) if a else None, row0, n, None)

    assert call(a=None) == hip.QW4_ERR_NULL
    assert call(dst=None) == hip.QW4_ERR_NULL
    assert call(dst=0x10008) == hip.QW4_ERR_ALIGN
    for row0, n in ((0, -1), (-1, 4), (0, 33), (30, 3), (2**31 - 1, 1), (1, 2**31 - 1)):
        assert call(row0=row0, n=n) == hip.QW4_ERR_SHAPE
    for a, st in _bad_rows(hip):
        assert call(a=a) == st
    assert call(n=0, dst=None) == hip.QW4_OK


def test_linear_refusals(hip):
    L = hip.lib()
    w = _weights(hip)

    def call(y=0x10000, w=w, a=_a8(hip), T=4, b=None, act=0, r=None):
        return L.qw4_a8_linear(P(y), C.byref(w) if w else None, C.byref(a) if a else None, T, P(b), act, P(r),
                               None, None)

    def f32(y=0x10000, w=w, a=_a8(hip), T=4):
        return L.qw4_a8_linear_f32(P(y), C.byref(w) if w else None, C.byref(a) if a else None, T, None, None)

    for f in (call, f32):
        assert f(T=0) == hip.QW4_ERR_M
        assert f(T=-1) == hip.QW4_ERR_M
        assert f(T=33) == hip.QW4_ERR_SCRATCH
        for name in ("y", "w", "a"):
            assert f(**{name: None}) == hip.QW4_ERR_NULL
        assert f(y=0x10008) == hip.QW4_ERR_ALIGN
        assert f(a=_a8(hip, in_f=640)) == hip.QW4_ERR_SHAPE      # of another product
        assert f(w=_weights(hip, out_f=200)) == hip.QW4_ERR_SHAPE
        wide = (1 << 23) + 128
        assert f(w=_weights(hip, in_f=wide), a=_a8(hip, in_f=wide)) == hip.QW4_ERR_SHAPE
        for a, st in _bad_rows(hip):
            assert f(a=a) == st
    assert call(act=5) == hip.QW4_ERR_ACT
    assert call(act=-1) == hip.QW4_ERR_ACT
    assert call(act=hip.ACT_SWIGLU, w=_weights(hip, out_f=192)) == hip.QW4_ERR_SHAPE
    assert call(b=0x40008) == hip.QW4_ERR_ALIGN
    assert call(r=0x40008) == hip.QW4_ERR_ALIGN


def test_logprobs_refusals(hip):
    L = hip.lib()

    def call(f=L.qw4_logprobs, lp=0x10000, e=0x20000, ids=0x30000, top=0x40000, x=0x50000, ld=4096, t=0x60000,
             T=4, n=4096, asked=1, k=5, ws=None):
        return f(P(lp), P(e), P(ids), P(top), P(x), ld, P(t), T, n, asked, k, C.byref(ws) if ws else None, None)

    for f, odd in ((L.qw4_logprobs, 0x50001), (L.qw4_logprobs_f32, 0x50002)):
        assert call(f, T=-1) == hip.QW4_ERR_M
        assert call(f, n=0) == hip.QW4_ERR_SHAPE
        assert call(f, ld=4095) == hip.QW4_ERR_SHAPE
        assert call(f, asked=-1) == hip.QW4_ERR_SHAPE
        assert call(f, k=-1) == hip.QW4_ERR_SHAPE
        assert call(f, k=33) == hip.QW4_ERR_SHAPE
        for name in ("x", "lp", "t", "ids", "top"):
            assert call(f, **{name: None}) == hip.QW4_ERR_NULL
        assert call(f, x=odd) == hip.QW4_ERR_ALIGN
        for name in ("lp", "e", "ids", "top", "t"):
            assert call(f, **{name: 0x70002}) == hip.QW4_ERR_ALIGN
        assert call(f, T=0, x=None, lp=None, t=None, ids=None, top=None) == hip.QW4_OK
        # a call that splits its rows needs its workspace
        need = hip.logprobs_workspace(1, 248320, 5)
        assert need > 0
        big = dict(T=1, n=248320, ld=248320)
        assert call(f, **big) == hip.QW4_ERR_SCRATCH
        assert call(f, ws=hip.GemmWorkspace(None, need), **big) == hip.QW4_ERR_SCRATCH
        assert call(f, ws=hip.GemmWorkspace(0x80000, need - 1), **big) == hip.QW4_ERR_SCRATCH
        assert call(f, ws=hip.GemmWorkspace(0x80008, need), **big) == hip.QW4_ERR_ALIGN
    for bad in ((0, 4096, 5), (4, 0, 5), (4, 4096, -1), (4, 4096, 33)):
        assert hip.logprobs_workspace(*bad) == 0


def test_binding_checks(hip):
    import torch

    q, s = torch.zeros(8, 256, dtype=torch.int8), torch.zeros(2, 8)
    with pytest.raises(ValueError):
        hip.a8_over(q.float(), s)
    with pytest.raises(ValueError):
        hip.a8_over(q, s[:1])
    with pytest.raises(ValueError):
        hip.a8_over(q[:, ::2], s)
    a = _a8(hip)
    x = torch.zeros(4, 512, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        hip.quantize_a8(a, x, 5, stream=0)
    with pytest.raises(ValueError):
        hip.quantize_a8(a, x.half(), 4, stream=0)
    with pytest.raises(ValueError):
        hip.quantize_a8(a, torch.zeros(4, 600, dtype=torch.bfloat16)[:, :500], 4, stream=0)
    with pytest.raises(ValueError):
        hip.quantize_a8(a, torch.zeros(512, 4, dtype=torch.bfloat16).t(), 4, stream=0)
    with pytest.raises(ValueError):
        hip.rmsnorm_a8(a, x, x[0], 5, 1e-6, stream=0)
    w = _weights(hip)
    with pytest.raises(ValueError):
        hip.linear_w4a8(torch.zeros(4, 256), w, a, 4, stream=0)
    with pytest.raises(ValueError):
        hip.linear_w4a8_f32(torch.zeros(3, 256), w, a, 4, stream=0)
    with pytest.raises(ValueError):
        hip.logprobs(torch.zeros(4), torch.zeros(4, 100), torch.zeros(4, dtype=torch.int64), 4, 100, stream=0)
    with pytest.raises(ValueError):
        hip.logprobs(torch.zeros(4), torch.zeros(4, 99), torch.zeros(4, dtype=torch.int32), 4, 100, stream=0)
    for targets in (0x3000, torch.zeros(4, 1, 1, dtype=torch.int32), torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ValueError):   # how many a row?
            hip.logprobs(torch.zeros(4), torch.zeros(4, 100), targets, 4, 100, stream=0)
    with pytest.raises(ValueError):   # rows of two targets, values of one
        hip.logprobs(torch.zeros(4), torch.zeros(4, 100), torch.zeros(8, 2, dtype=torch.int32), 4, 100, stream=0)
    with pytest.raises(hip.W4A16Error) as e:
        hip.logprobs(0x1000, 0x2000, 0x3000, 4, 100, top_k=40, top_ids=0x4000, top_logprobs=0x5000, asked=1, stream=0)
    assert e.value.status == hip.QW4_ERR_SHAPE
