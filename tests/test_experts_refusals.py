"""Argument checks of the expert layer's calls: status codes before any launch
(CPU only; the pointers are never dereferenced)."""
import ctypes as C

import pytest

P = C.c_void_p


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def _plan(hip, experts=8, pairs=64):
    return hip.ExpertPlan(0x1000, 0x2000, 0x3000, experts, pairs)


def test_route_refusals(hip):
    L = hip.lib()
    ids, w, x = P(0x10000), P(0x20000), P(0x30000)

    def route(T=4, E=8, k=2, plan=None, ids=ids, w=w, x=x, f=L.qw4_route):
        return f(ids, w, C.byref(plan) if plan is not None else None, x, T, E, k, 1, None)

    for f in (L.qw4_route, L.qw4_route_f32):
        assert route(T=-1, f=f) == hip.QW4_ERR_M
        assert route(E=0, f=f) == hip.QW4_ERR_SHAPE
        assert route(E=1025, f=f) == hip.QW4_ERR_SHAPE
        assert route(k=0, f=f) == hip.QW4_ERR_SHAPE
        assert route(k=9, f=f) == hip.QW4_ERR_SHAPE          # more than there are
        assert route(E=64, k=17, f=f) == hip.QW4_ERR_SHAPE
        assert route(T=1 << 30, f=f) == hip.QW4_ERR_SHAPE    # pair numbers beyond 32 bits
        assert route(ids=None, f=f) == hip.QW4_ERR_NULL
        assert route(w=None, f=f) == hip.QW4_ERR_NULL
        assert route(x=None, f=f) == hip.QW4_ERR_NULL
        assert route(plan=_plan(hip, experts=9), f=f) == hip.QW4_ERR_SHAPE
        assert route(plan=_plan(hip, pairs=7), f=f) == hip.QW4_ERR_SCRATCH
        bad = _plan(hip)
        bad.tokens = None
        assert route(plan=bad, f=f) == hip.QW4_ERR_NULL
        assert route(T=0, ids=None, w=None, x=None, f=f) == hip.QW4_OK


def test_plan_and_combine_refusals(hip):
    L = hip.lib()
    p = _plan(hip)
    assert L.qw4_plan_alloc(None, 8, 8) == hip.QW4_ERR_NULL
    for e, n in ((0, 8), (1025, 8), (8, 0)):
        assert L.qw4_plan_alloc(C.byref(hip.ExpertPlan()), e, n) == hip.QW4_ERR_SHAPE
    assert L.qw4_plan_free(None) == hip.QW4_ERR_NULL
    ids = P(0x10000)
    assert L.qw4_route_ids(C.byref(p), ids, -1, 2, None) == hip.QW4_ERR_M
    assert L.qw4_route_ids(C.byref(p), ids, 4, 17, None) == hip.QW4_ERR_SHAPE
    assert L.qw4_route_ids(C.byref(p), None, 4, 2, None) == hip.QW4_ERR_NULL
    assert L.qw4_route_ids(C.byref(p), ids, 33, 2, None) == hip.QW4_ERR_SCRATCH
    assert L.qw4_route_ids(None, ids, 4, 2, None) == hip.QW4_ERR_NULL

    def combine(T=4, k=2, dim=64, out=0x10000, y=0x20000, w=0x30000, r=None, plan=p):
        return L.qw4_combine(P(out), P(y), C.byref(plan), P(w), T, k, dim, P(r), None)

    assert combine(T=-1) == hip.QW4_ERR_M
    assert combine(k=0) == hip.QW4_ERR_SHAPE
    assert combine(k=17) == hip.QW4_ERR_SHAPE
    assert combine(dim=60) == hip.QW4_ERR_SHAPE
    assert combine(dim=0) == hip.QW4_ERR_SHAPE
    assert combine(T=33) == hip.QW4_ERR_SCRATCH
    for name in ("out", "y", "w"):
        assert combine(**{name: None}) == hip.QW4_ERR_NULL
    for name in ("out", "y", "r"):
        assert combine(**{name: 0x40008}) == hip.QW4_ERR_ALIGN
    assert combine(T=0, out=None, y=None, w=None) == hip.QW4_OK


def test_binding_checks(hip):
    import torch

    a = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError):
        hip.expert_plan_over(a, a, a[:4])
    with pytest.raises(ValueError):
        hip.expert_plan_over(a, a.long(), a.long())
    with pytest.raises(ValueError):
        hip.expert_plan_over(a, a[::2], a[::2])
    with pytest.raises(ValueError):   # ids too small for T top_k
        hip.route_experts(a, torch.zeros(16), torch.zeros(64, dtype=torch.bfloat16), 8, 8, 2, True, stream=0)
    with pytest.raises(hip.W4A16Error) as e:
        hip.route_experts(0x1000, 0x2000, 0x3000, 1, 8, 9, True, stream=0)
    assert e.value.status == hip.QW4_ERR_SHAPE


def _weights(hip, out_f=256, in_f=512):
    w = hip.W4A16Weights()
    w.qweight, w.scale, w.zeros = 0x1000, 0x2000, 0x3000
    w.out_f, w.in_f, w.group_size, w.num_groups = out_f, in_f, 128, in_f // 128
    return w


def test_linear_epilogue_refusals(hip):
    L = hip.lib()
    w = _weights(hip)

    def call(T=4, act=0, y=0x10000, x=0x20000, b=None, r=None, w=w, s=None):
        return L.qw4_linear_epilogue(P(y), C.byref(w) if w else None, P(x), T, P(b), act, P(r),
                                     C.byref(s) if s else None, None, None)

    assert call(T=0) == hip.QW4_ERR_M
    assert call(y=None) == hip.QW4_ERR_NULL
    assert call(x=None) == hip.QW4_ERR_NULL
    assert call(w=None) == hip.QW4_ERR_NULL
    assert call(act=5) == hip.QW4_ERR_ACT
    assert call(act=-1) == hip.QW4_ERR_ACT
    assert call(act=hip.ACT_SWIGLU, w=_weights(hip, out_f=192)) == hip.QW4_ERR_SHAPE
    assert call(w=_weights(hip, out_f=200)) == hip.QW4_ERR_SHAPE
    for name in ("y", "x", "b", "r"):
        assert call(**{name: 0x40008}) == hip.QW4_ERR_ALIGN
    assert call(T=1 << 23) == hip.QW4_ERR_SHAPE   # x beyond 32-bit offsets


def test_gemm_grouped_refusals(hip):
    L = hip.lib()
    w = _weights(hip, out_f=1024)

    def call(pairs=16, x_rows=16, gather=0, act=0, y=0x10000, x=0x20000, b=None, w=w, plan=_plan(hip)):
        return L.qw4_gemm_grouped(P(y), C.byref(w) if w else None, P(x), x_rows,
                                  C.byref(plan) if plan else None, pairs, gather, P(b), act, None, None)

    assert call(w=None) == hip.QW4_ERR_NULL
    assert call(plan=None) == hip.QW4_ERR_NULL
    assert call(y=None) == hip.QW4_ERR_NULL
    assert call(x=None) == hip.QW4_ERR_NULL
    assert call(pairs=-1) == hip.QW4_ERR_M
    assert call(pairs=65, x_rows=65) == hip.QW4_ERR_SCRATCH
    assert call(x_rows=15) == hip.QW4_ERR_SHAPE                       # in order: a row for each position
    assert call(gather=1, x_rows=0) == hip.QW4_ERR_SHAPE
    assert call(act=7) == hip.QW4_ERR_ACT
    assert call(act=hip.ACT_SWIGLU, w=_weights(hip, out_f=512)) == hip.QW4_ERR_SHAPE   # 64 rows an expert
    assert call(plan=_plan(hip, experts=7)) == hip.QW4_ERR_SHAPE      # 1024 rows are no 7 experts
    assert call(plan=_plan(hip, experts=32)) == hip.QW4_ERR_SHAPE     # 32 rows an expert
    assert call(plan=_plan(hip, experts=0)) == hip.QW4_ERR_SHAPE
    assert call(gather=1, x_rows=1 << 22) == hip.QW4_ERR_SHAPE        # 4 GiB of x
    bad = _plan(hip)
    bad.tokens = None
    assert call(gather=1, plan=bad) == hip.QW4_ERR_NULL
    bad.offsets = None
    assert call(plan=bad) == hip.QW4_ERR_NULL
    for name in ("y", "x", "b"):
        assert call(**{name: 0x40008}) == hip.QW4_ERR_ALIGN
    assert call(pairs=0, y=None, x=None) == hip.QW4_OK


def test_tune_grouped(hip):
    for form in (-1, 6):
        with pytest.raises(hip.W4A16Error):
            hip.tune_grouped(form)
    hip.tune_grouped(4)
    hip.tune_grouped()


def test_epilogue_workspace(hip):
    w = _weights(hip, out_f=256, in_f=512)
    # x in 16 bits, an exponent a row and a weight row, each from a multiple of 256 bytes
    assert hip.epilogue_workspace(w, 100) == 100 * 512 * 2 + 512 + 1024
    assert hip.epilogue_workspace(w, 0) == 1024
    assert hip.epilogue_workspace(w, -1) == 0
    assert hip.lib().qw4_epilogue_workspace(None, 4) == 0
