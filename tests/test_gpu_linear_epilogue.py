"""qw4_linear_epilogue against the formula in 64 bits: every activation with and
without bias and residual, one row to several tiles, through each path (decode and
verify kernels, prefill tiles whole and split), nothing written outside y."""
import math

import numpy as np
import pytest

from gpu_util import dev, repack_from_logical

pytestmark = pytest.mark.gpu

ACTS = ("none", "silu", "gelu", "gelu_tanh", "swiglu")


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


@pytest.fixture(scope="module")
def ws(hip):
    w = hip.gemm_workspace_alloc(256 << 20)
    yield w
    hip.gemm_workspace_free(w)


def activation(v, act):
    """f and a bound on |f'| near v, in 64 bits (torch, CPU)."""
    import torch

    if act == "none":
        return v
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
    g, u = v.chunk(2, dim=1)
    return g * torch.sigmoid(g) * u


def check(y, x, wq, bias, act, residual, rows, rounded, bits=8):
    """y[rows] against the formula. Errors: the product's (fp32 sums: K 2^-24 of the
    terms' absolute sum at most; weights rounded to `bits` bits: 2^-bits of each term, which
    over K random terms stays below 2^-bits sqrt(sum of squares) x 6), through the activation
    (|f'| <= 1.13 for the smooth ones; swiglu: each factor's error times the other), f's
    own few ulp, and the rounding to bf16 (half a step: 2^-8)."""
    import torch

    xf = x[rows].double()
    v = xf @ wq.t()
    sumabs = xf.abs() @ wq.abs().t()
    ev = 2.0 ** -24 * (wq.shape[1] ** 0.5 + 8) * sumabs
    if rounded:
        ev = ev + 6 * 2.0 ** -bits * ((xf ** 2) @ (wq ** 2).t()).sqrt()
    if bias is not None:
        v = v + bias.double()
        ev = ev + 2.0 ** -24 * v.abs()
    f = activation(v, act)
    if act == "swiglu":
        (g, u), (eg, eu) = v.chunk(2, dim=1), ev.chunk(2, dim=1)
        ef = 1.13 * (eg * u.abs() + eg * eu) + (g * torch.sigmoid(g)).abs() * eu + 2.0 ** -21 * f.abs()
    else:
        ef = 1.13 * ev + 2.0 ** -20 * f.abs()
    r = 0 if residual is None else residual[rows].double()
    ref = f + r
    ef = ef + 2.0 ** -24 * ref.abs()
    tol = 2.0 ** -8 * (ref.abs() + ef) + ef + 1e-30
    err = (y[rows].double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


def make(hip, orc, N, K, seed):
    import torch

    q, zp, s = orc.gen_weights(N, K, seed=seed)
    w = repack_from_logical(hip, orc, q, zp, s, "ct")
    sf = (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    wq = (q.astype(np.float64) - np.repeat(zp, 128, axis=1)) * np.repeat(sf, 128, axis=1)
    return w, torch.from_numpy(wq)


def bf(t):
    import torch

    return t.to(torch.bfloat16)


def run(hip, w, x, T, scratch, space, bias, act, residual, alias):
    import torch

    width = w.out_f // 2 if act == "swiglu" else w.out_f
    big = torch.full((T + 2, width), 7.0, dtype=torch.bfloat16, device="cuda")
    y = big[1:T + 1]
    r = residual.cuda() if residual is not None else None
    if alias:
        y.copy_(r)
        r = y
    hip.linear_epilogue_w4a16(y, w, x.cuda(), T, scratch, space,
                              bias=bias.cuda() if bias is not None else None,
                              act=getattr(hip, "ACT_" + act.upper()), residual=r)
    torch.cuda.synchronize()
    assert (big[0] == 7.0).all() and (big[T + 1] == 7.0).all()
    return y.cpu()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("N,K", [(128, 128), (384, 640), (1152, 2176), (5120, 4096)])
def test_epilogue(hip, orc, ws, N, K, act):
    import torch

    g = torch.Generator().manual_seed(N + K)
    w, wq = make(hip, orc, N, K, N + K)
    scratch = hip.gemv_scratch_alloc(K, N, 128, 16)
    width = N // 2 if act == "swiglu" else N
    for T in (1, 2, 9, 16, 17, 33, 100, 300):
        x = bf(torch.randn(T, K, generator=g) * (8.0 / K ** 0.5))
        rows = list(range(T)) if T <= 17 else sorted({0, T - 1, T // 2, 31, 32, T // 3})
        for bias, residual in ((False, False), (True, False), (False, True), (True, True)):
            b = bf(torch.randn(N, generator=g)) if bias else None
            r = bf(torch.randn(T, width, generator=g)) if residual else None
            for s in (scratch, None):
                for space in (None, ws):
                    print(f"epilogue {N}x{K} T={T} {act} bias={bias} res={residual} scratch={s is not None} "
                          f"ws={space is not None}", flush=True)
                    y = run(hip, w, x, T, s, space, b, act, r, alias=residual and bias)
                    small = s is not None and T <= hip.linear_max_t(w)
                    # a gated product with a workspace has fp16 operands
                    bits = 11 if act == "swiglu" and space is not None else 8
                    check(y, x, wq, b, act, r, rows, rounded=not small, bits=bits)
    hip.awq_free(w)
    hip.gemv_scratch_free(scratch)


# every tile height, whole and with each split schedule (see test_gpu_gemm_rows.py's plans)
HEIGHTS = [(60, 33280, 384), (70, 33280, 384), (98, 33280, 384), (133, 33280, 384), (161, 33280, 384),
           (196, 33280, 384), (450, 22528, 384), (500, 9472, 8448), (900, 17408, 4096), (133, 9984, 5120),
           (60, 70656, 2048), (300, 34944, 2048), (520, 26624, 2048), (1100, 17408, 5120),
           (70, 256, 2048), (133, 256, 2048), (400, 256, 2048), (259, 256, 2176), (700, 2816, 2176),
           (400, 2816, 8192), (450, 5760, 8192)]


@pytest.mark.parametrize("T,N,K", HEIGHTS)
def test_epilogue_tiles(hip, orc, ws, T, N, K):
    """The plain product of the same call (qw4_gemm), through the epilogue's formula:
    both sum in the same order, so without bias, activation or residual they are equal
    bit for bit, and gated -- fp16 operands -- they are the product's halves up to its
    rounding and that of its bf16 weights: 2^-8 of each term, over K random terms below 6
    times 2^-8 of the root of their squares' sum."""
    import torch

    G = K // 128
    q = torch.empty(K // 8 * N, dtype=torch.int32, device="cuda")
    s = torch.empty(G * N, dtype=torch.int16, device="cuda")
    z = torch.empty(G * N // 8, dtype=torch.int32, device="cuda")
    hip.gen_awq_k(q, s, z, N, K, N + K, 3)
    w = hip.awq_alloc_fused(N, K)
    hip.awq_repack_awq_into(w, 0, q, s, z, N, hip.LAYOUT_AWQ_K)
    g = torch.Generator().manual_seed(T)
    x = bf(torch.randn(T, K, generator=g) * (8.0 / K ** 0.5)).cuda()
    bias = bf(torch.randn(N, generator=g)).cuda()
    half = bf(torch.randn(T, N // 2, generator=g)).cuda()
    print(f"epilogue tiles {T} {N}x{K}", flush=True)
    plain = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    hip.gemm_w4a16(plain, w, x, T, ws)
    same = torch.empty_like(plain)
    hip.linear_epilogue_w4a16(same, w, x, T, None, ws)
    full = torch.empty_like(plain)
    hip.linear_epilogue_w4a16(full, w, x, T, None, ws, bias=bias, act=hip.ACT_SILU, residual=plain)
    glu = torch.empty(T, N // 2, dtype=torch.bfloat16, device="cuda")
    hip.linear_epilogue_w4a16(glu, w, x, T, None, ws, bias=bias, act=hip.ACT_SWIGLU, residual=half)
    torch.cuda.synchronize()
    assert torch.equal(same, plain)
    p = plain.double()
    ep = 2.0 ** -8 * p.abs()          # the plain product's own rounding
    v = p + bias.double()
    f = v * torch.sigmoid(v) + p
    tol = 1.13 * ep + 2.0 ** -8 * (f.abs() + 2 * ep) + 1e-6
    assert ((full.double() - f).abs() <= tol).all()
    wd = torch.empty(N, K, dtype=torch.bfloat16, device="cuda")
    hip.w4a16_dequant_rows(wd, w, 0, N)
    wd = wd.float() ** 2
    ep = ep + 6 * 2.0 ** -8 * (x.float() ** 2 @ wd.t()).sqrt().double()
    (a, u), (ea, eu) = v.chunk(2, dim=1), ep.chunk(2, dim=1)
    sa = a * torch.sigmoid(a)
    f = sa * u + half.double()
    e = 1.13 * ea * (u.abs() + eu) + sa.abs() * eu
    assert ((glu.double() - f).abs() <= e + 2.0 ** -8 * (f.abs() + e) + 1e-6).all()
    hip.awq_free(w)


@pytest.mark.parametrize("T", [130, 1000])
def test_gated_range(hip, orc, ws, T):
    """The fp16 operands of a gated product over bf16's range: rows and weight rows of
    very large and very small values, a scale far above the others of its row, rows of
    zeros; rows with Inf or NaN are NaN or Inf at every output and leave the others alone."""
    import torch

    I, K = 320, 1024
    N = 2 * I
    q, zp, s = orc.gen_weights(N, K, seed=T)
    sf = (s.astype(np.uint32) << 16).view(np.float32).copy()
    g = torch.Generator().manual_seed(T)
    # gate rows keep their size (silu would saturate), up rows spread over 2^-90 .. 2^60
    sf[I:] *= 2.0 ** np.random.default_rng(T).integers(-90, 60, (I, 1))
    sf[I::7, 3] *= 2.0 ** 20
    s = (sf.view(np.uint32) >> 16).astype(np.uint16)
    w = repack_from_logical(hip, orc, q, zp, s, "ct")
    sd = (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    wq = torch.from_numpy((q.astype(np.float64) - np.repeat(zp, 128, axis=1)) * np.repeat(sd, 128, axis=1))
    x = torch.randn(T, K, generator=g) * (8.0 / K ** 0.5)
    x[1::9] *= 2.0 ** -60
    x[2::9] = 0
    x[3::9, ::2] *= 2.0 ** -30
    x[4::9, 5] = 2.0 ** 10
    x = bf(x)
    bad = x.clone()
    bad[7, 3], bad[60, 9], bad[61, 0] = float("inf"), float("nan"), -float("inf")
    for xi in (x, bad):
        print(f"gated range T={T}", flush=True)
        y = torch.full((T + 2, I), 7.0, dtype=torch.bfloat16, device="cuda")
        hip.linear_epilogue_w4a16(y[1:T + 1], w, xi.cuda(), T, None, ws, act=hip.ACT_SWIGLU)
        torch.cuda.synchronize()
        assert (y[0] == 7.0).all() and (y[T + 1] == 7.0).all()
        got = y[1:T + 1].cpu()
        if xi is bad:
            hit = torch.zeros(T, dtype=torch.bool)
            hit[[7, 60, 61]] = True
            assert not torch.isfinite(got[60]).any()
            assert torch.equal(got[~hit], clean[~hit])
        else:
            clean = got
            check(got, x, wq, None, "swiglu", None, list(range(0, T, 3)) + [1, 2, 4, T - 1], rounded=True, bits=11)
    hip.awq_free(w)
