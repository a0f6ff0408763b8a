"""Products of 8-bit rows and INT4 weights (qw4_a8_linear, qw4_a8_linear_f32) against the
formula in 64 bits."""
import math

import pytest
import torch

from a8_util import product, random_rows, random_weights, sum_tolerance, to_layout

pytestmark = pytest.mark.gpu
BF16 = dict(dtype=torch.bfloat16, device="cuda")


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


@pytest.fixture(scope="module")
def ws(hip):
    w = hip.gemm_workspace_alloc(256 << 20)
    yield w
    hip.gemm_workspace_free(w)


# every row count around the 16- and 32-row blocks and the tiles' edges, odd column and
# group counts
SHAPES = [(1, 64, 128), (2, 64, 256), (3, 128, 128), (5, 192, 640), (8, 320, 384), (9, 1024, 1024), (15, 64, 1152),
          (16, 576, 512), (17, 64, 256), (24, 128, 1280), (31, 320, 128), (32, 64, 384), (33, 192, 640),
          (47, 256, 1024), (48, 1088, 256), (64, 64, 2048), (65, 320, 384), (77, 640, 1664), (96, 128, 128),
          (100, 64, 4096), (127, 512, 256), (128, 192, 384), (129, 64, 512), (160, 256, 256), (193, 448, 640),
          (224, 64, 128), (255, 320, 256), (256, 256, 256), (257, 64, 384), (300, 576, 896), (511, 128, 128),
          (513, 832, 256), (777, 64, 1024), (1025, 192, 128)]


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("T,n,k", SHAPES)
def test_integers_are_exact(hip, ws, T, n, k, space):
    """With scales of 1 and sums below 2^24 every value is the integer itself."""
    w, less, s = random_weights(hip, n, k, n + k, scale=1.0)
    g = torch.Generator().manual_seed(T)
    most = min(127, (1 << 24) // (15 * k))   # 15 most k <= 2^24
    q = torch.randint(-most, most + 1, (T, k), generator=g).to(torch.int8).cuda()
    rows = T + 3
    codes = torch.full((rows, k), 99, dtype=torch.int8, device="cuda")
    codes[:T] = to_layout(q)
    scale = torch.full((k // 128, rows), float("nan"), device="cuda")   # rows behind T count for nothing
    scale[:, :T] = 1.0
    y = torch.full((T + 2, n), -7.0, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws if space else None)
    torch.cuda.synchronize()
    want = torch.matmul(q.double(), less.t().contiguous())
    assert torch.equal(y[:T].double(), want)
    assert torch.all(y[T:] == -7.0)
    hip.awq_free(w)


@pytest.mark.parametrize("T,n,k", [(1, 320, 5120), (4, 64, 17408), (9, 192, 5120), (16, 128, 8320), (30, 64, 17408),
                                   (60, 192, 5120), (130, 320, 5120), (300, 256, 4096), (40, 64, 40960)])
@pytest.mark.parametrize("space", [False, True])
def test_f32(hip, ws, T, n, k, space):
    w, less, s = random_weights(hip, n, k, 7)
    q, scale = random_rows(T, k, 8)
    y = torch.zeros(T, n, device="cuda")
    codes = to_layout(q)
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws if space else None)
    torch.cuda.synchronize()
    want, size = product(q, scale, less, s)
    assert torch.all((y.double() - want).abs() <= sum_tolerance(size, k // 128))
    hip.awq_free(w)


def _act(v, act, up):
    """The activation in 64 bits; how far it moves by errors `tol` of its arguments, with
    its own roundings (exp: |v| 2^-24 and 2^-22; the erfc fit 1.2e-7; products)."""
    if act == "none":
        return v, lambda tol: tol
    if act == "silu":
        return v * torch.sigmoid(v), lambda tol: 1.1 * tol + (v.abs() + 16) * 2.0 ** -23 * (v * torch.sigmoid(v)).abs()
    if act == "gelu":
        y = v * torch.special.ndtr(v)
        return y, lambda tol: 1.13 * tol + (v * v + 32) * 2.0 ** -23 * y.abs()
    if act == "gelu_tanh":
        y = v * torch.sigmoid(math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3))
        return y, lambda tol: 1.13 * tol + (4 * v.abs() + v.abs() ** 3 + 32) * 2.0 ** -23 * y.abs()
    gate, u = v[:, :up], v[:, up:]
    y = gate * torch.sigmoid(gate) * u
    return y, lambda tol: (1.1 * u.abs() * tol[:, :up] + (gate * torch.sigmoid(gate)).abs() * tol[:, up:]
                           + (gate.abs() + 20) * 2.0 ** -23 * y.abs())


EPILOGUES = [("none", False, False), ("none", True, False), ("none", False, True), ("silu", True, True),
             ("gelu", True, False), ("gelu_tanh", False, True), ("swiglu", False, False), ("swiglu", True, True)]


@pytest.mark.parametrize("act,bias,residual", EPILOGUES)
@pytest.mark.parametrize("T,n,k", [(1, 384, 1024), (7, 128, 640), (16, 256, 5120), (21, 384, 384), (40, 640, 1280),
                                   (70, 128, 2048), (150, 384, 512), (260, 512, 896), (600, 1280, 256)])
@pytest.mark.parametrize("space", [False, True])
def test_epilogues(hip, ws, T, n, k, act, bias, residual, space):
    w, less, s = random_weights(hip, n, k, 3)
    q, scale = random_rows(T, k, 4)
    g = torch.Generator().manual_seed(5)
    up = n // 2 if act == "swiglu" else 0
    width = n - up
    b = torch.randn(n, generator=g).to(torch.bfloat16).cuda() if bias else None
    r = torch.randn(T, width, generator=g).to(torch.bfloat16).cuda() if residual else None
    y = torch.full((T + 1, width), 9.0, **BF16)
    codes = to_layout(q)
    hip.linear_w4a8(y, w, hip.a8_over(codes, scale), T, ws if space else None, bias=b,
                    act=getattr(hip, "ACT_" + act.upper()), residual=r)
    torch.cuda.synchronize()
    v, size = product(q, scale, less, s)
    tol = sum_tolerance(size, k // 128)
    if bias:
        v = v + b.double()
        tol = tol + 2.0 ** -24 * v.abs()
    want, moved = _act(v, act, up)
    tol = moved(tol)
    if residual:
        want = want + r.double()
    assert torch.all((y[:T].double() - want).abs() <= tol + (2.0 ** -8 + 2.0 ** -23) * want.abs() + 2.0 ** -23 * tol)
    assert torch.all(y[T:] == 9.0)
    if residual:   # over the residual itself
        z = r.clone()
        hip.linear_w4a8(z, w, hip.a8_over(codes, scale), T, ws if space else None, bias=b,
                        act=getattr(hip, "ACT_" + act.upper()), residual=z)
        torch.cuda.synchronize()
        assert torch.equal(z, y[:T])
    hip.awq_free(w)


@pytest.mark.parametrize("T", [1, 6, 16, 30, 100, 300])
def test_nonfinite_scales_stay_in_their_rows(hip, ws, T):
    n, k = 192, 1024
    w, less, s = random_weights(hip, n, k, 3)
    q, scale = random_rows(T, k, 4)
    codes = to_layout(q)
    clean = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(clean, w, hip.a8_over(codes, scale), T, ws)
    bad = scale.clone()
    rows = sorted({0, T // 2, T - 1})
    for i, row in enumerate(rows):
        bad[(3 * i) % 8, row] = float("nan")
    y = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, bad), T, ws)
    torch.cuda.synchronize()
    assert torch.all(torch.isnan(y[rows]))
    others = [t for t in range(T) if t not in rows]
    assert torch.equal(y[others], clean[others])
    hip.awq_free(w)


@pytest.mark.parametrize("T", [1, 5, 16, 20, 33, 64, 100, 200])
def test_extreme_codes_and_scales(hip, ws, T):
    """All codes at +-127 against all weights at +-15, scales from 2^-60 to 2^60."""
    n, k = 128, 640
    q = torch.where(torch.arange(T)[:, None] % 2 == 0, 127, -127).expand(T, k).to(torch.int8).cuda()
    shifts = torch.arange(k // 128)
    scale = torch.exp2((30.0 * shifts - 60)[:, None].expand(-1, T)).contiguous().cuda()
    nib = torch.full((n, k // 8), -1, dtype=torch.int32)      # q = 15
    nib[1::2] = 0                                              # q = 0
    zp = torch.full((n // 8, k // 128), -0x0F0F0F10, dtype=torch.int32)   # 0xF0F0F0F0: 0 for even rows, 15 for odd ones
    s = torch.ones(n, k // 128, dtype=torch.bfloat16)
    w = hip.awq_repack(nib.cuda(), s.cuda(), zp.cuda(), n, k)
    y = torch.zeros(T, n, device="cuda")
    codes = to_layout(q)
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws)
    torch.cuda.synchronize()
    sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0).double().cuda()
    one = 128 * 15 * q[:, :1].double() * sign
    want = one * scale.double().sum(0)[:, None]
    assert torch.all((y.double() - want).abs() <= (k // 128 * 2 + 8) * 2.0 ** -24 * want.abs())
    hip.awq_free(w)


def test_rows_do_not_depend_on_their_neighbours(hip, ws):
    """A call of more rows repeats a call's rows where both run the same kernel; across
    kernels the sums' order differs by roundings only."""
    n, k = 320, 5120
    w, less, s = random_weights(hip, n, k, 3)
    q, scale = random_rows(300, k, 4)
    codes = to_layout(q)
    want, size = product(q, scale, less, s)
    tol = sum_tolerance(size, k // 128)
    for T in (1, 16, 17, 64, 300):
        y = torch.zeros(T, n, device="cuda")
        hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws)
        z = torch.zeros(T, n, device="cuda")
        hip.linear_w4a8_f32(z, w, hip.a8_over(codes, scale), T, ws)
        torch.cuda.synchronize()
        assert torch.equal(y, z)
        assert torch.all((y.double() - want[:T]).abs() <= tol[:T])
    hip.awq_free(w)


def test_small_workspaces(hip):
    """A workspace too small to split tiles, or none of its bytes: the same values as without."""
    n, k, T = 128, 4096, 200
    w, less, s = random_weights(hip, n, k, 3)
    q, scale = random_rows(T, k, 4)
    codes = to_layout(q)
    a = hip.a8_over(codes, scale)
    y, z = torch.zeros(T, n, device="cuda"), torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, a, T)
    buf = torch.full((1 << 14,), 7, dtype=torch.uint8, device="cuda")
    for size in (0, 100, 1 << 12):
        hip.linear_w4a8_f32(z, w, a, T, hip.GemmWorkspace(buf.data_ptr(), size))
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.all(buf[size:] == 7)
    hip.awq_free(w)


@pytest.mark.parametrize("T", [33, 34, 47, 48, 49, 50, 63, 64])
@pytest.mark.parametrize("n,k", [(128, 128), (384, 1024), (4224, 640), (256, 2944), (128, 3200), (1280, 4992), (128, 5120),
                                 (17408, 640), (256, 5248)])
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_three_and_four_blocks_of_rows(hip, T, n, k, act):
    w, less, s = random_weights(hip, n, k, T)
    q, scale = random_rows(T + 2, k, n)
    codes = to_layout(q)
    a = hip.a8_over(codes, scale)   # of two rows more than the call's
    up = n // 2 if act == "swiglu" else 0
    y = torch.full((T + 1, n - up), 9.0, **BF16)
    f = torch.full((T + 1, n), 9.0, device="cuda")
    hip.linear_w4a8(y, w, a, T, None, act=getattr(hip, "ACT_" + act.upper()))
    hip.linear_w4a8_f32(f, w, a, T, None)
    torch.cuda.synchronize()
    v, size = product(q[:T], scale[:, :T], less, s)
    tol = sum_tolerance(size, k // 128)
    assert torch.all((f[:T].double() - v).abs() <= tol)
    want, moved = _act(v, act, up)
    tol = moved(tol)
    assert torch.all((y[:T].double() - want).abs() <= tol + (2.0 ** -8 + 2.0 ** -23) * want.abs() + 2.0 ** -23 * tol)
    assert torch.all(y[T:] == 9.0) and torch.all(f[T:] == 9.0)
    hip.awq_free(w)
