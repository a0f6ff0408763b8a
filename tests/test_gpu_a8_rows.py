"""Rows of activations in 8 bits (qw4_a8_quantize, qw4_a8_rmsnorm, qw4_a8_dequant_rows)
against the formulas in 64 bits."""
import pytest
import torch

from a8_util import from_layout

pytestmark = pytest.mark.gpu
GROUP = 128
BF16 = dict(dtype=torch.bfloat16, device="cuda")


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


def _buffers(hip, rows, dim):
    """8-bit rows over tensors full of a pattern, so that what is not written shows."""
    q = torch.full((rows, dim), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((dim // GROUP, rows), -3.0, device="cuda")
    return hip.a8_over(q, scale), q, scale


def _hidden(rows, dim, seed):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(0.5 * torch.randn(dim, generator=g))
    return (torch.randn(rows, dim, generator=g) * spread).to(torch.bfloat16).cuda()


def _check(y, q, scale, T, scale_tol):
    """Codes and scales of the first T rows against the values y [T][dim] in 64 bits; rows
    behind them are as they were."""
    torch.cuda.synchronize()
    assert torch.all(q[T:] == 77) and torch.all(scale[:, T:] == -3.0)
    codes = from_layout(q[:T]).double().view(T, -1, GROUP)
    v = y.view(T, -1, GROUP)
    top = v.abs().amax(2)
    assert torch.all((scale[:, :T].t().double() - top / 127).abs() <= scale_tol * top / 127 + 1e-45)
    # the quotient's roundings (inverse, product: 2^-24 of up to 127 each; the values' own
    # few), beside the half that a code is off by
    exact = v * torch.where(top > 0, 127 / top, top)[:, :, None]
    assert torch.all((codes - exact).abs() <= 0.5 + 127 * 8 * 2.0 ** -24)
    assert codes.abs().max() <= 127


@pytest.mark.parametrize("rows,dim,T", [(1, 128, 1), (5, 128, 3), (4, 384, 4), (3, 640, 2), (9, 5120, 9), (16, 17408, 16),
                                        (700, 256, 650), (1, 33024, 1), (70, 4096, 70)])
def test_quantize(hip, rows, dim, T):
    x = _hidden(rows, dim, dim + T)
    a, q, scale = _buffers(hip, rows, dim)
    hip.quantize_a8(a, x, T)
    _check(x[:T].double(), q, scale, T, 2.0 ** -24)
    y = torch.full((rows, dim), 5.0, **BF16)
    hip.a8_dequant_rows(y, a, 0, T)
    torch.cuda.synchronize()
    want = from_layout(q[:T]).double() * torch.repeat_interleave(scale[:, :T].t().double(), GROUP, dim=1)
    assert torch.all((y[:T].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -24) * want.abs())
    assert torch.all(y[T:] == 5.0)
    if T > 2:   # rows in the middle
        hip.a8_dequant_rows(y, a, 1, T - 2)
        torch.cuda.synchronize()
        assert torch.all((y[:T - 2].double() - want[1:T - 1]).abs() <= (2.0 ** -8 + 2.0 ** -24) * want[1:T - 1].abs())


@pytest.mark.parametrize("first,beside", [(0, 8), (8, 24), (128, 1000)])
def test_quantize_columns_of_a_buffer(hip, first, beside):
    T, dim = 33, 640
    x = _hidden(T, first + dim + beside, 3)
    a, q, scale = _buffers(hip, T, dim)
    hip.quantize_a8(a, x[:, first:first + dim], T)
    _check(x[:, first:first + dim].double(), q, scale, T, 2.0 ** -24)


def test_codes_of_exact_values(hip):
    """Codes times a power of two come back as they were."""
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(-127, 128, (12, 1024), generator=g)
    codes.view(12, 8, 128)[:, :, 5] = 127
    exponents = torch.randint(-20, 20, (12, 8), generator=g)
    step = torch.exp2(exponents.double())
    x = (codes.double().view(12, 8, 128) * step[:, :, None]).view(12, 1024).to(torch.bfloat16).cuda()
    a, q, scale = _buffers(hip, 12, 1024)
    hip.quantize_a8(a, x, 12)
    torch.cuda.synchronize()
    assert torch.equal(from_layout(q).cpu(), codes.to(torch.int8))
    assert torch.equal(scale.t().double().cpu(), step)


def test_zero_small_and_nonfinite_groups(hip):
    x = _hidden(8, 512, 9)
    x[0, :128] = 0
    x[1, 128:256] = -0.0
    x[2, :128] = 2.0 ** -101
    x[3, 256:384] = 2.0 ** -100
    x[4, 7] = float("nan")
    x[5, 300] = float("inf")
    x[6, 500] = float("-inf")
    x[7, :] = 3.3e38
    a, q, scale = _buffers(hip, 8, 512)
    hip.quantize_a8(a, x, 8)
    torch.cuda.synchronize()
    s, codes = scale.t().cpu(), from_layout(q).cpu().view(8, 4, 128)
    assert s[0, 0] == 0 and not codes[0, 0].any()
    assert s[1, 1] == 0 and not codes[1, 1].any()
    assert s[2, 0] == 0 and not codes[2, 0].any()
    assert s[3, 2] == 2.0 ** -100 / 127 or s[3, 2] == torch.tensor(2.0 ** -100) / 127
    assert torch.all(codes[3, 2] == 127)
    for row, group in ((4, 0), (5, 2), (6, 3)):
        assert torch.isnan(s[row, group])
        others = [g for g in range(4) if g != group]
        assert torch.all(torch.isfinite(s[row, others]))
    assert torch.all(codes[7] == 127) and torch.all(torch.isfinite(s[7]))
    y = torch.zeros(8, 512, **BF16)
    hip.a8_dequant_rows(y, a, 0, 8)
    torch.cuda.synchronize()
    assert torch.all(torch.isnan(y[4, :128])) and torch.all(torch.isfinite(y[4, 128:]))


def _norm_tolerance(dim):
    """Relative error of a normed value: the sum of squares' roundings (4 a chunk of 8 in a
    thread's row of chunks, 6 and 16 joins; halved by the root), and 10 at the end."""
    return ((4 * ((dim + 8191) // 8192) + 24) / 2 + 10) * 2.0 ** -24


NORMS = [(1, 128), (3, 384), (1, 5120), (16, 5120), (9, 8192), (2, 8320), (5, 17408), (512, 640), (513, 640), (600, 4096),
         (520, 5120), (515, 12544)]


@pytest.mark.parametrize("rows,dim", NORMS)
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm(hip, rows, dim, residual):
    T = rows if rows < 5 else rows - 2
    h, w = _hidden(rows, dim, dim), 0.3 * _hidden(1, dim, 5)[0]
    r = _hidden(rows, dim, dim + 1) if residual else None
    a, q, scale = _buffers(hip, rows, dim)
    out = torch.full((rows, dim), 5.0, **BF16)
    before = h.clone()
    hip.rmsnorm_a8(a, h, w, T, 1e-6, residual=r, out=out)
    torch.cuda.synchronize()
    assert torch.equal(h, before)
    if residual:
        want = (h[:T].float() + r[:T].float()).to(torch.bfloat16)
        assert torch.equal(out[:T], want) and torch.all(out[T:] == 5.0)
    else:
        want = h[:T]
        assert torch.all(out == 5.0)
    v = want.double()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6) * (1 + w.double())
    _check(y, q, scale, T, _norm_tolerance(dim))


@pytest.mark.parametrize("rows,dim", [(1, 5120), (600, 4096), (3, 17408), (520, 12544)])
def test_rmsnorm_in_place(hip, rows, dim):
    """h_out over h, and over the residual: the same as apart."""
    h, r, w = _hidden(rows, dim, 1), _hidden(rows, dim, 2), _hidden(1, dim, 3)[0]
    a, q, scale = _buffers(hip, rows, dim)
    out = torch.zeros(rows, dim, **BF16)
    hip.rmsnorm_a8(a, h, w, rows, 1e-5, residual=r, out=out)
    for over in (0, 1):
        b, q2, scale2 = _buffers(hip, rows, dim)
        hh, rr = h.clone(), r.clone()
        hip.rmsnorm_a8(b, hh, w, rows, 1e-5, residual=rr, out=rr if over else hh)
        torch.cuda.synchronize()
        assert torch.equal(rr if over else hh, out)
        assert torch.equal(q, q2) and torch.equal(scale, scale2)


def test_rmsnorm_is_the_norm_and_the_codes(hip):
    """Within a rounding to bf16 of qw4_rmsnorm's rows brought to 8 bits."""
    T, dim = 20, 5120
    h, w = _hidden(T, dim, 1), 0.3 * _hidden(1, dim, 2)[0]
    a, q, scale = _buffers(hip, T, dim)
    hip.rmsnorm_a8(a, h, w, T, 1e-6)
    y = torch.zeros(T, dim, **BF16)
    hip.rmsnorm(y, h, w, T, dim, 1e-6)
    torch.cuda.synchronize()
    exact = y.double().view(T, -1, GROUP)
    codes = from_layout(q).double().view(T, -1, GROUP)
    s = scale.t().double()[:, :, None]
    assert torch.all((codes * s - exact).abs() <= 0.5001 * s + 2.0 ** -8 * exact.abs())


def test_rmsnorm_zero_and_nonfinite_rows(hip):
    h, w = _hidden(4, 1024, 1), _hidden(1, 1024, 2)[0]
    h[0] = 0
    h[1, 100] = float("nan")
    h[2, 100] = float("inf")
    a, q, scale = _buffers(hip, 4, 1024)
    hip.rmsnorm_a8(a, h, w, 4, 1e-6)
    torch.cuda.synchronize()
    s = scale.t()
    assert torch.all(s[0] == 0) and not q[0].any()
    assert torch.all(torch.isnan(s[1]))            # the row's mean is NaN
    assert torch.isnan(s[2, 0]) and torch.all(s[2, 1:] == 0)   # 1 / rms is 0, 0 Inf NaN
    assert torch.all(torch.isfinite(s[3]))


def test_no_rows(hip):
    a, q, scale = _buffers(hip, 2, 256)
    x = _hidden(2, 256, 1)
    hip.quantize_a8(a, x, 0)
    hip.rmsnorm_a8(a, x, x[0].contiguous(), 0, 1e-6)
    hip.a8_dequant_rows(x, a, 2, 0)
    torch.cuda.synchronize()
    assert torch.all(q == 77) and torch.all(scale == -3.0)


def test_allocated_rows(hip):
    """The library's own arrays, and offsets beyond 2^31 bytes of rows."""
    rows, dim = 170000, 17408   # 2.96e9 codes
    a = hip.a8_alloc(rows, dim)
    x = _hidden(64, dim, 4)
    big = torch.zeros(rows, dim, **BF16)
    big[-64:] = x
    hip.quantize_a8(a, big, rows)
    y = torch.zeros(64, dim, **BF16)
    hip.a8_dequant_rows(y, a, rows - 64, 64)
    b = hip.a8_alloc(64, dim)
    z = torch.zeros(64, dim, **BF16)
    hip.quantize_a8(b, x, 64)
    hip.a8_dequant_rows(z, b, 0, 64)
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    hip.a8_free(a)
    hip.a8_free(b)
    assert not a.q and not a.scale
