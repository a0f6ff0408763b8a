"""Scales in products of 8-bit rows: all their bits count, and what Inf does."""
import pytest
import torch

from a8_util import product, random_rows, random_weights, sum_tolerance, to_layout

pytestmark = pytest.mark.gpu
GROUP = 128
# row counts of every kernel: few rows in one to four blocks, tiles of every height
ROWS = [1, 3, 7, 16, 17, 32, 33, 48, 50, 64, 77, 100, 128, 150, 200, 300, 700]


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


@pytest.fixture(scope="module")
def ws(hip):
    w = hip.gemm_workspace_alloc(256 << 20)
    yield w
    hip.gemm_workspace_free(w)


def _one_group(T, k, seed):
    """Rows whose codes are zeros outside one group, scales whose last bits are ones."""
    q, _ = random_rows(T, k, seed)
    g = torch.Generator().manual_seed(seed + 1)
    at = torch.randint(0, k // GROUP, (T,), generator=g).cuda()
    q = q.view(T, -1, GROUP)
    q = torch.where(torch.arange(k // GROUP, device="cuda")[None, :, None] == at[:, None, None], q, torch.zeros_like(q))
    bits = torch.randint(0, 1 << 21, (k // GROUP, T), generator=g, dtype=torch.int32)
    exponent = torch.randint(127 - 60, 127 + 60, (k // GROUP, T), generator=g, dtype=torch.int32)
    scale = ((exponent << 23) | (bits << 2) | 3).view(torch.float32).cuda()
    return q.view(T, k), scale


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("n,k", [(192, 128), (320, 640), (64, 5120), (64, 11008)])
@pytest.mark.parametrize("T", ROWS)
def test_a_groups_product_is_rounded_once(hip, ws, T, n, k, space):
    """Weight scales of 1 and one group that is not zeros: every value is its integer times the
    row's scale, to the nearest fp32."""
    w, less, s = random_weights(hip, n, k, n + T, scale=1.0)
    q, scale = _one_group(T, k, T + k)
    codes = to_layout(q)
    y = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws if space else None)
    torch.cuda.synchronize()
    v, _ = product(q, scale, less, s)   # one product of 18 and 24 bits: exact
    assert torch.equal(y, v.float())
    hip.awq_free(w)


@pytest.mark.parametrize("T", ROWS)
def test_a_groups_product_is_rounded_twice(hip, ws, T):
    """Weight scales of 8 bits: by the weight's scale, then by the row's."""
    n, k = 128, 1280
    w, less, s = random_weights(hip, n, k, T)
    q, scale = _one_group(T, k, T + 5)
    codes = to_layout(q)
    y = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws)
    torch.cuda.synchronize()
    v, _ = product(q, scale, less, s)
    assert torch.all((y.double() - v).abs() <= (2.0 ** -23 + 2.0 ** -47) * v.abs())
    hip.awq_free(w)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T", [1, 6, 16, 30, 40, 60, 100, 300])
def test_a_nonfinite_scale_of_a_row(hip, ws, T, value):
    """Inf times a sum is Inf of its sign, or NaN where the sum is 0; other rows stay."""
    n, k = 192, 1024
    w, less, s = random_weights(hip, n, k, 3)
    q, scale = random_rows(T, k, 4)
    codes = to_layout(q)
    clean = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(clean, w, hip.a8_over(codes, scale), T, ws)
    bad, rows = scale.clone(), sorted({0, T // 2, T - 1})
    for i, row in enumerate(rows):
        bad[(3 * i) % 8, row] = value
    y = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, bad), T, ws)
    torch.cuda.synchronize()
    for i, row in enumerate(rows):
        at = slice((3 * i) % 8 * GROUP, ((3 * i) % 8 + 1) * GROUP)
        want = (less[:, at] * q[row, at].double()).sum(1) * value
        assert torch.equal(y[row].double().nan_to_num(7.0), want.nan_to_num(7.0))
    others = [t for t in range(T) if t not in rows]
    assert torch.equal(y[others], clean[others])
    hip.awq_free(w)


@pytest.mark.parametrize("T", [2, 20, 40, 130])
def test_the_largest_and_smallest_rows(hip, ws, T):
    """Scales up to fp32's largest over 15 128 127, and down to 2^-100 / 127."""
    n, k = 128, 256
    w, less, s = random_weights(hip, n, k, 6)
    q, scale = random_rows(T, k, 7)
    scale[0] = 1.0e33
    scale[:, T // 2] = 2.0 ** -100 / 127
    codes = to_layout(q)
    y = torch.zeros(T, n, device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws)
    torch.cuda.synchronize()
    v, size = product(q, scale, less, s)
    assert torch.isfinite(y).all()
    assert torch.all((y.double() - v).abs() <= sum_tolerance(size, 2))
    hip.awq_free(w)
