"""A row's product in 8 bits does not depend on the rows beside it, nor on its place."""
import pytest
import torch

from a8_util import random_rows, random_weights, to_layout

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


def _products(hip, w, q, scale, n, ws=None):
    T = q.shape[0]
    codes, scale = to_layout(q), scale.contiguous()
    y = torch.full((T, n), float("nan"), device="cuda")
    hip.linear_w4a8_f32(y, w, hip.a8_over(codes, scale), T, ws)
    torch.cuda.synchronize()
    return y


@pytest.mark.parametrize("n,k,most", [(320, 128, 48), (320, 5120, 48), (64, 4992, 48), (17408, 640, 48),
                                      (192, 17408, 16), (192, 10240, 32)])
def test_a_larger_call_repeats_a_smaller_ones_rows(hip, n, k, most):
    """The kernel for few rows sums a row's groups in one order whatever the number of rows: up
    to 48, or to 16 and 32 of more inputs, every call's rows are the largest call's, bit for bit."""
    w, _, _ = random_weights(hip, n, k, 3)
    q, scale = random_rows(most, k, 4)
    full = _products(hip, w, q, scale, n)
    assert torch.isfinite(full).all()
    low = 17 if (k, most) == (10240, 32) else 1   # up to 16 rows of 10240 inputs: in 16 waves
    for T in range(low, most):
        assert torch.equal(_products(hip, w, q[:T], scale[:, :T], n), full[:T]), T
    hip.awq_free(w)


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("n,k", [(320, 1280), (128, 5120)])
@pytest.mark.parametrize("T", [2, 9, 17, 40, 64, 65, 100, 200, 300, 700])
def test_rows_in_another_order(hip, T, n, k, space):
    """Rows in another order give results in that order; rows beside one that are replaced, by
    NaN too, do not change it."""
    w, _, _ = random_weights(hip, n, k, 5)
    q, scale = random_rows(T, k, 6)
    ws = hip.gemm_workspace_alloc(256 << 20) if space else None
    y = _products(hip, w, q, scale, n, ws)
    assert torch.isfinite(y).all()
    order = torch.randperm(T, generator=torch.Generator().manual_seed(T)).cuda()
    assert torch.equal(_products(hip, w, q[order], scale[:, order], n, ws), y[order])
    other, others = random_rows(T, k, 7)
    others[0] = float("nan")
    for row in sorted({0, T // 3, T - 1}):
        p, s = other.clone(), others.clone()
        p[row], s[:, row] = q[row], scale[:, row]
        z = _products(hip, w, p, s, n, ws)
        assert torch.equal(z[row], y[row])
        assert torch.isnan(z).sum() == (T - 1) * n
    if space:
        hip.gemm_workspace_free(ws)
    hip.awq_free(w)
