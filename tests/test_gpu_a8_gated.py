"""Gated products of 17 to 32 8-bit rows around the numbers of inputs where one kernel takes over
from another, against the formula in 64 bits."""
import pytest
import torch

from a8_util import product, random_rows, random_weights, sum_tolerance, to_layout

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


@pytest.mark.parametrize("space", [False, True])
@pytest.mark.parametrize("k", [5120, 5248, 6016, 8064, 8192, 8320, 10240, 10368])
@pytest.mark.parametrize("n", [256, 1408])
@pytest.mark.parametrize("T", [17, 24, 32, 33])
def test_gated(hip, T, n, k, space):
    w, less, s = random_weights(hip, n, k, T)
    q, scale = random_rows(T + 1, k, n)
    up, ws = n // 2, hip.gemm_workspace_alloc(256 << 20) if space else None
    y = torch.full((T + 1, up), 9.0, dtype=torch.bfloat16, device="cuda")
    codes = to_layout(q)
    hip.linear_w4a8(y, w, hip.a8_over(codes, scale), T, ws, act=hip.ACT_SWIGLU)
    torch.cuda.synchronize()
    v, size = product(q[:T], scale[:, :T], less, s)
    tol = sum_tolerance(size, k // 128)
    gate, u, f = v[:, :up], v[:, up:], v[:, :up] * torch.sigmoid(v[:, :up])
    # silu's slope is below 1.1; exp's argument |gate| 2^-24, its and the quotient's steps 20
    off = 1.1 * tol[:, :up] * (u.abs() + tol[:, up:]) + f.abs() * tol[:, up:] + (gate.abs() + 20) * 2.0 ** -23 * (f * u).abs()
    assert torch.all((y[:T].double() - f * u).abs() <= off + (2.0 ** -8 + 2.0 ** -23) * (f * u).abs() + 2.0 ** -8 * off)
    assert torch.all(y[T:] == 9.0)
    if space:
        hip.gemm_workspace_free(ws)
    hip.awq_free(w)
