"""Products of 8-bit rows whose weights, codes or outputs lie past 32-bit offsets."""
import pytest
import torch

from a8_util import GROUP, product, random_rows, random_weights, sum_tolerance, to_layout

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


@pytest.fixture(scope="module")
def wide(hip):
    """Weights of 2^21 + 128 rows of 4224 inputs: 4.4 GB of words. Their first, some middle and
    last rows in 64 bits."""
    n, k = (1 << 21) + 128, 4224
    g = torch.Generator("cuda").manual_seed(5)
    words = lambda *s: torch.randint(-(1 << 31), (1 << 31) - 1, s, generator=g, dtype=torch.int32, device="cuda")  # noqa: E731
    packed, zeros = words(n, k // 8), words(n // 8, k // GROUP)
    scales = (0.001 + 0.01 * torch.rand(n, k // GROUP, generator=g, device="cuda")).to(torch.bfloat16)
    w = hip.awq_repack(packed, scales, zeros, n, k)
    torch.cuda.synchronize()
    at = torch.cat([torch.arange(64), torch.arange(n // 2 + 64 - 32, n // 2 + 64 + 32), torch.arange(n - 128, n)]).cuda()
    shifts = 4 * torch.arange(8, device="cuda")
    q = ((packed[at].long()[:, :, None] >> shifts) & 15).view(len(at), -1, GROUP)
    z = (zeros[at // 8].long() >> (4 * (at % 8))[:, None]) & 15
    less = (q - z[:, :, None]).double().view(len(at), k)
    ws = scales[at].double()
    del packed, zeros, scales
    yield n, k, w, at, less, ws
    hip.awq_free(w)


@pytest.mark.parametrize("T", [1, 9, 20, 40, 300])
def test_weights_past_4_gib(hip, wide, T):
    n, k, w, at, less, ws = wide
    q, scale = random_rows(T, k, T)
    codes = to_layout(q)
    a = hip.a8_over(codes, scale)
    y = torch.zeros(T, n, device="cuda")
    space = hip.gemm_workspace_alloc(128 << 20)
    hip.linear_w4a8_f32(y, w, a, T, space)
    v, size = product(q, scale, less, ws)
    assert ((y[:, at].double() - v).abs() <= sum_tolerance(size, k // GROUP)).all()
    hip.gemm_workspace_free(space)


T, K, SOME = 270000, 17408, 500   # 4.7 GB of codes: 540 times the same rows


def parts(y):
    """The first rows, some past 4 GiB and the last."""
    return y[:SOME], y[T // SOME // 2 * SOME:][:SOME], y[T - SOME:]


def test_quantized_codes_past_4_gib(hip):
    x = torch.randn(SOME, K, device="cuda").bfloat16()
    a, one = hip.a8_alloc(T, K), hip.a8_alloc(SOME, K)
    hip.quantize_a8(one, x, SOME)
    hip.quantize_a8(a, x.repeat(T // SOME, 1), T)
    want, got = (torch.empty(SOME, K, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    hip.a8_dequant_rows(want, one, 0, SOME)
    for first in (0, T // SOME // 2 * SOME, T - SOME):
        hip.a8_dequant_rows(got, a, first, SOME)
        assert torch.equal(got, want)
    hip.a8_free(a)
    hip.a8_free(one)


@pytest.mark.parametrize("space", [False, True])
def test_codes_past_4_gib(hip, space):
    n = 128
    w, less, ws = random_weights(hip, n, K, 3)
    q, scale = random_rows(SOME, K, 4)
    codes, scales = to_layout(q).repeat(T // SOME, 1), scale.repeat(1, T // SOME)
    a = hip.a8_over(codes, scales)
    y = torch.zeros(T, n, device="cuda")
    room = hip.gemm_workspace_alloc(128 << 20) if space else None
    hip.linear_w4a8_f32(y, w, a, T, room)
    v, size = product(q, scale, less, ws)
    for rows in parts(y):
        assert ((rows.double() - v).abs() <= sum_tolerance(size, K // GROUP)).all()
    if space:
        hip.gemm_workspace_free(room)
    hip.awq_free(w)
