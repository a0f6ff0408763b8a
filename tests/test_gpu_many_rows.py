"""Rows past what one launch takes (its grid has fewer than 2^32 threads): rmsnorm of 2^24
rows, as the heads of a long prompt are, argmax of 2^26 short rows."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    yield w4a16_hip
    torch.cuda.empty_cache()


def test_rmsnorm_many(hip):
    """Each row as a call of 600 rows computes it."""
    import torch

    rows, dim = (1 << 24) + 700, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.empty(dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    out = torch.full((rows + 1, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    print(f"rmsnorm {rows}x{dim}", flush=True)
    hip.rmsnorm(out, x, w, rows, dim, 1e-6)
    some = torch.empty(600, dim, dtype=torch.bfloat16, device="cuda")
    for first in (0, (1 << 23) - 300, rows // 2, (1 << 24) - 300, rows - 600):
        hip.rmsnorm(some, x[first:first + 600], w, 600, dim, 1e-6)
        torch.cuda.synchronize()
        assert torch.equal(out[first:first + 600], some), first
    assert (out[rows] == 7.0).all()


def test_argmax_many(hip):
    import torch

    rows, n = (1 << 26) + 9, 8
    r = torch.arange(rows, device="cuda")
    want = (r ^ (r >> 5)) % n
    x = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    x[r, want] = 1.0
    out = torch.full((rows + 1,), -7, dtype=torch.int32, device="cuda")
    print(f"argmax_rows {rows}x{n}", flush=True)
    hip.argmax_rows(out, x, rows, n)
    torch.cuda.synchronize()
    assert torch.equal(out[:rows].long(), want) and int(out[rows]) == -7
