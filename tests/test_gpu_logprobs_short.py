"""Log probabilities of rows that hold no whole 16 bytes between their boundaries, or few, with
alternatives: what lies before and behind them counts for nothing."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


@pytest.mark.parametrize("beside", [float("inf"), float("nan"), 3.0e38, -3.0e38])
@pytest.mark.parametrize("f32", [False, True])
def test_short_rows(hip, f32, beside):
    """Rows of 1 to 24 logits at every place of 16 bytes, each in a buffer of `beside`, the last
    one's last logit at the buffer's end."""
    dtype, per, T = (torch.float32, 4, 3) if f32 else (torch.bfloat16, 8, 3)
    g = torch.Generator().manual_seed(11)
    for n in range(1, 25):
        for first in range(per):
            x = (2.5 * torch.randn(T, n, generator=g)).to(dtype)
            ld = -(-(first + n) // per) * per + per
            buffer = torch.full(((T - 1) * ld + first + n,), beside, dtype=dtype, device="cuda")
            view = buffer.as_strided((T, n), (ld, 1), first)
            view.copy_(x)
            k = min(5, n + 1)
            lp, e = torch.zeros(T, n, device="cuda"), torch.zeros(T, device="cuda")
            ids, top = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(T, k, device="cuda")
            asked = torch.arange(n, dtype=torch.int32, device="cuda").repeat(T, 1)
            hip.logprobs(lp, view, asked, T, n, entropy=e, top_ids=ids, top_logprobs=top, top_k=k)
            torch.cuda.synchronize()
            want = torch.log_softmax(x.double(), 1)
            # x - m, less the log: half a step of up to 20 each; the log's own few steps of at most log 24
            tol = 2.0 ** -24 * (2 * 20 + 64)
            assert ((lp.cpu().double() - want).abs() <= tol).all(), (n, first)
            assert ((e.cpu().double() + (want.exp() * want).sum(1)).abs() <= 64 * 2.0 ** -24 * (1 + math.log(24))).all()
            best = torch.argsort(-x.double(), dim=1, stable=True)[:, :k]
            value = torch.gather(want, 1, best)
            if k > n:
                best = torch.cat([best, torch.full((T, 1), -1)], 1)
                value = torch.cat([value, torch.full((T, 1), -math.inf, dtype=torch.float64)], 1)
            assert torch.equal(ids.cpu().long(), best), (n, first)
            off = (top.cpu().double() - value).abs()
            assert ((off <= tol) | ((top.cpu() == -math.inf) & (value == -math.inf))).all(), (n, first)
