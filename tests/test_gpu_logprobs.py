"""Log probabilities, entropy and top alternatives of rows of logits (qw4_logprobs,
qw4_logprobs_f32) against the formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


def _run(hip, x, asked, k, ws_extra=0):
    """lp, entropy, ids, top of x [T][n] (any row stride), with guards behind each output."""
    T, n = x.shape
    cols = asked.shape[1]
    lp = torch.full((T + 1, cols), 55.0, device="cuda")
    entropy = torch.full((T + 1,), 55.0, device="cuda")
    ids = torch.full((T + 1, k), 55, dtype=torch.int32, device="cuda")
    top = torch.full((T + 1, k), 55.0, device="cuda")
    size = hip.logprobs_workspace(T, n, k)
    buf = torch.full((size + 64,), 7, dtype=torch.uint8, device="cuda")
    hip.logprobs(lp, x, asked, T, n, hip.GemmWorkspace(buf.data_ptr(), size), entropy=entropy, top_ids=ids,
                 top_logprobs=top, top_k=k)
    torch.cuda.synchronize()
    assert torch.all(buf[size:] == 7)
    for out in (lp, entropy, ids, top):
        assert torch.all(out[T:] == 55)
    return lp[:T].double(), entropy[:T].double(), ids[:T], top[:T].double()


def _exact(x, asked, k):
    """The formulas over finite logits and -Inf in 64 bits, on the CPU."""
    x = x.detach().cpu().double()
    T, n = x.shape
    m = x.amax(1, keepdim=True)
    some = m > -INF
    y = torch.where(some, x - m, -INF)
    e = torch.exp(y)
    best = torch.argsort(-x, dim=1, stable=True)[:, :k]
    s = e.sum(1, keepdim=True) - some.double()        # without the largest
    small = s < 1e-3
    if small.any():   # the others' own sum, where the difference would lose it
        order = torch.sort(e, dim=1).values
        s = torch.where(small, order[:, :-1].sum(1, keepdim=True) if n > 1 else torch.zeros_like(s), s)
    log = torch.log1p(s)
    base = m + log
    p = torch.where(some, e / (1 + s), 0.0)
    entropy = torch.where(p > 0, -p * torch.where(p > 0, y - log, 0.0), 0.0).sum(1)
    a = asked.cpu().long()
    inside = (a >= 0) & (a < n)
    picked = torch.gather(x, 1, a.clamp(0, n - 1))
    lp = torch.where(inside, torch.where(some, (picked - m) - log, -INF), 0.0)
    top = torch.gather(x, 1, best)
    ids = torch.where(top > -INF, best, -1).to(torch.int32)
    top = torch.where(some, (top - m) - log, -INF)
    if top.shape[1] < k:   # fewer logits than asked for
        more = k - top.shape[1]
        ids = torch.cat([ids, torch.full((T, more), -1, dtype=torch.int32)], 1)
        top = torch.cat([top, torch.full((T, more), -INF, dtype=torch.float64)], 1)
    second = torch.topk(x, 2, dim=1).values[:, 1:] if n > 1 else m
    gap = torch.where(second > -INF, m - second, 0.0)[:, 0]   # how far below the largest the sum's terms begin
    return [v.cuda() for v in (lp, entropy, ids, top, s[:, 0], gap)]


def _check(hip, x, asked, k):
    lp, entropy, ids, top = _run(hip, x, asked, k)
    wlp, went, wids, wtop, s, gap = _exact(x, asked, k)
    assert torch.equal(ids, wids)
    # s: a lane's sums (n / 256 of them at most, and the joins), exp (its argument's two
    # roundings, 2^-24 |d| each, |d| up to 20 beyond the gap where a term still counts, and
    # the instruction's 2^-22): relative; below fp32's range terms are zeros
    rel = (x.shape[1] / 256 + 80 + 2 * gap) * 2.0 ** -24
    log = torch.log1p(s)

    def near(got, want, tol):
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        fine = torch.isfinite(want)
        off = (got - want).abs()
        assert torch.all((off <= tol)[fine]), float((off - tol)[fine].max())

    near(lp, wlp, (rel * log)[:, None] + 2.0 ** -22 * wlp.abs() + 1e-36)
    near(top, wtop, (rel * log)[:, None] + 2.0 ** -22 * wtop.abs() + 1e-36)
    near(entropy, went, 4 * rel * went + 1e-34)


def _logits(T, n, seed, f32, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    x = sigma * torch.randn(T, n, generator=g)
    return x.cuda() if f32 else x.to(torch.bfloat16).cuda()


def _asked(T, n, count, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, n, (T, count), generator=g).to(torch.int32).cuda()


SIZES = [(1, 1), (2, 2), (3, 7), (1, 8), (4, 9), (2, 63), (3, 64), (1, 65), (5, 511), (2, 512), (1, 513), (3, 2047),
         (2, 2048), (1, 4099), (7, 8191), (2, 32003), (513, 777), (600, 2051), (40, 20000), (1, 248320), (9, 248320),
         (100, 50001)]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,n", SIZES)
def test_sizes(hip, T, n, f32):
    k = min(20, max(1, n // 2))
    _check(hip, _logits(T, n, n, f32), _asked(T, n, 1 + n % 3, T), k)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("k", [0, 1, 2, 13, 31, 32])
@pytest.mark.parametrize("T,n", [(1, 20000), (3, 40), (520, 600)])
def test_alternatives(hip, T, n, k, f32):
    _check(hip, _logits(T, n, 3, f32), _asked(T, n, 70 if T == 1 else 2, 4), k)


@pytest.mark.parametrize("f32", [False, True])
def test_more_alternatives_than_logits(hip, f32):
    _check(hip, _logits(4, 5, 3, f32), _asked(4, 5, 1, 4), 32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("first,beside", [(0, 1), (1, 0), (3, 2), (5, 64), (7, 1)])
def test_columns_of_a_buffer(hip, first, beside, f32):
    """Rows that begin and end anywhere; what lies beside them would be the largest."""
    T, n = 11, 1537
    x = _logits(T, first + n + beside, 3, f32)
    x[:, :first] = 1000.0
    x[:, first + n:] = NAN
    _check(hip, x[:, first:first + n], _asked(T, n, 2, 4), 8)


@pytest.mark.parametrize("f32", [False, True])
def test_ties_take_the_lowest_index(hip, f32):
    for T, n, levels in ((2, 5000, 1), (3, 4097, 3), (1, 100000, 2), (515, 700, 4)):
        g = torch.Generator().manual_seed(n)
        x = torch.randint(0, levels, (T, n), generator=g).float().cuda()
        _check(hip, x if f32 else x.to(torch.bfloat16), _asked(T, n, 1, 1), 32)
    zeros = torch.zeros(2, 3000)
    zeros[0, ::2] = -0.0
    zeros[1, 1::2] = -0.0
    _check(hip, zeros.cuda() if f32 else zeros.to(torch.bfloat16).cuda(), _asked(2, 3000, 1, 1), 10)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rising", [False, True])
def test_sorted_rows(hip, rising, f32):
    for T, n in ((1, 70000), (2, 9000), (512, 1200)):
        x = torch.sort(_logits(T, n, 3, True), dim=1, descending=not rising).values
        _check(hip, x if f32 else x.to(torch.bfloat16), _asked(T, n, 1, 1), 20)


@pytest.mark.parametrize("f32", [False, True])
def test_likely_tokens(hip, f32):
    """One token nearly certain: log probability and entropy keep their precision."""
    x = _logits(12, 32000, 3, f32, 1.0)
    for t in range(12):
        x[t, 100 * t + 7] = 10.0 + 3 * t
    asked = torch.stack([torch.arange(12) * 100 + 7, torch.arange(12)], 1).to(torch.int32).cuda()
    _check(hip, x, asked, 5)


@pytest.mark.parametrize("f32", [False, True])
def test_large_and_shifted_logits(hip, f32):
    x = _logits(6, 3000, 3, f32)
    x[1] += 300
    x[2] -= 300
    x[3] *= 1000
    x[4] = x[4] * 1e30
    x[5] = x[5] * 1e-30
    _check(hip, x, _asked(6, 3000, 3, 1), 20)


@pytest.mark.parametrize("f32", [False, True])
def test_masked_tokens(hip, f32):
    """-Inf: some, all but one, all; the type's lowest value is a value."""
    n = 5000
    x = _logits(7, n, 3, f32)
    g = torch.Generator().manual_seed(1)
    x[0, torch.rand(n, generator=g).cuda() < 0.99] = -INF
    keep = x[1, 4321].clone()
    x[1] = -INF
    x[1, 4321] = keep
    x[2] = -INF
    x[3, :4990] = -INF
    x[4, 10:] = -INF
    lowest = torch.finfo(x.dtype).min
    x[5] = lowest
    x[6, 1:] = lowest
    asked = torch.tensor([[0, 4321, 4999, -1, n, -100]] * 7, dtype=torch.int32).cuda()
    _check(hip, x, asked, 20)
    lp, entropy, ids, top = _run(hip, x, asked, 20)
    assert torch.all(lp[:, 3:] == 0)
    assert entropy[2] == 0 and torch.all(ids[2] == -1) and torch.all(top[2] == -INF) and torch.all(lp[2, :3] == -INF)
    assert entropy[1] == 0 and lp[1, 1] == 0 and lp[1, 0] == -INF
    assert abs(float(entropy[5]) - math.log(n)) < 1e-5


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("n", [700, 60000])
def test_nan_and_inf(hip, n, f32):
    """Their rows' numbers are NaN, the others' and the order of the rest are not."""
    x = _logits(8, n, 3, f32)
    clean = _run(hip, x, _asked(8, n, 2, 1), 6)
    bad = x.clone()
    bad[1, n // 3] = NAN
    bad[2, 0] = INF
    bad[3, n - 1] = NAN
    bad[4, :] = NAN
    bad[5, 5] = INF
    bad[5, n - 5] = INF
    bad[6, :] = -INF
    bad[6, 100] = NAN
    lp, entropy, ids, top = _run(hip, bad, _asked(8, n, 2, 1), 6)
    for t in (1, 2, 3, 4, 5, 6):
        assert torch.isnan(entropy[t]) and torch.all(torch.isnan(lp[t])) and torch.all(torch.isnan(top[t]))
    for t in (0, 7):
        for got, want in zip((lp, entropy, ids, top), clean):
            assert torch.equal(got[t], want[t])
    seen = torch.where(torch.isnan(bad), -INF, bad.double()).cpu()
    best = torch.argsort(-seen, dim=1, stable=True)[:, :6]
    want = torch.where(torch.gather(seen, 1, best) > -INF, best, -1).to(torch.int32).cuda()
    assert torch.equal(ids, want)


def test_what_is_not_asked_for(hip):
    x = _logits(3, 1000, 3, True)
    asked = _asked(3, 1000, 2, 1)
    lp, entropy, ids, top = _run(hip, x, asked, 4)
    one = torch.zeros(3, 2, device="cuda")
    hip.logprobs(one, x, asked, 3, 1000)
    two = torch.zeros(3, device="cuda")
    hip.logprobs(None, x, None, 3, 1000, entropy=two)
    i, v = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(3, 4, device="cuda")
    hip.logprobs(None, x, None, 3, 1000, top_ids=i, top_logprobs=v, top_k=4)
    hip.logprobs(None, x, None, 0, 1000)
    hip.logprobs(None, x, None, 3, 1000)
    torch.cuda.synchronize()
    rel = 2.0 ** -18   # with and without the list a block's new largest is met in another order
    assert torch.all((one.double() - lp).abs() <= rel * lp.abs())
    assert torch.all((two.double() - entropy).abs() <= rel * entropy)
    assert torch.equal(i, ids) and torch.equal(v.double(), top)


def test_offsets_beyond_32_bits(hip):
    """Rows that lie beyond 2^31 elements and 2^32 bytes."""
    T, n = 9000, 248320
    x = torch.zeros(T, n, dtype=torch.bfloat16, device="cuda")   # 4.47 GB, 2.23e9 logits
    tail = _logits(16, n, 3, False)
    x[-16:] = tail
    asked = _asked(T, n, 1, 1)
    lp, entropy, ids, top = _run(hip, x, asked, 3)
    wlp, went, wids, wtop = _run(hip, tail.contiguous().repeat(40, 1), asked[-16:].repeat(40, 1), 3)   # whole rows too
    assert torch.equal(ids[-16:], wids[:16]) and torch.equal(top[-16:], wtop[:16])
    assert torch.equal(lp[-16:], wlp[:16]) and torch.equal(entropy[-16:], went[:16])
    assert torch.all(ids[:-16] == torch.arange(3, dtype=torch.int32, device="cuda"))
    assert torch.all((entropy[:-16] - math.log(n)).abs() < 1e-4)
