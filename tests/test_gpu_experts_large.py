"""Rows and columns past 2^31 elements and 2^32 bytes: each call's last rows, which a
32-bit offset would misplace, against the formula in 64 bits."""
import pytest

from test_gpu_linear_epilogue import bf, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    yield w4a16_hip
    torch.cuda.empty_cache()


class Rows:
    """Rows of a device tensor, copied when indexed by a list."""

    def __init__(self, t):
        self.t = t

    def __getitem__(self, rows):
        import torch

        return torch.stack([self.t[r] for r in rows]).cpu()


@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_epilogue_large_y(hip, orc, act):
    """T x width of 2^31 elements and more; bias, residual in y."""
    import torch

    N, K = (65536, 128) if act == "none" else (65536, 256)
    width = N // 2 if act == "swiglu" else N
    T = (1 << 31) // width + 300
    w, wq = make(hip, orc, N, K, 51)
    g = torch.Generator().manual_seed(5)
    x = bf(torch.randn(T, K, generator=g) * (8.0 / K ** 0.5)).cuda()
    bias = bf(torch.randn(N, generator=g))
    y = torch.zeros(T, width, dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, T // 2, T - 301, T - 300, T - 299, T - 33, T - 1]
    res = bf(torch.randn(len(rows), width, generator=g))
    full = {r: res[i] for i, r in enumerate(rows)}
    for r, v in full.items():
        y[r] = v.cuda()
    ws = hip.gemm_workspace_alloc((256 << 20) + hip.epilogue_workspace(w, T))
    print(f"large y {act} T={T}", flush=True)
    hip.linear_epilogue_w4a16(y, w, x, T, None, ws, bias=bias.cuda(), act=getattr(hip, "ACT_" + act.upper()), residual=y)
    torch.cuda.synchronize()

    class Res:
        def __getitem__(self, rs):
            return torch.stack([full[r] for r in rs])

    check(Rows(y), Rows(x), wq, bias, act, Res(), rows, rounded=True, bits=11 if act == "swiglu" else 8)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


@pytest.mark.parametrize("act,E", [("none", 3), ("swiglu", 3), ("none", 1024)])
def test_grouped_large(hip, orc, act, E):
    """x in the plan's order of more than 4 GiB, then y of more."""
    import torch

    for n, K in ((128, 2048), (4096, 128)) if E == 3 else ((64, 256), (128, 128)):
        R = (1 << 31) // max(n // (2 if act == "swiglu" else 1), K) + 1000
        w, wq = make(hip, orc, E * n, K, 52)
        g = torch.Generator(device="cuda").manual_seed(6)
        x = torch.empty(R, K, dtype=torch.bfloat16, device="cuda").normal_(0, 8.0 / K ** 0.5, generator=g)
        width = n // 2 if act == "swiglu" else n
        y = torch.full((R + 1, width), 7.0, dtype=torch.bfloat16, device="cuda")
        cut = torch.linspace(0, R, E + 1).round().to(torch.int64)
        cut[-1] = R
        offsets = cut.to(torch.int32).cuda()
        tokens = torch.zeros(R, dtype=torch.int32, device="cuda")
        plan = hip.expert_plan_over(offsets, tokens, tokens)
        ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R))
        for space in (None, ws) if act == "swiglu" else (None,):
            print(f"grouped large {act} E={E} {n}x{K} R={R} ws={space is not None}", flush=True)
            y.fill_(7.0)
            hip.gemm_grouped_w4a16(y[:R], w, x, plan, R, False, act=getattr(hip, "ACT_" + act.upper()), ws=space)
            torch.cuda.synchronize()
            assert (y[R] == 7.0).all()
            for e in sorted({0, E // 2, E - 1}):
                lo, hi = int(cut[e]), int(cut[e + 1])
                check(Rows(y), Rows(x), wq[e * n:(e + 1) * n], None, act, None, [lo, (lo + hi) // 2, hi - 1],
                      rounded=True, bits=8 if space is None else 11)
        hip.gemm_workspace_free(ws)
        hip.awq_free(w)
        del x, y


def test_combine_large(hip):
    import torch

    T, k, dim = (1 << 31) // (2 * 4096) + 500, 2, 4096
    y = torch.zeros(T * k, dim, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    y[-1000:].normal_(generator=g)
    y[:1000].normal_(generator=g)
    pos = torch.arange(T * k - 1, -1, -1, dtype=torch.int32, device="cuda")
    wt = torch.rand(T * k, device="cuda", generator=g)
    offsets = torch.zeros(9, dtype=torch.int32, device="cuda")
    plan = hip.expert_plan_over(offsets, pos, pos)
    out = torch.full((T + 1, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    print(f"combine large T={T}", flush=True)
    hip.combine_experts(out, y, wt, T, k, dim, plan)
    torch.cuda.synchronize()
    assert (out[T] == 7.0).all()
    for t in (0, 3, 499, T // 2, T - 500, T - 1):
        terms = torch.stack([wt[t * k + j].double() * y[int(pos[t * k + j])].double() for j in range(k)])
        ref, sums = terms.sum(0), (k + 1) * 2.0 ** -24 * terms.abs().sum(0)
        assert ((out[t].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + sums) + sums).all()


def test_route_large(hip):
    """Ids and weights past 2^24 tokens' worth of logits, the plan of 2^25 pairs."""
    import torch

    T, E, k = (1 << 24) + 5, 128, 2   # logits of 4 GiB
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    t = torch.arange(T, device="cuda")
    logits[t, (t * 7) % E] = 2.0
    logits[t, (t * 7 + 5) % E] = 1.0
    ids = torch.empty(T * k, dtype=torch.int32, device="cuda")
    wt = torch.empty(T * k, device="cuda")
    plan_t = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T * k, T * k)]
    plan = hip.expert_plan_over(*plan_t)
    print(f"route large T={T}", flush=True)
    hip.route_experts(ids, wt, logits, T, E, k, True, plan)
    torch.cuda.synchronize()
    want = torch.stack([(t * 7) % E, (t * 7 + 5) % E], 1).to(torch.int32).view(-1)
    assert torch.equal(ids, want)
    counts = torch.bincount(want.long(), minlength=E)
    assert torch.equal(plan_t[0][1:].long(), counts.cumsum(0)) and int(plan_t[0][0]) == 0
    order = torch.sort(want.long(), stable=True).indices
    assert torch.equal(plan_t[1].long(), order // k)
    assert torch.equal(plan_t[2][order].long(), torch.arange(T * k, device="cuda"))
    e = float(torch.tensor(-1.0).double().exp())
    assert (wt.view(T, k).double() - torch.tensor([1 / (1 + e), e / (1 + e)], device="cuda").double()).abs().max() < 64 * 2.0 ** -24
