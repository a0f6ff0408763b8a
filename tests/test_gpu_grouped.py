"""qw4_gemm_grouped against the formula in 64 bits: experts with no, one and many rows,
row counts around the tile heights, gathered and in order, every activation, tokens
outside x, rows behind the last expert, offsets of no plan, a router's own plan; and a
whole layer of experts, eager and captured."""
import numpy as np
import pytest

from test_gpu_linear_epilogue import ACTS, activation, bf, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def i32(a):
    import torch

    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


# (experts, weight rows an expert, K, rows of each expert; those not listed have none)
CASES = {
    "one row": (1, 128, 128, [1]),
    "none and ones": (6, 256, 256, [0, 1, 0, 0, 1, 0]),
    "few": (8, 384, 640, [3, 0, 16, 1, 17, 2, 0, 15]),
    "many experts": (64, 128, 384, [i % 4 for i in range(64)]),
    "all experts": (1024, 128, 128, [(i * 7) % 3 for i in range(1024)]),
    "last of many": (700, 128, 256, [0] * 699 + [40]),
    "tiles": (5, 1152, 2176, [64, 65, 0, 129, 31]),
    "wide": (3, 2176, 1152, [33, 257, 100]),
    "ragged": (4, 640, 5120, [300, 1, 500, 0]),
    "long K": (3, 256, 8448, [5, 0, 40]),
    "long K, one row each": (4, 256, 17408, [1, 1, 0, 1]),
}


@pytest.mark.parametrize("case", CASES)
def test_grouped(hip, orc, case):
    import torch

    E, n, K, counts = CASES[case]
    g = torch.Generator().manual_seed(E + n + K)
    w, wq = make(hip, orc, E * n, K, E + K)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    R = int(offsets[-1])
    behind = 5
    x_rows = max(3, R // 2)
    tokens = torch.randint(0, x_rows, (R + behind,), generator=g).numpy()
    tokens[R:] = -1
    if R > 8:
        tokens[R // 2], tokens[R // 3] = -1, x_rows + 7   # no row of x: zeros
    ws = hip.gemm_workspace_alloc(256 << 20)
    do, dt = i32(offsets), i32(tokens)
    plan = hip.expert_plan_over(do, dt, dt)
    for act in ACTS:
        width = n // 2 if act == "swiglu" else n
        for gather in (False, True):
            xs = bf(torch.randn(x_rows if gather else R + behind, K, generator=g) * (8.0 / K ** 0.5))
            rows = xs
            if gather:
                t = torch.tensor(tokens[:R])
                live = (t >= 0) & (t < x_rows)
                rows = torch.where(live[:, None], xs[t.clamp(0, x_rows - 1)], torch.zeros(()).bfloat16())
            for bias in (None, bf(torch.randn(E * n, generator=g))):
                print(f"grouped {case}: {act} gather={gather} bias={bias is not None}", flush=True)
                y = torch.full((R + behind + 1, width), 7.0, dtype=torch.bfloat16, device="cuda")
                dx = xs.cuda()
                hip.gemm_grouped_w4a16(y[:R + behind], w, dx, plan, R + behind, gather,
                                       bias=bias.cuda() if bias is not None else None,
                                       act=getattr(hip, "ACT_" + act.upper()), ws=ws)
                again = torch.full_like(y, 7.0)
                hip.gemm_grouped_w4a16(again[:R + behind], w, dx, plan, R + behind, gather,
                                       bias=bias.cuda() if bias is not None else None,
                                       act=getattr(hip, "ACT_" + act.upper()), ws=None)
                torch.cuda.synchronize()
                assert (y[R:] == 7.0).all() and (again[R:] == 7.0).all()
                got, got2 = y.cpu(), again.cpu()
                seen = 0
                for e in range(E):
                    lo, hi = int(offsets[e]), int(offsets[e + 1])
                    if lo == hi or (seen > 40 and hi - lo < 3):
                        continue
                    seen += 1
                    pick = sorted({lo, hi - 1, (lo + hi) // 2, min(lo + 63, hi - 1), min(lo + 64, hi - 1)})
                    b = None if bias is None else bias[e * n:(e + 1) * n]
                    for out in (got, got2):
                        check(out, rows, wq[e * n:(e + 1) * n], b, act, None, pick, rounded=True)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


@pytest.mark.parametrize("form", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("case", CASES)
def test_grouped_forms(hip, orc, case, form):
    """Every kernel of the call (qw4_tune_grouped) on every case; the two that stream the
    weights use them exactly, and give the same bits."""
    import torch

    E, n, K, counts = CASES[case]
    exact = form == 1 and K <= 8192 or form == 2 and K <= 5120
    g = torch.Generator().manual_seed(E + n + K)
    w, wq = make(hip, orc, E * n, K, E + K)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    R = int(offsets[-1])
    tokens = torch.randint(0, R + 2, (R + 3,), generator=g).to(torch.int32)
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R + 3))
    do, dt = i32(offsets), tokens.cuda()
    plan = hip.expert_plan_over(do, dt, dt)
    bias = bf(torch.randn(E * n, generator=g))
    xs = bf(torch.randn(R + 3, K, generator=g) * (8.0 / K ** 0.5))
    dx, db = xs.cuda(), bias.cuda()
    try:
        for act in ("none", "swiglu", "gelu"):
            width = n // 2 if act == "swiglu" else n
            for gather in (False, True):
                rows = xs[tokens[:R].long()] if gather else xs
                outs = []
                for f in ((form, 3 - form) if exact and K <= 5120 else (form,)):
                    print(f"grouped form {f} {case}: {act} gather={gather}", flush=True)
                    y = torch.full((R + 4, width), 7.0, dtype=torch.bfloat16, device="cuda")
                    hip.tune_grouped(f)
                    hip.gemm_grouped_w4a16(y[:R + 3], w, dx, plan, R + 3, gather, bias=db,
                                           act=getattr(hip, "ACT_" + act.upper()), ws=ws)
                    torch.cuda.synchronize()
                    assert (y[R:] == 7.0).all()
                    outs.append(y.cpu())
                assert all(torch.equal(o, outs[0]) for o in outs)
                seen = 0
                for e in range(E):
                    lo, hi = int(offsets[e]), int(offsets[e + 1])
                    if lo == hi or (seen > 20 and hi - lo < 3):
                        continue
                    seen += 1
                    pick = sorted({lo, hi - 1, (lo + hi) // 2, min(lo + 63, hi - 1), min(lo + 64, hi - 1)})
                    check(outs[0], rows, wq[e * n:(e + 1) * n], bias[e * n:(e + 1) * n], act, None, pick,
                          rounded=not exact, bits=11 if act == "swiglu" and form > 2 else 8)
    finally:
        hip.tune_grouped(0)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


@pytest.mark.parametrize("form", [1, 2, 3, 4, 5])
def test_grouped_forms_bad_offsets(hip, orc, form):
    """As below, through every kernel."""
    import torch

    E, n, K, R = 4, 128, 256, 600
    w, _ = make(hip, orc, E * n, K, 5)
    x = bf(torch.randn(R, K)).cuda()
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R))
    tokens = i32(np.random.default_rng(1).integers(-(1 << 31), (1 << 31) - 1, R))
    try:
        hip.tune_grouped(form)
        for offsets in ([-5, 10, 3, 700, 1 << 30], [600, 500, 40, 30, 20], [0, 0, 0, 0, -1], [1 << 30] * 5,
                        [-(1 << 31), (1 << 31) - 1, 0, (1 << 31) - 1, 0]):
            plan = hip.expert_plan_over(i32(offsets), tokens, tokens)
            for act in (hip.ACT_NONE, hip.ACT_SWIGLU):
                for gather in (False, True):
                    print(f"form {form} bad offsets {offsets} {act} {gather}", flush=True)
                    y = torch.full((R + 2, n // 2 if act else n), 7.0, dtype=torch.bfloat16, device="cuda")
                    hip.gemm_grouped_w4a16(y[1:R + 1], w, x, plan, R, gather, act=act, ws=ws)
                    torch.cuda.synchronize()
                    assert (y[0] == 7.0).all() and (y[R + 1] == 7.0).all()
    finally:
        hip.tune_grouped(0)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


def test_grouped_bad_offsets(hip, orc):
    """Offsets that no plan has write no row outside y and read none outside x."""
    import torch

    E, n, K, R = 4, 128, 256, 50
    w, _ = make(hip, orc, E * n, K, 5)
    x = bf(torch.randn(R, K)).cuda()
    for offsets in ([-5, 10, 3, 70, 1 << 30], [60, 50, 40, 30, 20], [0, 0, 0, 0, -1], [1 << 30] * 5,
                    [-(1 << 31), (1 << 31) - 1, 0, (1 << 31) - 1, 0]):
        tokens = i32(np.random.default_rng(1).integers(-(1 << 31), (1 << 31) - 1, R))
        plan = hip.expert_plan_over(i32(offsets), tokens, tokens)
        for act in (hip.ACT_NONE, hip.ACT_SWIGLU):
            for gather in (False, True):
                print(f"bad offsets {offsets} {act} {gather}", flush=True)
                width = n // 2 if act else n
                y = torch.full((R + 2, width), 7.0, dtype=torch.bfloat16, device="cuda")
                hip.gemm_grouped_w4a16(y[1:R + 1], w, x, plan, R, gather, act=act)
                torch.cuda.synchronize()
                assert (y[0] == 7.0).all() and (y[R + 1] == 7.0).all()
    hip.awq_free(w)


@pytest.mark.parametrize("T,E,k,H,I", [(1, 16, 4, 512, 256), (7, 16, 4, 512, 256), (40, 8, 2, 640, 384),
                                       (333, 16, 4, 512, 256)])
def test_layer_of_experts(hip, orc, T, E, k, H, I):
    """Router, gate|up with swiglu, down, weighted sum with residual -- against 64 bits,
    and captured in a graph whose replays route new logits as the eager calls do."""
    import torch

    g = torch.Generator().manual_seed(T + H)
    wu, qu = make(hip, orc, E * 2 * I, H, 11)
    wd, qd = make(hip, orc, E * H, I, 12)
    x = bf(torch.randn(T, H, generator=g) * (4.0 / H ** 0.5))
    res = bf(torch.randn(T, H, generator=g))
    logits = [bf(torch.randn(T, E, generator=g)) for _ in range(3)]
    if T > 5:
        logits[1][T - 2:] = -float("inf")   # padding
    dx, dr, dl = x.cuda(), res.cuda(), logits[0].cuda()
    ids = torch.zeros(T * k, dtype=torch.int32, device="cuda")
    wt = torch.zeros(T * k, device="cuda")
    h = torch.zeros(T * k, I, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    plan = hip.expert_plan_alloc(E, T * k)
    ws = hip.gemm_workspace_alloc(256 << 20)

    def run():
        hip.route_experts(ids, wt, dl, T, E, k, True, plan)
        hip.gemm_grouped_w4a16(h, wu, dx, plan, T * k, True, act=hip.ACT_SWIGLU, ws=ws)
        hip.gemm_grouped_w4a16(y, wd, h, plan, T * k, False, ws=ws)
        hip.combine_experts(out, y, wt, T, k, H, plan, residual=dr)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for rep, lg in enumerate(logits + logits[:1]):
        dl.copy_(lg)
        out.zero_()
        run()
        torch.cuda.synchronize()
        eager = out.clone()
        hidden = h.clone()
        out.zero_()
        h.fill_(float("nan"))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), rep
        # the formula, each step from the step before it in 64 bits
        chosen, weight = ids.cpu().view(T, k).long(), wt.cpu().double().view(T, k)
        from gpu_util import download

        pos = torch.from_numpy(download(plan.pos, 4 * T * k).view(np.int32).copy()).view(T, k).long()
        for t in sorted({0, T - 1, T // 2}):
            ref, bound = res[t].double(), 0.0
            for j in range(k):
                e = int(chosen[t, j])
                if e < 0:
                    continue
                v = qu[e * 2 * I:(e + 1) * 2 * I] @ x[t].double()
                hid = activation(v[None], "swiglu")[0]
                got = hidden[pos[t, j]].cpu().double()
                # bf16 weights (6 sigma of K random terms) on both factors, then one rounding
                ev = 6 * 2.0 ** -8 * (qu[e * 2 * I:(e + 1) * 2 * I] ** 2 @ x[t].double() ** 2).sqrt() + 1e-6
                gt, up = v[:I], v[I:]
                eh = 1.13 * ev[:I] * (up.abs() + ev[I:]) + (gt * torch.sigmoid(gt)).abs() * ev[I:]
                assert ((got - hid).abs() <= eh + 2.0 ** -8 * (hid.abs() + eh)).all()
                down = qd[e * H:(e + 1) * H]
                row = down @ got
                ed = 6 * 2.0 ** -8 * (down ** 2 @ got ** 2).sqrt() + 2.0 ** -8 * row.abs() + 1e-6
                ref = ref + weight[t, j] * row
                bound = bound + weight[t, j] * ed
            err = (out[t].cpu().double() - ref).abs()
            assert (err <= bound + 2.0 ** -8 * (ref.abs() + bound) + 1e-6).all()
    del graph
    hip.expert_plan_free(plan)
    hip.gemm_workspace_free(ws)
    hip.awq_free(wu)
    hip.awq_free(wd)
