"""Rows of x with Inf or NaN: no output of theirs is finite, and every other row is what
it is without them, bit for bit -- through the fp16 operands of a gated product, and
through every kernel of the products grouped by expert."""
import pytest
import torch

from test_gpu_linear_epilogue import bf, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def poisoned(x, rows):
    bad = x.clone()
    for i, r in enumerate(rows):
        bad[r, (7 * i + 3) % x.shape[1]] = (float("inf"), float("nan"), -float("inf"))[i % 3]
    return bad


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("T", [130, 259, 1000])
def test_dense(hip, orc, T, act):
    N, K = 640, 1024
    w, _ = make(hip, orc, N, K, T)
    ws = hip.gemm_workspace_alloc(256 << 20)
    x = bf(torch.randn(T, K, generator=torch.Generator().manual_seed(T)) * (8.0 / K ** 0.5))
    rows = [0, 7, 60, 61, T - 2, T - 1]
    out = {}
    for space in (None, ws):
        for name, xi in (("clean", x), ("bad", poisoned(x, rows))):
            print(f"nonfinite T={T} {act} {name} ws={space is not None}", flush=True)
            y = torch.empty(T, N // 2 if act == "swiglu" else N, dtype=torch.bfloat16, device="cuda")
            hip.linear_epilogue_w4a16(y, w, xi.cuda(), T, None, space, act=getattr(hip, "ACT_" + act.upper()))
            torch.cuda.synchronize()
            out[name] = y.cpu()
        other = torch.ones(T, dtype=torch.bool)
        other[rows] = False
        assert not torch.isfinite(out["bad"][rows]).any()
        assert torch.isfinite(out["clean"]).all() and torch.equal(out["bad"][other], out["clean"][other])
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


@pytest.mark.parametrize("form", [0, 1, 2, 3, 4, 5])
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_grouped(hip, orc, act, form):
    E, n, K = 4, 256, 640
    counts = [70, 0, 5, 300]
    R = sum(counts)
    w, _ = make(hip, orc, E * n, K, 7)
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R))
    g = torch.Generator().manual_seed(form)
    x = bf(torch.randn(R, K, generator=g) * (8.0 / K ** 0.5))
    off = torch.tensor([0, 70, 70, 75, R], dtype=torch.int32).cuda()
    tokens = torch.randperm(R, generator=g)
    plan_tokens = tokens.to(torch.int32).cuda()
    plan = hip.expert_plan_over(off, plan_tokens, plan_tokens)
    rows = [0, 17, 69, 72, 75, 200, 331, R - 1]   # positions in the plan
    other = torch.ones(R, dtype=torch.bool)
    other[rows] = False
    hip.tune_grouped(form)
    for gather in (False, True):
        at = tokens[rows].tolist() if gather else rows   # their rows of x
        for space in (None, ws):
            out = {}
            for name, xi in (("clean", x), ("bad", poisoned(x, at))):
                print(f"nonfinite form {form} {act} gather={gather} ws={space is not None} {name}", flush=True)
                y = torch.empty(R, n // 2 if act == "swiglu" else n, dtype=torch.bfloat16, device="cuda")
                hip.gemm_grouped_w4a16(y, w, xi.cuda(), plan, R, gather, act=getattr(hip, "ACT_" + act.upper()),
                                       ws=space)
                torch.cuda.synchronize()
                out[name] = y.cpu()
            assert not torch.isfinite(out["bad"][rows]).any()
            assert torch.isfinite(out["clean"]).all() and torch.equal(out["bad"][other], out["clean"][other])
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)
