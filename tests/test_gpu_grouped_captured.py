"""qw4_gemm_grouped captured once and replayed over new rows, another routing and another
workspace's content, as eager calls of the same inputs compute it: ungated tiles with fp16
operands (the rows and exponents in the workspace), and each other kernel."""
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


@pytest.mark.parametrize("form", [0, 1, 3, 4, 5])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
def test_captured(hip, orc, act, gather, form):
    E, n, K, T, k = 8, 384, 640, 120, 3
    R = T * k
    w, _ = make(hip, orc, E * n, K, 71)
    g = torch.Generator().manual_seed(form)
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R))
    rows = T if gather else R
    xs = [bf(torch.randn(rows, K, generator=g) * (8.0 / K ** 0.5)).cuda() for _ in range(4)]
    ids = [torch.randint(-1, E, (T, k), generator=g, dtype=torch.int32).cuda() for _ in range(4)]
    ids[2][:, :] = 5   # one expert with every pair
    bias = bf(torch.randn(E * n, generator=g)).cuda()
    plan = hip.expert_plan_alloc(E, R)
    x, chosen = xs[0].clone(), ids[0].clone()
    y = torch.empty(R, n // 2 if act == "swiglu" else n, dtype=torch.bfloat16, device="cuda")
    hip.tune_grouped(form)

    def run():
        hip.route_expert_ids(plan, chosen, T, k)
        hip.gemm_grouped_w4a16(y, w, x, plan, R, gather, bias=bias, act=getattr(hip, "ACT_" + act.upper()), ws=ws)

    print(f"captured grouped form {form} {act} gather={gather}", flush=True)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    other = torch.empty(rows, E * n // 2, dtype=torch.bfloat16, device="cuda")
    for i in (0, 1, 2, 3, 1):
        x.copy_(xs[i])
        chosen.copy_(ids[i])
        y.fill_(7.0)
        run()
        torch.cuda.synchronize()
        eager = y.clone()
        hip.linear_epilogue_w4a16(other, w, xs[3 - i], rows, None, ws, act=hip.ACT_SWIGLU)   # other work in the workspace
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager), i
    del graph
    hip.expert_plan_free(plan)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)
