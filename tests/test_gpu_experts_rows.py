"""Rows past what one launch takes (its grid has fewer than 2^32 threads): 2^24 tokens of
the weighted sum, 2^26 of the router, 2^24 rows of the fp16 operands' pass."""
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


def test_combine_rows(hip):
    import torch

    T, dim = (1 << 24) + 3, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    y = torch.empty(T, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    res = torch.empty(T, dim, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    wt = torch.rand(T, device="cuda", generator=g)
    pos = torch.arange(T - 1, -1, -1, dtype=torch.int32, device="cuda")
    pos[::3] = -1
    offsets = torch.zeros(9, dtype=torch.int32, device="cuda")
    plan = hip.expert_plan_over(offsets, pos, pos)
    out = torch.full((T + 1, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    print(f"combine rows T={T}", flush=True)
    hip.combine_experts(out, y, wt, T, 1, dim, plan, residual=res)
    torch.cuda.synchronize()
    assert (out[T] == 7.0).all()
    term = wt[:, None].double() * y.flip(0).double()
    term[::3] = 0
    ref = res.double() + term
    # two terms added in fp32, one rounding to bf16
    sums = 2 * 2.0 ** -24 * (res.double().abs() + term.abs())
    assert ((out[:T].double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + sums) + sums).all()


@pytest.mark.parametrize("f32", [False, True])
def test_route_rows(hip, f32):
    import torch

    T, E = (1 << 26) + 5, 2
    t = torch.arange(T, device="cuda")
    logits = torch.zeros(T, E, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    want = ((t >> 3) ^ t) & 1
    logits[t, want] = 1.0
    ids = torch.full((T + 1,), -7, dtype=torch.int32, device="cuda")
    wt = torch.full((T + 1,), -7.0, device="cuda")
    arrays = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (E + 1, T, T)]
    plan = hip.expert_plan_over(*arrays)
    print(f"route rows T={T} f32={f32}", flush=True)
    (hip.route_experts_f32 if f32 else hip.route_experts)(ids, wt, logits, T, E, 1, True, plan)
    torch.cuda.synchronize()
    assert torch.equal(ids[:T].long(), want) and int(ids[T]) == -7
    assert (wt[:T] == 1.0).all() and float(wt[T]) == -7.0
    ones = int(want.sum())
    assert arrays[0].tolist() == [0, T - ones, T]
    assert torch.equal(arrays[1][:T - ones].long(), t[want == 0]) and torch.equal(arrays[1][T - ones:].long(), t[want == 1])
    assert torch.equal(arrays[2][arrays[1].long()].long(), t)


class Rows:
    """Rows of a device tensor, copied when indexed by a list."""

    def __init__(self, t):
        self.t = t

    def __getitem__(self, rows):
        import torch

        return torch.stack([self.t[r] for r in rows]).cpu()


def test_half_rows(hip, orc):
    import torch

    E, n, K = 2, 128, 128
    R = (1 << 24) + 5
    w, wq = make(hip, orc, E * n, K, 61)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(R, K, dtype=torch.bfloat16, device="cuda").normal_(0, 8.0 / K ** 0.5, generator=g)
    y = torch.full((R + 1, n // 2), 7.0, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, R - 40, R], dtype=torch.int32).cuda()
    tokens = torch.zeros(R, dtype=torch.int32, device="cuda")
    plan = hip.expert_plan_over(offsets, tokens, tokens)
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(w, R))
    print(f"half rows R={R}", flush=True)
    hip.gemm_grouped_w4a16(y[:R], w, x, plan, R, False, act=hip.ACT_SWIGLU, ws=ws)
    torch.cuda.synchronize()
    assert (y[R] == 7.0).all()
    for e, rows in ((0, [0, (1 << 22) - 1, 1 << 22, (1 << 23) + 1, R - 41]), (1, [R - 40, R - 6, R - 5, R - 1])):
        check(Rows(y), Rows(x), wq[e * n:(e + 1) * n], None, "swiglu", None, rows, rounded=True, bits=11)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)
