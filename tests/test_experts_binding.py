"""What the Python calls of a product with an epilogue and of a layer of experts refuse:
tensors of another type, with gaps, in host memory or on another GPU, whose addresses the
kernels would read as something else (CPU only: every call ends before its launch)."""
import pytest
import torch

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
T, E, K, N, TOP = 4, 8, 256, 128, 2


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def weights(hip, rows):
    return hip.W4A16Weights(0x1000, 0x2000, 0x3000, rows, K, 128, K // 128)


def calls(hip):
    """name: (call with arguments by name, {argument: (shape, type)})"""
    plan = hip.ExpertPlan(0x1000, 0x2000, 0x3000, E, 64)
    wd, we = weights(hip, N), weights(hip, E * N)
    R = T * TOP
    return {
        "linear_epilogue": (lambda y, x, bias, residual: hip.linear_epilogue_w4a16(
            y, wd, x, T, bias=bias, residual=residual, stream=0),
            {"y": ((T, N), BF), "x": ((T, K), BF), "bias": ((N,), BF), "residual": ((T, N), BF)}),
        "route": (lambda ids, weights, logits: hip.route_experts(
            ids, weights, logits, T, E, TOP, True, plan, stream=0),
            {"ids": ((R,), I32), "weights": ((R,), F32), "logits": ((T, E), BF)}),
        "route_f32": (lambda ids, weights, logits: hip.route_experts_f32(
            ids, weights, logits, T, E, TOP, True, plan, stream=0),
            {"ids": ((R,), I32), "weights": ((R,), F32), "logits": ((T, E), F32)}),
        "route_ids": (lambda ids: hip.route_expert_ids(plan, ids, T, TOP, stream=0), {"ids": ((T, TOP), I32)}),
        "grouped": (lambda y, x, bias: hip.gemm_grouped_w4a16(
            y, we, x, plan, R, True, bias=bias, x_rows=T, stream=0),
            {"y": ((R, N), BF), "x": ((T, K), BF), "bias": ((E * N,), BF)}),
        "combine": (lambda out, y, weights, residual: hip.combine_experts(
            out, y, weights, T, TOP, N, plan, residual=residual, stream=0),
            {"out": ((T, N), BF), "y": ((R, N), BF), "weights": ((T, TOP), F32), "residual": ((T, N), BF)}),
        "plan": (lambda offsets, tokens, pos: hip.expert_plan_over(offsets, tokens, pos),
                 {"offsets": ((E + 1,), I32), "tokens": ((R,), I32), "pos": ((R,), I32)}),
    }


class On:
    """A tensor as the binding sees it, on GPU `device`."""

    def __init__(self, shape, dtype, device):
        t = torch.empty(shape, dtype=dtype)
        self.nbytes, self.dtype, self.device_index = t.nbytes, dtype, device
        self.numel, self.is_contiguous, self.element_size = t.numel, t.is_contiguous, t.element_size

    def get_device(self):
        return self.device_index

    def data_ptr(self):
        return 0x10000


ALL = [(c, a) for c, n in (("linear_epilogue", ("y", "x", "bias", "residual")), ("route", ("ids", "weights", "logits")),
                           ("route_f32", ("ids", "weights", "logits")), ("route_ids", ("ids",)),
                           ("grouped", ("y", "x", "bias")), ("combine", ("out", "y", "weights", "residual")),
                           ("plan", ("offsets", "tokens", "pos"))) for a in n]


@pytest.mark.parametrize("name,arg", ALL)
def test_refused(hip, name, arg):
    call, args = calls(hip)[name]
    # the other arguments: raw addresses, which are trusted (the plan takes tensors alone)
    here = hip._place(0)[0] if name != "plan" else 0
    rest = {a: 0x10000 if name != "plan" else On(s, d, here) for a, (s, d) in args.items()}
    shape, dtype = args[arg]
    wrong = {BF: (F32, torch.float16, torch.uint8), F32: (BF, torch.float64, I32), I32: (torch.int64, F32, torch.int16)}
    for d in wrong[dtype]:
        big = (8 * shape[0],) + shape[1:]   # enough bytes in any type
        with pytest.raises(ValueError, match="type"):
            call(**{**rest, arg: torch.empty(big if name != "plan" else shape, dtype=d)})
    gaps = torch.empty(shape[:-1] + (2 * shape[-1],), dtype=dtype)[..., ::2]
    assert not gaps.is_contiguous()
    with pytest.raises(ValueError, match="contiguous"):
        call(**{**rest, arg: gaps})
    whole = torch.empty(shape, dtype=dtype)
    with pytest.raises(ValueError, match="GPU"):
        call(**{**rest, arg: whole})
    with pytest.raises(ValueError, match="GPU"):
        call(**{**rest, arg: On(shape, dtype, here + 1)})


@pytest.mark.parametrize("name,arg", [p for p in ALL if p[0] != "plan"])
def test_short(hip, name, arg):
    call, args = calls(hip)[name]
    shape, dtype = args[arg]
    n = 1
    for s in shape:
        n *= s
    with pytest.raises(ValueError, match="holds"):
        call(**{**{a: 0x10000 for a in args}, arg: torch.empty(n - 1, dtype=dtype)})


def test_sixteen_bit_views(hip):
    """int16 views of bf16 are bf16 (no other framework of the host has the type)."""
    call, args = calls(hip)["linear_epilogue"]
    with pytest.raises(ValueError, match="GPU"):   # past the type
        call(**{**{a: 0x10000 for a in args}, "x": torch.empty((T, K), dtype=torch.int16)})


def test_plan_of_another_gpu(hip):
    """A plan's arrays lie on one GPU, which need not be the current one yet."""
    _, args = calls(hip)["plan"]
    on = {a: On(s, d, 1) for a, (s, d) in args.items()}
    p = hip.expert_plan_over(**on)
    assert (p.offsets, p.tokens, p.pos, p.experts, p.max_pairs) == (0x10000, 0x10000, 0x10000, E, T * TOP)
    with pytest.raises(ValueError, match="GPU"):
        hip.expert_plan_over(**{**on, "pos": On(*args["pos"], 0)})
