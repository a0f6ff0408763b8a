"""The calls of a layer of experts and of a product with an epilogue as a server makes
them: captured and replayed with other work in between, on streams of their own at the
same time, from two threads, over a part of the experts, and with workspaces that are
too small or not aligned."""
import threading

import pytest

from test_gpu_linear_epilogue import bf, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


# weight, rows, activation: decode and verify passes, two blocks of rows in one pass, a
# last pass of one row, tiles of the prefill product whole and split over k
CAPTURED = [(1152, 2176, 1, "silu"), (1152, 2176, 1, "swiglu"), (1152, 2176, 7, "gelu"), (5120, 4096, 17, "none"),
            (5120, 4096, 24, "swiglu"), (1152, 2176, 33, "gelu_tanh"), (256, 2176, 259, "silu"),
            (256, 2176, 259, "swiglu"), (1152, 2176, 700, "swiglu"), (9472, 2176, 500, "swiglu")]


@pytest.mark.parametrize("N,K,T,act", CAPTURED)
def test_epilogue_captured(hip, orc, N, K, T, act):
    """Replays with new x, y as the residual, equal the eager calls, whatever ran between
    them in the same scratch and workspace."""
    import torch

    w, _ = make(hip, orc, N, K, N + T)
    width = N // 2 if act == "swiglu" else N
    g = torch.Generator().manual_seed(T)
    xs = [bf(torch.randn(T, K, generator=g) * (8.0 / K ** 0.5)).cuda() for _ in range(4)]
    bias, res = bf(torch.randn(N, generator=g)).cuda(), bf(torch.randn(T, width, generator=g)).cuda()
    scratch = hip.gemv_scratch_alloc(K, N, 128, 16)
    ws = hip.gemm_workspace_alloc(256 << 20)
    x, y = xs[0].clone(), res.clone()

    def run():
        hip.linear_epilogue_w4a16(y, w, x, T, scratch, ws, bias=bias, act=getattr(hip, "ACT_" + act.upper()),
                                  residual=y)

    print(f"captured {N}x{K} T={T} {act}", flush=True)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    other = torch.empty(300, N, dtype=torch.bfloat16, device="cuda")
    ox = bf(torch.randn(300, K, generator=g)).cuda()
    for xi in xs:
        x.copy_(xi)
        y.copy_(res)
        run()
        torch.cuda.synchronize()
        eager = y.clone()
        hip.linear_epilogue_w4a16(other, w, ox, 300, scratch, ws, act=hip.ACT_GELU)   # other work in the workspace
        y.copy_(res)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
    del graph
    hip.gemv_scratch_free(scratch)
    hip.gemm_workspace_free(ws)
    hip.awq_free(w)


class Layer:
    """A layer of experts with buffers, a plan and a workspace of its own."""

    def __init__(self, hip, wu, wd, T, E, k, H, I, seed, first=0, experts=None):
        import torch

        g = torch.Generator().manual_seed(seed)
        self.hip, self.wu, self.wd, self.dims = hip, wu, wd, (T, E, k, H)
        self.x = bf(torch.randn(T, H, generator=g) * (4.0 / H ** 0.5)).cuda()
        self.logits = torch.randn(T, E, generator=g).cuda()
        self.ids = torch.zeros(T * k, dtype=torch.int32, device="cuda")
        self.wt = torch.zeros(T * k, device="cuda")
        self.h = torch.zeros(T * k, I, dtype=torch.bfloat16, device="cuda")
        self.y = torch.zeros(T * k, H, dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        self.plan = hip.expert_plan_alloc(E if experts is None else experts, T * k)
        self.first, self.whole = first, experts is None
        self.ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(wu, T))
        torch.cuda.synchronize()

    def run(self, stream=None):
        hip, (T, E, k, H) = self.hip, self.dims
        hip.route_experts_f32(self.ids, self.wt, self.logits, T, E, k, True, self.plan if self.whole else None, stream)
        if not self.whole:   # this part's experts alone
            hip.route_expert_ids(self.plan, self.ids - self.first, T, k, stream)
        hip.gemm_grouped_w4a16(self.h, self.wu, self.x, self.plan, T * k, True, act=hip.ACT_SWIGLU, ws=self.ws,
                               stream=stream)
        hip.gemm_grouped_w4a16(self.y, self.wd, self.h, self.plan, T * k, False, stream=stream)
        hip.combine_experts(self.out, self.y, self.wt, T, k, H, self.plan, residual=self.x, stream=stream)

    def free(self):
        self.hip.expert_plan_free(self.plan)
        self.hip.gemm_workspace_free(self.ws)


@pytest.mark.parametrize("threads", [False, True])
def test_layers_at_once(hip, orc, threads):
    """Layers over the same weights on a stream each, queued together or by a thread
    each, give what each gives alone."""
    import torch

    E, k, H, I = 16, 4, 640, 384
    wu, wd = make(hip, orc, E * 2 * I, H, 21)[0], make(hip, orc, E * H, I, 22)[0]
    layers = [Layer(hip, wu, wd, T, E, k, H, I, T) for T in (1, 13, 90, 700)]
    alone = []
    for a in layers:
        a.run()
        torch.cuda.synchronize()
        alone.append(a.out.clone())
    streams = [torch.cuda.Stream() for _ in layers]
    for rep in range(3):
        print(f"layers at once {threads} {rep}", flush=True)
        for a in layers:
            a.out.zero_()
            a.h.fill_(float("nan"))
            a.y.fill_(float("nan"))
        torch.cuda.synchronize()
        if threads:
            failed = []

            def work(a, s):
                try:
                    for _ in range(5):
                        a.run(s)
                except Exception as e:   # a thread's exception would be lost
                    failed.append(e)

            ts = [threading.Thread(target=work, args=p) for p in zip(layers, streams)]
            for t in ts:
                t.start()
            for t in ts:
                t.join()
            assert not failed, failed
        else:
            for _ in range(5):
                for a, s in zip(layers, streams):
                    a.run(s)
        torch.cuda.synchronize()
        for a, ref in zip(layers, alone):
            assert torch.equal(a.out, ref)
    for a in layers:
        a.free()
    hip.awq_free(wu)
    hip.awq_free(wd)


@pytest.mark.parametrize("T", [1, 40, 333])
def test_experts_in_parts(hip, orc, T):
    """The experts in two halves, each with the plan of its own ids, as two GPUs would
    hold them: the halves' sums are the whole's. Each row of y is the same up to the tiles
    that its half takes, so weights rounded to bf16 or not: 2^-8 of each term, 6 of K random
    ones, per factor; and one rounding of each half."""
    import torch

    E, k, H, I = 16, 4, 512, 256
    (wu, qu), (wd, qd) = make(hip, orc, E * 2 * I, H, 31), make(hip, orc, E * H, I, 32)
    whole = Layer(hip, wu, wd, T, E, k, H, I, T)
    whole.run()
    halves = []
    for part in range(2):
        e0 = part * E // 2
        rows_u, rows_d = E * I, E * H // 2
        hu, hd = sub_experts(hip, wu, rows_u * part, rows_u), sub_experts(hip, wd, rows_d * part, rows_d)
        a = Layer(hip, hu, hd, T, E, k, H, I, T, first=e0, experts=E // 2)
        a.run()
        halves.append(a)
    torch.cuda.synchronize()
    assert torch.equal(halves[0].ids, whole.ids)
    x = whole.x.double()
    got = sum(a.out.double() for a in halves) - x   # the residual once
    ref = whole.out.double()
    # the bound of a row: hidden values from gate and up, then down
    tol = torch.zeros_like(ref)
    ids, wt = whole.ids.view(T, k).cpu(), whole.wt.view(T, k).cpu().double()
    xc = x.cpu()
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            u, d = qu[e * 2 * I:(e + 1) * 2 * I], qd[e * H:(e + 1) * H]
            v = u @ xc[t]
            ev = 6 * 2.0 ** -8 * ((u ** 2) @ xc[t] ** 2).sqrt()
            hid = v[:I] * torch.sigmoid(v[:I]) * v[I:]
            eh = 1.13 * ev[:I] * (v[I:].abs() + ev[I:]) + (v[:I] * torch.sigmoid(v[:I])).abs() * ev[I:]
            eh = eh + 2.0 ** -8 * (hid.abs() + eh)
            row = d @ hid
            # eh's signs are those of random roundings: 6 of them, not their sum
            er = 6 * ((d ** 2) @ (eh ** 2 + (2.0 ** -8 * hid) ** 2)).sqrt()
            er = er + 2.0 ** -8 * (row.abs() + er)
            tol[t] += (wt[t, j] * er).cuda()
    tol = 2 * tol + 2.0 ** -8 * (ref.abs() + sum(a.out.double().abs() for a in halves) + 2 * tol)
    assert ((got - ref).abs() <= tol).all()
    for a in halves:
        a.free()
    whole.free()
    hip.awq_free(wu)
    hip.awq_free(wd)


def sub_experts(hip, w, row0, rows):
    """Weight rows [row0, row0 + rows) of w in place: its blocks of 64 rows x a group
    (4096 bytes of weights, 160 of scales with zero points, 32 of zero points) go row by row."""
    at = row0 // 64 * w.num_groups
    return hip.W4A16Weights(w.qweight + at * 4096, w.scale + at * 160, w.zeros + at * 32, rows, w.in_f,
                            w.group_size, w.num_groups)


def test_workspace_sizes(hip, orc):
    """A gated product takes fp16 operands from the size that qw4_epilogue_workspace
    gives; with a byte less, or a workspace off its 256-byte line, it is the product without
    one, and nothing behind the workspace's end is written."""
    import torch

    T, E, n, K = 300, 2, 512, 512
    w, _ = make(hip, orc, E * n, K, 41)
    x = bf(torch.randn(T, K, generator=torch.Generator().manual_seed(1)) * (8.0 / K ** 0.5)).cuda()
    offsets = torch.tensor([0, 180, T], dtype=torch.int32).cuda()
    tokens = torch.arange(T, dtype=torch.int32).cuda()
    plan = hip.expert_plan_over(offsets, tokens, tokens)
    need = hip.epilogue_workspace(w, T)
    buf = torch.full((need + 4096,), 7, dtype=torch.uint8, device="cuda")
    base = (buf.data_ptr() + 255) & ~255
    calls = {
        "grouped": lambda y, ws: hip.gemm_grouped_w4a16(y, w, x, plan, T, False, act=hip.ACT_SWIGLU, ws=ws),
        "gathered": lambda y, ws: hip.gemm_grouped_w4a16(y, w, x, plan, T, True, act=hip.ACT_SWIGLU, ws=ws),
        "dense": lambda y, ws: hip.linear_epilogue_w4a16(y, w, x, T, None, ws, act=hip.ACT_SWIGLU),
    }
    hip.tune_grouped(3)   # the tiles, which take them
    for name, call in calls.items():
        width = E * n // 2 if name == "dense" else n // 2

        def out(ptr, size):
            y = torch.zeros(T, width, dtype=torch.bfloat16, device="cuda")
            ws = None
            if size is not None:
                ws = hip.GemmWorkspace()
                ws.buf, ws.bytes = ptr, size
            buf.fill_(7)
            call(y, ws)
            torch.cuda.synchronize()
            end = base - buf.data_ptr() + need
            assert (buf[end:] == 7).all()
            return y
        print(f"workspace {name}", flush=True)
        none = out(None, None)
        assert not torch.equal(out(base, need), none)
        assert torch.equal(out(base, need - 1), none)
        assert torch.equal(out(base + 128, need), none)
        assert torch.equal(out(base, 0), none)
    hip.tune_grouped(0)
    hip.awq_free(w)
