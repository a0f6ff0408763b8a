"""The 8-bit rows, their products and log probabilities as a program runs them: one after
the other, captured and replayed, on two streams, beside the rows of others."""
import ctypes
import math
import threading

import pytest
import torch

from a8_util import GROUP, from_layout, product, random_rows, random_weights, sum_tolerance, to_layout

pytestmark = pytest.mark.gpu

HIDDEN, INTER, VOCAB, EPS = 640, 1280, 2112, 1e-6


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


@pytest.fixture(scope="module")
def model(hip):
    """Two layers of gate|up and down with their norms, a head with its norm."""
    layers = []
    for i in range(2):
        up, down = (random_weights(hip, n, k, 40 + 2 * i + j) for j, (n, k) in
                    enumerate(((2 * INTER, HIDDEN), (HIDDEN, INTER))))
        layers.append((norm_weights(i), up, down))
    head = random_weights(hip, VOCAB, HIDDEN, 50)
    yield layers, norm_weights(9), head
    for _, up, down in layers:
        hip.awq_free(up[0])
        hip.awq_free(down[0])
    hip.awq_free(head[0])


def norm_weights(seed):
    return (0.1 * torch.randn(HIDDEN, generator=torch.Generator().manual_seed(seed))).bfloat16().cuda()


class Buffers:
    """What a pass of up to `rows` rows keeps."""

    def __init__(self, hip, rows, top_k=5, asked=2):
        bf16 = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        f32 = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        self.hip, self.rows, self.top_k, self.asked = hip, rows, top_k, asked
        self.a, self.b = hip.a8_alloc(rows, HIDDEN), hip.a8_alloc(rows, INTER)
        self.h, self.mid, self.back = bf16(rows, HIDDEN), bf16(rows, INTER), bf16(rows, HIDDEN)
        self.logits, self.lp = f32(rows, VOCAB), f32(rows, asked)
        self.entropy, self.top = f32(rows), f32(rows, top_k)
        self.ids = torch.zeros(rows, top_k, dtype=torch.int32, device="cuda")
        self.targets = torch.zeros(rows, asked, dtype=torch.int32, device="cuda")
        self.ws = hip.gemm_workspace_alloc(max(256 << 20, hip.logprobs_workspace(rows, VOCAB, top_k)))

    def free(self):
        self.hip.a8_free(self.a)
        self.hip.a8_free(self.b)
        self.hip.gemm_workspace_free(self.ws)

    def outputs(self):
        return [t.clone() for t in (self.h, self.logits, self.lp, self.entropy, self.ids, self.top)]


def run(hip, model, s, x, T):
    """The pass: every layer's down projection is added by the next norm."""
    layers, last, head = model
    s.h[:T].copy_(x[:T])
    residual = None
    for norm, up, down in layers:
        hip.rmsnorm_a8(s.a, s.h, norm, T, EPS, residual=residual, out=s.h if residual is not None else None)
        hip.linear_w4a8(s.mid, up[0], s.a, T, s.ws, act=hip.ACT_SWIGLU)
        hip.quantize_a8(s.b, s.mid, T)
        hip.linear_w4a8(s.back, down[0], s.b, T, s.ws)
        residual = s.back
    hip.rmsnorm_a8(s.a, s.h, last, T, EPS, residual=residual, out=s.h)
    hip.linear_w4a8_f32(s.logits, head[0], s.a, T, s.ws)
    hip.logprobs(s.lp, s.logits, s.targets, T, VOCAB, s.ws, entropy=s.entropy, top_ids=s.ids,
                 top_logprobs=s.top, top_k=s.top_k)


def rows(T, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, HIDDEN, generator=g) * (0.5 + torch.rand(HIDDEN, generator=g))
    return x.bfloat16().cuda(), torch.randint(0, VOCAB, (T, 2), generator=g, dtype=torch.int32).cuda()


def quantized(v):
    """Values in 8 bits, and how far apart codes of the same values may come out: v has a
    relative error of 2^-22 (fp32 norms), so the code of a value that close to the middle
    of two may be either, one step of its group's."""
    g = v.view(v.shape[0], -1, GROUP)
    scale = g.abs().amax(-1, keepdim=True) / 127
    x = torch.where(scale > 0, g / scale, torch.zeros_like(g))
    q = torch.round(x)
    close = ((x - torch.floor(x) - 0.5).abs() < x.abs() * 2.0 ** -21).double()
    return (q * scale).view_as(v), (close * scale).view_as(v)


def bf16_near(got, want, tolerance):
    """got, rounded to bf16, is within `tolerance` of want before that rounding."""
    bad = (got.double() - want).abs() > tolerance + want.abs() * 2.0 ** -8 + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {(got.double() - want).abs()[bad].max()}"


@pytest.mark.parametrize("T", [1, 2, 9, 16, 31, 40, 77, 130, 300])
def test_a_pass(hip, model, T):
    """Step by step: each step's result against 64 bits over what the step before stored."""
    layers, last, head = model
    s = Buffers(hip, T)
    x, s.targets[:] = rows(T, T)
    h, residual = x.double(), None

    def norm(w):
        nonlocal h
        if residual is not None:
            h = (h + s.back.double()).float().bfloat16().double()   # one rounding of an exact sum
        return h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * (1 + w.double())

    def linear(weights, a, values):
        """The product over the stored codes; those against the values' own."""
        w, less, ws = weights
        q, scale = from_layout(a.q_tensor), a.scale_tensor
        stored = q.double() * scale.t().double().repeat_interleave(GROUP, 1)
        want, spread = quantized(values)
        assert ((stored - want).abs() <= spread + want.abs() * 2.0 ** -21 + 1e-30).all()
        v, size = product(q, scale, less, ws)
        return v, sum_tolerance(size, q.shape[1] // GROUP)

    def codes(a, k):
        a.q_tensor, a.scale_tensor = read_rows(a, T, k)
        return a

    s.h.copy_(x)
    for w, up, down in layers:
        hip.rmsnorm_a8(s.a, s.h, w, T, EPS, residual=residual, out=s.h if residual is not None else None)
        v, tol = linear(up, codes(s.a, HIDDEN), norm(w))
        assert (s.h.double() == h).all()
        hip.linear_w4a8(s.mid, up[0], s.a, T, s.ws, act=hip.ACT_SWIGLU)
        gate, u = v[:, :INTER], v[:, INTER:]
        tg, tu = tol[:, :INTER], tol[:, INTER:]
        silu = gate * torch.sigmoid(gate)
        # silu's slope is below 1.1; its own fp32 steps 8
        bf16_near(s.mid, silu * u, 1.1 * tg * (u.abs() + tu) + silu.abs() * tu + (silu * u).abs() * 8 * 2.0 ** -24)
        hip.quantize_a8(s.b, s.mid, T)
        v, tol = linear(down, codes(s.b, INTER), s.mid.double())
        hip.linear_w4a8(s.back, down[0], s.b, T, s.ws)
        bf16_near(s.back, v, tol)
        residual = s.back
    hip.rmsnorm_a8(s.a, s.h, last, T, EPS, residual=residual, out=s.h)
    v, tol = linear(head, codes(s.a, HIDDEN), norm(last))
    hip.linear_w4a8_f32(s.logits, head[0], s.a, T, s.ws)
    assert ((s.logits.double() - v).abs() <= tol).all()
    hip.logprobs(s.lp, s.logits, s.targets, T, VOCAB, s.ws, entropy=s.entropy, top_ids=s.ids,
                 top_logprobs=s.top, top_k=s.top_k)
    z = s.logits.double()
    full = torch.log_softmax(z, 1)
    # x - m and less the log: half a step of each; the log a few steps of at most log n
    close = 2.0 ** -24 * (2 * (z.amax(1, keepdim=True) - z.amin(1, keepdim=True)) + 64)
    assert ((s.lp.double() - full.gather(1, s.targets.long())).abs() <= close).all()
    assert (s.ids.long() == torch.sort(z, dim=1, descending=True, stable=True).indices[:, :s.top_k]).all()
    assert ((s.top.double() - full.gather(1, s.ids.long())).abs() <= close).all()
    entropy = -(full.exp() * full).sum(1)
    assert ((s.entropy.double() - entropy).abs() <= 64 * 2.0 ** -24 * (1 + math.log(VOCAB))).all()
    # and all of it in a row gives the same
    before = s.outputs()
    run(hip, model, s, x, T)
    for one, two in zip(before, s.outputs()):
        assert torch.equal(one, two)
    s.free()


def read_rows(a, T, k):
    """The codes [T][k] and scales [k/128][T] that a holds, as tensors."""
    q = torch.zeros(T, k, dtype=torch.int8, device="cuda")
    scale = torch.zeros(k // GROUP, a.max_rows, device="cuda")
    torch.cuda.synchronize()
    copy = ctypes.CDLL("libamdhip64.so").hipMemcpy
    for t, p in ((q, a.q), (scale, a.scale)):
        assert copy(ctypes.c_void_p(t.data_ptr()), ctypes.cast(p, ctypes.c_void_p),
                    ctypes.c_size_t(t.numel() * t.element_size()), 3) == 0
    torch.cuda.synchronize()
    return q, scale[:, :T].contiguous()


@pytest.mark.parametrize("T", [1, 9, 40, 200])
def test_captured_and_replayed(hip, model, T):
    """A captured pass replayed over other inputs, with eager passes over the same buffers and
    workspace in between."""
    s = Buffers(hip, T)
    inputs = [rows(T, 100 + i) for i in range(3)]
    x = inputs[0][0].clone()
    s.targets[:] = inputs[0][1]
    eager = []
    for xi, ti in inputs:
        s.targets[:] = ti
        run(hip, model, s, xi, T)
        eager.append(s.outputs())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(hip, model, s, x, T)
    for i in (1, 2, 0, 1):
        x.copy_(inputs[i][0])
        s.targets[:] = inputs[i][1]
        graph.replay()
        torch.cuda.synchronize()
        for one, two in zip(eager[i], s.outputs()):
            assert torch.equal(one, two)
        other = (i + 1) % 3
        s.targets[:] = inputs[other][1]
        run(hip, model, s, inputs[other][0], T)
        torch.cuda.synchronize()
        for one, two in zip(eager[other], s.outputs()):
            assert torch.equal(one, two)
    del graph
    s.free()


@pytest.mark.parametrize("T", [9, 70])
def test_two_graphs_share_their_buffers(hip, model, T):
    s = Buffers(hip, T)
    (x0, t0), (x1, _) = rows(T, 7), rows(T, 8)
    s.targets[:] = t0
    want = []
    for x in (x0, x1):
        run(hip, model, s, x, T)
        want.append(s.outputs())
    torch.cuda.synchronize()
    graphs = []
    for x in (x0, x1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(hip, model, s, x, T)
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        torch.cuda.synchronize()
        for one, two in zip(want[i], s.outputs()):
            assert torch.equal(one, two)
    del graphs
    s.free()


@pytest.mark.parametrize("T", [1, 12, 90])
def test_two_streams(hip, model, T):
    """Passes at the same time on two streams, each with its buffers and workspace."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    kept = [Buffers(hip, T) for _ in range(2)]
    inputs = [rows(T, 200 + i) for i in range(2)]
    want = []
    for s, (x, t) in zip(kept, inputs):
        s.targets[:] = t
        run(hip, model, s, x, T)
        want.append(s.outputs())
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, s, (x, _) in zip(streams, kept, inputs):
            with torch.cuda.stream(stream):
                run(hip, model, s, x, T)
    torch.cuda.synchronize()
    for s, w in zip(kept, want):
        for one, two in zip(w, s.outputs()):
            assert torch.equal(one, two)
        s.free()


def test_two_threads(hip, model):
    """Host threads that launch at once, on their own streams and buffers, other row counts."""
    sizes = (9, 40, 24, 1)
    kept = [Buffers(hip, T) for T in sizes]
    inputs = [rows(T, 300 + T) for T in sizes]
    want = []
    for T, s, (x, t) in zip(sizes, kept, inputs):
        s.targets[:] = t
        run(hip, model, s, x, T)
        want.append(s.outputs())
    torch.cuda.synchronize()
    errors = []

    def work(T, s, x, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    run(hip, model, s, x, T)
                torch.cuda.current_stream().synchronize()
                for one, two in zip(w, s.outputs()):
                    assert torch.equal(one, two)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(T, s, x, w)) for T, s, (x, _), w in zip(sizes, kept, inputs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for s in kept:
        s.free()


@pytest.mark.parametrize("T,more", [(1, 3), (9, 7), (33, 31), (64, 200)])
def test_rows_behind_the_last(hip, model, T, more):
    """A batch of T rows in buffers of more: the others stay, whatever they hold."""
    s, exact = Buffers(hip, T + more), Buffers(hip, T)
    x, t = rows(T, 3)
    exact.targets[:] = t
    run(hip, model, exact, x, T)
    full, _ = rows(T + more, 4)
    s.targets[:] = 5
    run(hip, model, s, full, T + more)   # what an earlier, larger batch left
    for b in (s.h, s.logits, s.lp, s.entropy, s.top):
        b[T:] = float("nan")
    s.ids[T:] = -7
    s.targets[:T] = t
    s.targets[T:] = 1 << 30
    run(hip, model, s, x, T)
    torch.cuda.synchronize()
    for what, one, two in zip(("h", "logits", "lp", "entropy", "ids", "top"), exact.outputs(), s.outputs()):
        assert torch.equal(one, two[:T]), what
        rest = two[T:]
        assert (rest == -7).all() if rest.dtype == torch.int32 else rest.isnan().all(), (what, rest)
    exact.free()
    s.free()


@pytest.mark.parametrize("T", [3, 16, 31])
def test_captured_without_a_call_before(hip, T):
    """A shape whose first call is the captured one."""
    n, k = 192, 384 + GROUP * T
    w, less, ws = random_weights(hip, n, k, 60 + T)
    q, scale = random_rows(T, k, 61 + T)
    codes = to_layout(q)
    a = hip.a8_over(codes, scale)
    y = torch.zeros(T, n, device="cuda")
    space = hip.gemm_workspace_alloc(256 << 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip.linear_w4a8_f32(y, w, a, T, space)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        v, size = product(q, scale, less, ws)
        assert ((y.double() - v).abs() <= sum_tolerance(size, k // GROUP)).all()
    del graph
    hip.gemm_workspace_free(space)
    hip.awq_free(w)
