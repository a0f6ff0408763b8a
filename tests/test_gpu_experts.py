"""The router, its plan and the weighted sum of expert rows against plain 64-bit
forms: one token to thousands, expert counts around a wave's lane counts, ties,
masked experts, NaN and Inf logits, tokens that choose nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def route_ref(x, k, renorm):
    """x [T][E] float64 -> ids [T][k], weights [T][k], spread [T][k] = |v - largest|."""
    T, E = x.shape
    ids = np.full((T, k), -1, np.int64)
    w = np.zeros((T, k))
    spread = np.zeros((T, k))
    for t in range(T):
        live = [e for e in range(E) if x[t, e] > -np.inf]   # false for NaN
        order = sorted(live, key=lambda e: (-x[t, e], e))[:k]
        if not order:
            continue
        top = x[t, order[0]]

        def mass(e):
            return 1.0 if x[t, e] == top else np.exp(x[t, e] - top)

        total = sum(mass(e) for e in (order if renorm else live))
        for j, e in enumerate(order):
            ids[t, j], w[t, j] = e, mass(e) / total
            spread[t, j] = 0 if x[t, e] == top else min(abs(x[t, e] - top), 200.0)
    return ids, w, spread


def plan_ref(ids, E):
    T, k = ids.shape
    flat = ids.reshape(-1)
    live = (flat >= 0) & (flat < E)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[live], minlength=E)[:E])])
    order = [p for e in range(E) for p in np.nonzero(live & (flat == e))[0]]
    pos = np.full(T * k, -1, np.int64)
    pos[order] = np.arange(len(order))
    tokens = np.full(T * k, -1, np.int64)
    tokens[:len(order)] = np.array(order, np.int64) // k
    return offsets, tokens, pos


def logits_of(T, E, seed, kind):
    """Random logits on a coarse grid (so that they tie), exact in bf16, with rows
    of each awkward kind."""
    rng = np.random.default_rng(seed)
    x = np.round(rng.normal(size=(T, E)) * 4) / 4 if kind == "ties" else rng.normal(size=(T, E)) * 3
    if kind == "ties":
        x[rng.random((T, E)) < 0.2] = -np.inf          # masked experts
        x[rng.random((T, E)) < 0.05] = -0.0
        for t in range(0, T, 5):
            what = (t // 5) % 6
            if what == 0:
                x[t] = -np.inf                         # no expert at all
            elif what == 1:
                x[t, rng.integers(0, E)] = np.nan
            elif what == 2:
                x[t, rng.integers(0, E, 2)] = np.inf
            elif what == 3:
                x[t] = np.nan
            elif what == 4:
                x[t] = 0.0                             # every expert the same
            else:
                x[t] = -np.inf
                x[t, E - 1] = np.finfo(np.float32).min   # the lowest finite value (fp32)
    return x


SHAPES = [(0, 8, 2), (1, 1, 1), (1, 64, 8), (2, 16, 16), (3, 5, 2), (31, 65, 3), (32, 128, 8), (33, 64, 8),
          (64, 60, 4), (65, 60, 4), (200, 257, 4), (70, 1024, 16), (777, 60, 6), (1500, 513, 7), (4096, 128, 8)]


@pytest.mark.parametrize("kind", ["normal", "ties"])
@pytest.mark.parametrize("T,E,k", SHAPES)
def test_route(hip, T, E, k, kind):
    import torch

    for f32 in (False, True):
        x = torch.tensor(logits_of(T, E, 7 * T + E, kind), dtype=torch.float32)
        x = x if f32 else x.to(torch.bfloat16)
        ref = x.double().numpy()
        for renorm in (False, True):
            print(f"route T={T} E={E} k={k} {kind} f32={f32} renorm={renorm}", flush=True)
            d = x.cuda()
            guard = 3
            ids = torch.full((T * k + guard,), -77, dtype=torch.int32, device="cuda")
            w = torch.full((T * k + guard,), -77.0, device="cuda")
            offsets = torch.full((E + 1 + guard,), -77, dtype=torch.int32, device="cuda")
            tokens, pos = ids.clone(), ids.clone()
            plan = hip.expert_plan_over(offsets[:E + 1], tokens[:T * k], pos[:T * k])
            call = hip.route_experts_f32 if f32 else hip.route_experts
            call(ids, w, d, T, E, k, renorm, plan)
            torch.cuda.synchronize()
            want, ww, spread = route_ref(ref, k, renorm)
            got = ids[:T * k].cpu().numpy().reshape(T, k)
            assert np.array_equal(got, want)
            # per weight: the exponent's rounding (spread 2^-24), expf 2 ulp, up to 22 additions
            # of the sum, the terms' own errors in it, the division
            tol = (2 * np.maximum(spread, spread.max(initial=0) if not renorm else 0) + 64) * 2.0 ** -24
            gw = w[:T * k].cpu().double().numpy().reshape(T, k)
            assert (np.abs(gw - ww) <= tol * ww + 1e-37).all(), np.abs(gw - ww).max()
            o, tk, ps = plan_ref(want, E)
            assert np.array_equal(offsets[:E + 1].cpu().numpy(), o)
            assert np.array_equal(tokens[:T * k].cpu().numpy(), tk)
            assert np.array_equal(pos[:T * k].cpu().numpy(), ps)
            for t, n in ((ids, T * k), (w, T * k), (offsets, E + 1), (tokens, T * k), (pos, T * k)):
                assert (t[n:] == -77).all()
            if T:   # without a plan: the same choice
                ids2, w2 = torch.empty_like(ids), torch.empty_like(w)
                call(ids2, w2, d, T, E, k, renorm)
                assert torch.equal(ids2[:T * k], ids[:T * k]) and torch.equal(w2[:T * k], w[:T * k])


@pytest.mark.parametrize("T,E,k", [(0, 3, 1), (1, 1, 1), (1, 8, 16), (40, 7, 6), (43, 7, 6), (500, 33, 5), (9000, 1024, 16)])
def test_route_ids(hip, T, E, k):
    """Ids of another rule: some outside [0, experts), the same expert twice."""
    import torch

    rng = np.random.default_rng(T + E)
    ids = rng.integers(-2, E + 2, (T, k))
    ids[T // 3:T // 2] = E // 2
    p = hip.expert_plan_alloc(E, max(1, T * k) + 5)
    d = torch.tensor(ids, dtype=torch.int32).cuda()
    print(f"route_ids T={T} E={E} k={k}", flush=True)
    hip.route_expert_ids(p, d, T, k)
    torch.cuda.synchronize()
    from gpu_util import download

    want = plan_ref(ids, E)
    for ptr, ref in zip((p.offsets, p.tokens, p.pos), want):
        if len(ref):
            assert np.array_equal(download(ptr, 4 * len(ref)).view(np.int32), ref)
    hip.expert_plan_free(p)


@pytest.mark.parametrize("E,k", [(8, 1), (129, 3)])
def test_plan_edges(hip, E, k):
    """Pair counts around the plan's loads (4 a lane, 256 a wave, 8 loads ahead, 16 waves),
    ids on a 4-byte boundary, the arrays' ends left alone."""
    import torch

    rng = np.random.default_rng(E)
    for pairs in (129, 255, 256, 257, 4095, 4096, 4097, 4353, 30719, 32767, 32768, 32769, 36865, 70001):
        T = -(-pairs // k)
        n = T * k
        ids = rng.integers(-1, E + 1, (T, k))
        buf = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda")
        buf[1:] = torch.tensor(ids.reshape(-1), dtype=torch.int32)
        out = [torch.full((m + 3,), -77, dtype=torch.int32, device="cuda") for m in (E + 1, n, n)]
        plan = hip.expert_plan_over(*[o[:-3] for o in out])
        print(f"plan edges {n} pairs E={E}", flush=True)
        hip.route_expert_ids(plan, buf[1:], T, k)
        torch.cuda.synchronize()
        for o, ref in zip(out, plan_ref(ids, E)):
            assert np.array_equal(o[:-3].cpu().numpy(), ref)
            assert (o[-3:] == -77).all()


@pytest.mark.parametrize("residual", ["none", "other", "out"])
@pytest.mark.parametrize("T,k,dim", [(1, 1, 8), (1, 8, 2048), (9, 2, 2056), (5, 16, 5120), (130, 7, 88), (700, 8, 2048)])
def test_combine(hip, T, k, dim, residual):
    import torch

    g = torch.Generator().manual_seed(T + dim)
    n = T * k
    y = torch.randn(n, dim, generator=g).to(torch.bfloat16)
    w = torch.rand(T, k, generator=g)
    pos = torch.randperm(n, generator=g).to(torch.int32)
    drop = torch.rand(n, generator=g) < 0.3
    if T > 1:
        drop[:k] = True                 # a token without experts
    y[pos[drop].long()] = float("nan")  # rows of no pair
    w.view(-1)[drop] = float("inf")     # nor does their weight count
    pos[drop] = torch.where(torch.arange(int(drop.sum())) % 2 == 0, -1, n + 3).to(torch.int32)
    res = torch.randn(T, dim, generator=g).to(torch.bfloat16)
    terms = torch.zeros(k + 1, T, dim, dtype=torch.float64)
    if residual != "none":
        terms[k] = res.double()
    for j in range(k):
        p = pos.view(T, k)[:, j].long()
        live = (p >= 0) & (p < n)
        terms[j][live] = w[:, j:j + 1].double()[live] * y.double()[p[live]]
    ref = terms.sum(0)
    print(f"combine T={T} k={k} dim={dim} residual={residual}", flush=True)
    out = torch.full((T + 1, dim), 3.0, dtype=torch.bfloat16, device="cuda")
    if residual == "out":
        out[:T] = res.cuda()
    plan = hip.ExpertPlan(1, 1, 0, 8, n)   # the sum reads the positions alone (the others: any address)
    dpos = pos.cuda()
    plan.pos = dpos.data_ptr()
    r = None if residual == "none" else out if residual == "out" else res.cuda()
    hip.combine_experts(out, y.cuda(), w.cuda(), T, k, dim, plan, residual=r)
    torch.cuda.synchronize()
    # k + 1 fp32 additions over the terms, then one rounding to bf16
    sums = (k + 1) * 2.0 ** -24 * terms.abs().sum(0)
    tol = 2.0 ** -8 * (ref.abs() + sums) + sums
    assert ((out[:T].cpu().double() - ref).abs() <= tol).all()
    assert (out[T] == 3.0).all()
