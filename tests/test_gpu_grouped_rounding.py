"""To how many bits qw4_gemm_grouped may round weights, by sizes and workspace: up to the
rows an expert where qw4_linear uses a weight of that size exactly, not at all without a
workspace and to 11 bits with one, whichever kernel is the faster; beyond, as qw4_gemm.

Rows of x are x[k1] = 1, x[k2] = -1 within a group of 128, so a product is (q1 - q2) s, at
most 12 bits, exact in fp32: its bf16 is the nearest one where the weights were used
exactly, and off by both weights' roundings, half a step each, where they were not."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import torch

    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    yield w4a16_hip
    torch.cuda.empty_cache()


class Weights:
    """Random levels and zero points [rows][K], scales of a power of two times 1 .. 2."""

    def __init__(self, hip, rows, K):
        import torch

        g = torch.Generator(device="cuda").manual_seed(rows + K)
        i32 = dict(generator=g, device="cuda", dtype=torch.int32)
        self.packed = torch.randint(-(1 << 31), (1 << 31) - 1, (rows, K // 8), **i32)
        self.zp = torch.randint(-(1 << 31), (1 << 31) - 1, (rows // 8, K // 128), **i32)
        self.scale = ((1 + torch.rand(rows, K // 128, generator=g, device="cuda")) * 2.0 ** -6).bfloat16()
        self.w = hip.awq_alloc_fused(rows, K)
        hip.awq_repack_into(self.w, 0, self.packed, self.scale, self.zp, rows)

    def column(self, r0, r1, k):
        """(q - z) s of rows [r0, r1) at input k, in 64 bits."""
        q = (self.packed[r0:r1, k // 8] >> (4 * (k % 8))) & 15
        import torch

        r = torch.arange(r0, r1, device="cuda")
        z = (self.zp[r // 8, k // 128] >> (4 * (r % 8)).int()) & 15
        return (q - z).double() * self.scale[r0:r1, k // 128].double()


# experts, weight rows an expert, K, rows an expert in the mean (below the line "down" and
# "many" are faster in tiles)
CASES = {"down": (32, 5120, 2176, 125), "down, tens": (32, 5120, 2176, 25), "square": (8, 4096, 4096, 60),
         "many": (64, 2048, 1024, 64), "few": (8, 512, 640, 9), "prompt": (4, 2048, 1024, 600),
         "long K": (2, 256, 8448, 20)}


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_rounding(hip, case, gated):
    import torch

    E, n, K, mean = CASES[case]
    R = E * mean
    W = Weights(hip, E * n, K)
    # the line is qw4_linear's for one expert's weight
    one = hip.W4A16Weights(0x1000, 0x2000, 0x3000, n, K, 128, K // 128)
    few = mean <= hip.linear_max_t(one)
    assert few == (case != "prompt")
    g = torch.Generator().manual_seed(R)
    cut = torch.sort(torch.randint(0, R + 1, (E - 1,), generator=g)).values
    if case != "few":   # ragged, but none so short that the mean says little
        cut = (cut + 3 * torch.arange(1, E) * mean) // 4
    offsets = torch.cat([torch.zeros(1, dtype=cut.dtype), cut, torch.tensor([R])])
    k1, k2 = torch.randint(0, K // 128, (R,), generator=g) * 128, 0
    k1, k2 = k1 + torch.randint(0, 64, (R,), generator=g), k1 + 64 + torch.randint(0, 64, (R,), generator=g)
    size = 16.0   # an exact factor; gated sums near 1
    x = torch.zeros(R, K, dtype=torch.bfloat16)
    x[torch.arange(R), k1], x[torch.arange(R), k2] = size, -size
    perm = torch.randperm(R, generator=g)
    act = hip.ACT_SWIGLU if gated else hip.ACT_NONE
    width = n // 2 if gated else n
    ws = hip.gemm_workspace_alloc(hip.epilogue_workspace(W.w, R))
    off = offsets.to(torch.int32).cuda()
    for gather in (False, True):
        xs = x if not gather else torch.empty_like(x).index_copy_(0, perm, x)   # row perm[i] is position i's
        dx, tokens = xs.cuda(), perm.to(torch.int32).cuda()
        plan = hip.expert_plan_over(off, tokens, tokens)
        for space in (None, ws):
            print(f"rounding {case} gated={gated} gather={gather} ws={space is not None}", flush=True)
            y = torch.full((R, width), 7.0, dtype=torch.bfloat16, device="cuda")
            hip.gemm_grouped_w4a16(y, W.w, dx, plan, R, gather, act=act, ws=space)
            torch.cuda.synchronize()
            # bits of the weights: None exact
            if few and K <= 8192:
                bits = 11 if space is not None else None
            else:
                bits = 11 if space is not None and (gated or few) else 8
            told = 0   # outputs that weights rounded to 8 bits would put outside the bound
            for e in range(E):
                lo, hi = int(offsets[e]), int(offsets[e + 1])
                for i in sorted({lo, (lo + hi) // 2, hi - 1} if hi > lo else ()):
                    a, b = (size * W.column(e * n, (e + 1) * n, int(k)) for k in (k1[i], k2[i]))
                    got = y[i].double()

                    def value(r):
                        v = r(a) - r(b)
                        if not gated:
                            return v
                        gate, up = v.chunk(2)
                        return gate * torch.sigmoid(gate) * up

                    ref = value(lambda t: t)
                    # each weight off by half a step: 2^-bits of it
                    ev = torch.zeros_like(a) if bits is None else 2.0 ** -bits * (a.abs() + b.abs())
                    if gated:
                        (vg, vu), (eg, eu) = (a - b).chunk(2), ev.chunk(2)
                        # |silu'| <= 1.1; exp, 1/x and three products in fp32: 2^-20
                        ev = 1.1 * eg * (vu.abs() + eu) + (vg * torch.sigmoid(vg)).abs() * eu + 2.0 ** -20 * ref.abs()
                    tol = 2.0 ** -8 * (ref.abs() + ev) + ev + 1e-30
                    assert ((got - ref).abs() <= tol).all(), (e, i, float(((got - ref).abs() / tol).max()))
                    if bits is None and not gated:   # the nearest bf16 itself
                        assert torch.equal(y[i], ref.float().bfloat16())
                    eight = value(lambda t: t.float().bfloat16().double()).float().bfloat16().double()
                    told += int(((eight - ref).abs() > tol).sum())
                    if bits == 8 and not gated:
                        assert torch.equal(got, eight)
            assert bits == 8 or told > 0
    hip.gemm_workspace_free(ws)
    hip.awq_free(W.w)
