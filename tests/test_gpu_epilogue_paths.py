"""qw4_linear_epilogue's decode and verify kernels at the sizes of real projections, with a
scratch: gated and ungated units of 16, 32 and 64 rows, more than eight output units a
workgroup, two row blocks, rows staged whole, group-major items, K beyond a workgroup's
registers. Bias and residual, also in y; a sample of columns against 64 bits."""
import pytest
import torch

from test_gpu_linear_epilogue import activation, bf, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    import w4a16_hip

    w4a16_hip.lib()
    yield w4a16_hip
    torch.cuda.empty_cache()


class Weights:
    """Random levels, zero points and scales [N][K], on the GPU."""

    def __init__(self, hip, N, K):
        g = torch.Generator(device="cuda").manual_seed(N + K)
        i32 = dict(generator=g, device="cuda", dtype=torch.int32)
        self.packed = torch.randint(-(1 << 31), (1 << 31) - 1, (N, K // 8), **i32)
        self.zp = torch.randint(-(1 << 31), (1 << 31) - 1, (N // 8, K // 128), **i32)
        self.scale = ((1 + torch.rand(N, K // 128, generator=g, device="cuda")) * 2.0 ** -6).bfloat16()
        self.w = hip.awq_alloc_fused(N, K)
        hip.awq_repack_into(self.w, 0, self.packed, self.scale, self.zp, N)

    def rows(self, n):
        """(q - z) and s of rows n (a tensor), in 64 bits: [n][K / 128][128], [n][K / 128]."""
        shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
        q = ((self.packed[n][:, :, None] >> shift) & 15).double().view(len(n), -1, 128)
        z = ((self.zp[n // 8] >> (4 * (n % 8)).int()[:, None]) & 15).double()
        return q - z[:, :, None], self.scale[n].double()


def check_columns(y, x, W, cols, up, bias, act, residual):
    """y's columns `cols` against the formula. The sums of a group are those of (128 + q) x
    less (128 + z) x, each off by 128 additions of random rounding, 2^-24 of a partial sum
    of at most 143 |x| a term: 6 sigma over sqrt(3), twice, is 80 x 2^-24 of them; the
    groups' are independent. The sum of the groups, activation and rounding: see check() of
    test_gpu_linear_epilogue."""
    xf = x.double().cuda()
    T, K = xf.shape
    xa = xf.abs().view(T, -1, 128).sum(2)   # [T][G]

    def product(n):
        d, s = W.rows(n)
        w = (d * s[:, :, None]).view(len(n), K)
        v = xf @ w.t().contiguous()
        ev = 2.0 ** -24 * ((K ** 0.5 + 8) * (xf.abs() @ w.abs().t().contiguous()) +
                           80 * 143 * (xa ** 2 @ (s ** 2).t().contiguous()).sqrt())
        if bias is not None:
            v = v + bias[n.cpu()].double().cuda()
            ev = ev + 2.0 ** -24 * v.abs()
        return v, ev

    if act == "swiglu":
        (g, eg), (u, eu) = product(cols), product(cols + up)
        f = activation(torch.cat([g, u], 1), act)
        ef = 1.13 * eg * (u.abs() + eu) + (g * torch.sigmoid(g)).abs() * eu + 2.0 ** -20 * f.abs()
    else:
        v, ev = product(cols)
        f = activation(v, act)
        ef = 1.13 * ev + 2.0 ** -20 * f.abs()
    ref = f if residual is None else f + residual[:, cols.cpu()].double().cuda()
    tol = 2.0 ** -8 * (ref.abs() + ef) + ef + 2.0 ** -23 * ref.abs() + 1e-30
    err = (y[:, cols.cpu()].double().cuda() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


# weight rows, K, rows of x
SHAPES = [(9472, 640, (1, 2, 9, 16, 17, 32)), (34816, 5120, (1, 2, 9, 16, 17, 32)), (5120, 17408, (1, 2, 9, 16)),
          (24576, 8448, (1, 9, 16)), (65536, 128, (1, 3)), (131072, 256, (1, 2)), (524288, 128, (1, 2)), (1024, 65536, (1, 2, 9)), (256, 131072, (1, 16)), (20480, 2048, (1, 5, 24))]


@pytest.mark.parametrize("act", ["swiglu", "gelu", "none"])
@pytest.mark.parametrize("N,K,rows", SHAPES)
def test_paths(hip, N, K, rows, act):
    W = Weights(hip, N, K)
    scratch = hip.gemv_scratch_alloc(K, N, 128, 16)
    width = N // 2 if act == "swiglu" else N
    g = torch.Generator().manual_seed(N)
    cols = torch.randperm(width, generator=g)[:1200]
    edges = torch.arange(0, width, width // 16)
    edges = torch.cat([edges, (edges + 63).clamp(max=width - 1), torch.tensor([width - 64, width - 1])])
    cols = torch.unique(torch.cat([cols, edges])).cuda()
    for T in rows:
        assert T <= hip.linear_max_t(W.w)
        x = bf(torch.randn(T, K, generator=g) * (8.0 / K ** 0.5))
        for bias, residual, alias in ((False, False, False), (True, True, False), (True, True, True)):
            print(f"path {N}x{K} T={T} {act} bias={bias} residual={residual} alias={alias}", flush=True)
            b = bf(torch.randn(N, generator=g)) if bias else None
            r = bf(torch.randn(T, width, generator=g)) if residual else None
            y = run(hip, W.w, x, T, scratch, None, b, act, r, alias)
            check_columns(y, x, W, cols, width, b, act, r)
    hip.awq_free(W.w)
    hip.gemv_scratch_free(scratch)
