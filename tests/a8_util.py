"""Plain forms of the 8-bit rows and their products, in 64 bits, for the tests."""
from __future__ import annotations

import math

import torch

GROUP = 128
# place p of 32 consecutive inputs in a chunk of 8-bit rows holds input ORDER[p]
ORDER = [8 * w + e for half in ((0, 4, 1, 5), (2, 6, 3, 7)) for w in range(4) for e in half]


def to_layout(q):
    """Codes [T][k] in the library's order."""
    return q.view(q.shape[0], -1, 32)[:, :, ORDER].reshape(q.shape).contiguous()


def from_layout(q):
    inverse = [ORDER.index(i) for i in range(32)]
    return q.view(q.shape[0], -1, 32)[:, :, inverse].reshape(q.shape).contiguous()


def random_weights(hip, n, k, seed, scale=None):
    """Repacked weights, and (q - zp) [n][k] and the scales [n][k/128] in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    groups = k // GROUP
    q = torch.randint(0, 16, (n, k), generator=g)
    z = torch.randint(0, 16, (n, groups), generator=g)
    s = (0.5 + torch.rand(n, groups, generator=g)) * 0.15 / math.sqrt(k) if scale is None else \
        torch.full((n, groups), float(scale))
    s = s.to(torch.bfloat16)
    shifts = 4 * torch.arange(8)
    packed = (q.view(n, k // 8, 8) << shifts).sum(-1)
    zp = (z.view(n // 8, 8, groups) << shifts.view(1, 8, 1)).sum(1)
    i32 = lambda v: torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32).cuda()  # noqa: E731
    w = hip.awq_repack(i32(packed), s.cuda(), i32(zp), n, k)
    torch.cuda.synchronize()
    less = (q.view(n, groups, GROUP) - z[:, :, None]).double().view(n, k)
    return w, less.cuda(), s.double().cuda()


def random_rows(t, k, seed, unit=False):
    """Codes [t][k] int8 and scales [k/128][t] fp32 (1 with `unit`), on the GPU."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (t, k), generator=g).to(torch.int8)
    scale = torch.ones(k // GROUP, t) if unit else 0.001 + 0.02 * torch.rand(k // GROUP, t, generator=g)
    return q.cuda(), scale.cuda()


def product(q, scale, less, ws):
    """sum_g sx sw (less q) in 64 bits, and the sum of the terms' magnitudes."""
    t, k = q.shape
    v = torch.zeros(t, less.shape[0], dtype=torch.float64, device="cuda")
    size = torch.zeros_like(v)
    for g in range(k // GROUP):
        at = slice(g * GROUP, (g + 1) * GROUP)
        part = torch.matmul(q[:, at].double(), less[:, at].t().contiguous())
        part = part * scale[g].double()[:, None] * ws[:, g]
        v += part
        size += part.abs()
    return v, size


def sum_tolerance(size, groups):
    """Of a product's fp32 sums: one rounding a group for the scaled integer, one for the
    sum, a few at the end, each 2^-24 of at most `size`; scales to 22 bits."""
    return (2 * groups + 8) * 2.0 ** -24 * size + 2.0 ** -22 * size
