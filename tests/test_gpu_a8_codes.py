"""Codes of 8-bit rows where a value lies in the middle of two, and next to it."""
import pytest
import torch

from a8_util import from_layout

pytestmark = pytest.mark.gpu
GROUP = 128


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    return w4a16_hip


def _rows(hip, rows, dim):
    q = torch.full((rows, dim), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((dim // GROUP, rows), -3.0, device="cuda")
    return hip.a8_over(q, scale), q, scale


def _nearest(num, den):
    """num / den (den > 0) to the nearest integer, the even one of two as near."""
    low = torch.div(num, den, rounding_mode="floor")
    twice = 2 * (num - low * den)
    return low + ((twice > den) | ((twice == den) & (low % 2 != 0))).long()


@pytest.mark.parametrize("exponent", [-90, 0, 100])
def test_every_pair_of_mantissas(hip, exponent):
    """Each of bf16's 128 mantissas as a group's largest A, against every value V 2^-e up to
    it, of both signs: the code is 127 V / A in integers, rounded half to even. Values 2^-10
    of A and below have code 0."""
    top = torch.arange(128, 256)
    value = torch.arange(128, 256)
    row = []   # of each A: (V, e), its own first in every group
    for e in range(10):
        for sign in (1, -1):
            row.append(torch.stack([sign * value, torch.full_like(value, e)], 1))
    pairs = torch.cat(row)                                     # [2560][2]
    pairs = torch.cat([pairs, torch.zeros(-len(pairs) % (GROUP - 1), 2, dtype=torch.int64)])
    pairs = pairs.view(1, -1, GROUP - 1, 2).expand(128, -1, -1, -1)
    own = torch.stack([top, torch.zeros_like(top)], 1).view(128, 1, 1, 2).expand(-1, pairs.shape[1], 1, -1)
    v, e = torch.cat([own, pairs], 2).unbind(-1)               # [128][groups][128]
    v = torch.where((e == 0) & (v.abs() > top.view(128, 1, 1)), torch.zeros_like(v), v)
    want = _nearest(127 * v, top.view(128, 1, 1) << e)
    x = torch.ldexp(v.double(), (exponent - e).double()).view(128, -1).to(torch.bfloat16).cuda()
    a, q, _ = _rows(hip, 128, x.shape[1])
    hip.quantize_a8(a, x, 128)
    torch.cuda.synchronize()
    got = from_layout(q).cpu().long().view_as(want)
    assert torch.equal(got, want), f"{int((got != want).sum())} codes differ"


@pytest.mark.parametrize("T", [3, 600])
def test_half_of_a_norms_largest(hip, T):
    """A normed value that is exactly half its group's largest, 63.5: code 64, whatever the
    row's norm and the group's weight."""
    dim = 512
    g = torch.Generator().manual_seed(T)
    top = (1 + torch.rand(T, dim // GROUP, generator=g)).to(torch.bfloat16).float()
    h = top[:, :, None] * torch.where(torch.arange(GROUP) % 2 == 0, 0.5, -0.5)
    h[:, :, 7] = top
    h = h.view(T, dim).to(torch.bfloat16).cuda()
    w = (0.1 * torch.randn(dim // GROUP, generator=g)).to(torch.bfloat16).repeat_interleave(GROUP).cuda()
    a, q, _ = _rows(hip, T, dim)
    hip.rmsnorm_a8(a, h, w, T, 1e-6)
    torch.cuda.synchronize()
    want = torch.where(torch.arange(GROUP) % 2 == 0, 64, -64)
    want[7] = 127
    assert torch.equal(from_layout(q).cpu().long().view(T, -1, GROUP), want.expand(T, dim // GROUP, GROUP))
