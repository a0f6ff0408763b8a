"""The Python binding's checks around 8-bit rows and log probabilities: each refusal by what it
says, beside the call that is taken."""
import pytest
import torch

GPU = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import w4a16_hip

    w4a16_hip.lib()
    return w4a16_hip


def _over(hip, device):
    """a8_over's refusals that do not depend on where the tensors are."""
    q, s = torch.zeros(8, 256, dtype=torch.int8, device=device), torch.zeros(2, 8, device=device)
    with pytest.raises(ValueError, match="a8_over q: type torch.float32, needs torch.int8"):
        hip.a8_over(q.float(), s)
    with pytest.raises(ValueError, match="a8_over q: not contiguous"):
        hip.a8_over(torch.zeros(8, 512, dtype=torch.int8, device=device)[:, ::2], s)
    with pytest.raises(ValueError, match=r"a8_over q: shape \(8, 200\)"):
        hip.a8_over(torch.zeros(8, 200, dtype=torch.int8, device=device), s)
    with pytest.raises(ValueError, match=r"a8_over q: shape \(2, 8, 128\)"):
        hip.a8_over(torch.zeros(2, 8, 128, dtype=torch.int8, device=device), s)
    # scales of other rows than q has: a group's would be taken from another place
    for rows in (7, 9, 32):
        with pytest.raises(ValueError, match=r"a8_over scale: shape .*needs \(2, 8\)"):
            hip.a8_over(q, torch.zeros(2, rows, device=device))
    for shape in ((1, 8), (3, 8), (8, 2), (16,)):
        with pytest.raises(ValueError, match=r"a8_over scale: shape .*needs \(2, 8\)"):
            hip.a8_over(q, torch.zeros(shape, device=device))
    return q, s


def test_rows_over_tensors(hip):
    q, s = _over(hip, "cpu")
    with pytest.raises(ValueError, match="a8_over q: not on the call's GPU"):
        hip.a8_over(q, s)


def test_sizes_and_types(hip):
    a = hip.A8Rows(0x1000, 0x2000, 32, 512)
    w = hip.W4A16Weights()
    w.qweight, w.scale, w.zeros, w.out_f, w.in_f, w.group_size, w.num_groups = 0x1000, 0x2000, 0x3000, 256, 512, 128, 4
    x = torch.zeros(4, 512, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="quantize_a8 x: buffer holds 4096 bytes, needs 5120"):
        hip.quantize_a8(a, x, 5, stream=0)
    with pytest.raises(ValueError, match="quantize_a8 x: type torch.float16"):
        hip.quantize_a8(a, x.half(), 4, stream=0)
    with pytest.raises(ValueError, match="quantize_a8 x: needs 4 rows of 512"):
        hip.quantize_a8(a, torch.zeros(4, 600, dtype=torch.bfloat16)[:, :500], 4, stream=0)
    with pytest.raises(ValueError, match="quantize_a8 x: needs 4 rows of 512"):
        hip.quantize_a8(a, torch.zeros(512, 4, dtype=torch.bfloat16).t(), 4, stream=0)
    with pytest.raises(ValueError, match="rmsnorm_a8 h: buffer holds 4096 bytes, needs 5120"):
        hip.rmsnorm_a8(a, x, x[0], 5, 1e-6, stream=0)
    with pytest.raises(ValueError, match="rmsnorm_a8 out: type torch.float32"):
        hip.rmsnorm_a8(a, x, x[0], 4, 1e-6, out=x.float(), stream=0)
    with pytest.raises(ValueError, match="a8_dequant_rows dst: buffer holds 4096 bytes, needs 5120"):
        hip.a8_dequant_rows(x, a, 0, 5, stream=0)
    with pytest.raises(ValueError, match="linear_w4a8 y: type torch.float32, needs torch.bfloat16"):
        hip.linear_w4a8(torch.zeros(4, 256), w, a, 4, stream=0)
    with pytest.raises(ValueError, match="linear_w4a8_f32 y: buffer holds 2048 bytes, needs 4096"):
        hip.linear_w4a8_f32(torch.zeros(2, 256), w, a, 4, stream=0)
    with pytest.raises(ValueError, match="logprobs logits: needs 4 rows of 100"):
        hip.logprobs(torch.zeros(4), torch.zeros(4, 99), torch.zeros(4, dtype=torch.int32), 4, 100, stream=0)
    for targets in (0x3000, torch.zeros(4, 1, 1, dtype=torch.int32), torch.zeros((), dtype=torch.int32)):
        with pytest.raises(ValueError, match="targets of neither"):
            hip.logprobs(torch.zeros(4), torch.zeros(4, 100), targets, 4, 100, stream=0)


@GPU
def test_rows_over_tensors_on_the_gpu(hip):
    q, s = _over(hip, "cuda")
    with pytest.raises(ValueError, match="a8_over scale: type torch.float64"):
        hip.a8_over(q, s.double())
    with pytest.raises(ValueError, match="a8_over scale: not on the call's GPU"):
        hip.a8_over(q, s.cpu())
    a = hip.a8_over(q, s)
    assert (a.q, a.scale, a.max_rows, a.in_f) == (q.data_ptr(), s.data_ptr(), 8, 256)
    x = torch.ones(8, 256, dtype=torch.bfloat16, device="cuda")
    hip.quantize_a8(a, x, 8)
    torch.cuda.synchronize()
    assert torch.all(q == 127) and torch.all(s == torch.tensor(1.0) / 127)
    s.zero_()
    a = hip.a8_over(q[:3], torch.zeros(2, 3, device="cuda"))   # some of the rows, their own scales
    assert (a.max_rows, a.in_f) == (3, 256)


@GPU
def test_rows_and_products_on_the_gpu(hip):
    bf16 = dict(dtype=torch.bfloat16, device="cuda")
    q, s = torch.zeros(8, 512, dtype=torch.int8, device="cuda"), torch.zeros(4, 8, device="cuda")
    a, x, wide = hip.a8_over(q, s), torch.ones(8, 512, **bf16), torch.ones(8, 600, **bf16)
    hip.quantize_a8(a, x, 8)
    hip.quantize_a8(a, wide[:, :512], 8)
    hip.quantize_a8(a, x.view(torch.int16), 8)   # the same bits
    with pytest.raises(ValueError, match="quantize_a8 x: needs 8 rows"):
        hip.quantize_a8(a, wide[:7, :512], 8)
    with pytest.raises(ValueError, match="quantize_a8 x: not on the call's GPU"):
        hip.quantize_a8(a, x.cpu(), 8)
    hip.rmsnorm_a8(a, x, x[0], 8, 1e-6, residual=x, out=x)
    for name in ("residual", "out"):
        with pytest.raises(ValueError, match=f"rmsnorm_a8 {name}: buffer holds"):
            hip.rmsnorm_a8(a, x, x[0], 8, 1e-6, **{"residual": x, "out": x, name: x[:7]})
    with pytest.raises(ValueError, match="rmsnorm_a8 w: buffer holds"):
        hip.rmsnorm_a8(a, x, x[0, :504].contiguous(), 8, 1e-6)
    words = torch.zeros(128, 64, dtype=torch.int32, device="cuda")
    w = hip.awq_repack(words, torch.ones(128, 4, **bf16), torch.zeros(16, 4, dtype=torch.int32, device="cuda"), 128, 512)
    y, f = torch.zeros(8, 128, **bf16), torch.zeros(8, 128, device="cuda")
    bias = torch.zeros(128, **bf16)
    hip.linear_w4a8(y, w, a, 8, bias=bias, residual=y)
    hip.linear_w4a8(y[:, :64].contiguous(), w, a, 8, act=hip.ACT_SWIGLU)
    hip.linear_w4a8_f32(f, w, a, 8)
    with pytest.raises(ValueError, match="linear_w4a8 y: buffer holds"):
        hip.linear_w4a8(y[:7], w, a, 8)
    with pytest.raises(ValueError, match="linear_w4a8 y: not contiguous"):
        hip.linear_w4a8(torch.zeros(8, 256, **bf16)[:, :128], w, a, 8)
    with pytest.raises(ValueError, match="linear_w4a8 bias: buffer holds"):
        hip.linear_w4a8(y, w, a, 8, bias=bias[:64])
    with pytest.raises(ValueError, match="linear_w4a8 residual: type torch.float32"):
        hip.linear_w4a8(y, w, a, 8, residual=f)
    with pytest.raises(ValueError, match="linear_w4a8_f32 y: type torch.bfloat16"):
        hip.linear_w4a8_f32(y, w, a, 8)
    with pytest.raises(ValueError, match="linear_w4a8_f32 y: buffer holds"):
        hip.linear_w4a8_f32(f[:7], w, a, 8)
    torch.cuda.synchronize()
    hip.awq_free(w)


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_log_probabilities_on_the_gpu(hip, dtype):
    T, n, k = 8, 100, 5
    f32, i32 = dict(device="cuda"), dict(dtype=torch.int32, device="cuda")
    x, lp, e = torch.zeros(T, n, dtype=dtype, **f32), torch.zeros(T, 2, **f32), torch.zeros(T, **f32)
    ids, top, asked = torch.zeros(T, k, **i32), torch.zeros(T, k, **f32), torch.zeros(T, 2, **i32)

    def call(lp=lp, x=x, asked=asked, e=e, ids=ids, top=top):
        hip.logprobs(lp, x, asked, T, n, entropy=e, top_ids=ids, top_logprobs=top, top_k=k)

    call()
    call(lp=lp[:, 0].contiguous(), asked=asked[:, 0].contiguous())
    call(lp=None, asked=None)
    call(e=None)
    call(x=torch.zeros(T, n + 8, dtype=dtype, **f32)[:, 3:n + 3])
    for bad in (dict(lp=lp[:, 0].contiguous()), dict(e=e[:7]), dict(ids=ids[:7]), dict(top=top[:, :4].contiguous()),
                dict(asked=asked[:7])):
        with pytest.raises(ValueError, match="logprobs .*: buffer holds"):
            call(**bad)
    for bad in (dict(asked=asked.long()), dict(ids=ids.long()), dict(lp=lp.double()), dict(e=e.bfloat16()),
                dict(x=x.double())):
        with pytest.raises(ValueError, match="logprobs .*: type "):
            call(**bad)
    for name, t in (("lp", lp), ("x", x), ("asked", asked), ("e", e), ("ids", ids), ("top", top)):
        with pytest.raises(ValueError, match="logprobs .*: not on the call's GPU"):
            call(**{name: t.cpu()})
    torch.cuda.synchronize()
    assert torch.all((lp + torch.tensor(100.0).log().cuda()).abs() < 1e-5)
