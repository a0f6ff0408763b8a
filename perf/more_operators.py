"""The operators of a pass in 8-bit activations and of its answer, as cases that can be
timed and compared: rows brought to 8 bits with scales (with the residual's addition and
the rmsnorm before a projection, or as they are), the product of such rows and INT4
weights with its epilogue, and the log probabilities of given tokens with entropy and
top alternatives.

    own                   False: run() computes the plain form; True: the library's kernels
    listed()              the cases that stand for the range
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs, weights and buffers that a program has in hand
    run(state)            one pass through one operator, and its outputs
    work(case)            bytes and operations that a pass cannot do without
    exact(case, seed)     the outputs of the same inputs in 64 bits

Weights are INT4 group-128 as a checkpoint holds them (8 levels a word along the
inputs, zero points along the outputs, bf16 scales); hidden states are normal with a
spread between channels; logits are normal with a few likely tokens, and where a
grammar allows only some tokens the others are -inf.
"""
from __future__ import annotations

import math
import os
import sys
import weakref

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GROUP = 128
EPS = 1e-6
ACTS = ("none", "silu", "gelu", "gelu_tanh", "swiglu")
# hidden, qkv rows, attention width, intermediate and vocabulary of the benchmark's model
HIDDEN, QKV, ATTN, INTER, VOCAB = 5120, 7168, 4096, 17408, 248320
MAX_FLOPS = 2.0 * 4096 * HIDDEN * 2 * INTER
MAX_LOGITS = 1024 * VOCAB


def _hip():
    path = os.path.join(ROOT, "qwen38-3090-cuda-server_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import w4a16_hip

    return w4a16_hip


# ------------------------------------------------------------------- cases
def _norm(name, tokens, dim, residual):
    return {"name": name, "op": "norm", "tokens": tokens, "dim": dim, "residual": residual}


def _rows(name, tokens, dim, beside):
    return {"name": name, "op": "rows", "tokens": tokens, "dim": dim, "beside": beside}


def _linear(name, tokens, k, n, act, bias, residual, f32):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "act": act,
            "bias": bias, "residual": residual, "f32": f32}


def _logprobs(name, tokens, n, f32, asked, top_k, allowed, beside, pad):
    return {"name": name, "op": "logprobs", "tokens": tokens, "n": n, "f32": f32, "asked": asked,
            "top_k": top_k, "allowed": allowed, "beside": beside, "pad": pad}


def listed():
    return [
        # the norm before a projection of one decoded token: the smallest call, all latency
        _norm("norm_token", 1, HIDDEN, True),
        # the same for a full prompt chunk: bandwidth
        _norm("norm_prompt", 4096, HIDDEN, True),
        # a verify block's gated rows before the down projection
        _rows("rows_mid_verify", 9, INTER, 0),
        # attention rows of an odd prompt, columns of a wider buffer, before the output projection
        _rows("rows_attention_prompt", 2047, ATTN, QKV - ATTN),
        # the qkv projection of one token, with bias
        _linear("linear_qkv_token", 1, HIDDEN, QKV, "none", True, False, False),
        # the gate|up projection of a verify block (last token and eight drafts)
        _linear("linear_up_verify", 9, HIDDEN, 2 * INTER, "swiglu", False, False, False),
        # the down projection of a batch of decoding requests, added to the hidden states
        _linear("linear_down_batch", 77, INTER, HIDDEN, "none", False, True, False),
        # the output projection of an odd prompt, added to the hidden states
        _linear("linear_out_odd", 1001, ATTN, HIDDEN, "none", False, True, False),
        # the gate|up projection of a full prompt chunk
        _linear("linear_up_prompt", 4096, HIDDEN, 2 * INTER, "swiglu", False, False, False),
        # the head over a verify block, logits in 32 bits
        _linear("linear_head_verify", 9, HIDDEN, VOCAB, "none", False, False, True),
        # one decoded token with its alternatives
        _logprobs("logprobs_token", 1, VOCAB, True, 1, 20, 1.0, 0, 0),
        # a prompt's own tokens scored, logits in 16 bits, its last rows padding
        _logprobs("logprobs_prompt", 1000, VOCAB, False, 1, 5, 1.0, 0, 24),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    r = rng.random()
    tokens = _log_int(rng, 1, 4096)
    if r < 0.17:
        dim = GROUP * _log_int(rng, 4, 64)
        c = _norm("", tokens, dim, rng.random() < 0.7)
    elif r < 0.3:
        dim = GROUP * _log_int(rng, 4, 136)
        c = _rows("", tokens, dim, rng.choice((0, 8 * rng.randint(1, 400))))
    elif r < 0.7:
        k = rng.choice((HIDDEN, ATTN, INTER, GROUP * rng.randint(1, 70)))
        act = rng.choice(ACTS + ("swiglu", "none", "none"))
        n = 128 * rng.randint(2, 250) if act == "swiglu" else 64 * rng.randint(3, 300)
        tokens = rng.choice((1, rng.randint(2, 16), _log_int(rng, 17, 4096)))
        while 2.0 * tokens * k * n > MAX_FLOPS:
            tokens = tokens * 2 // 3
        f32 = act == "none" and rng.random() < 0.3
        c = _linear("", tokens, k, n, act, not f32 and rng.random() < 0.5, not f32 and rng.random() < 0.5, f32)
    else:
        n = rng.choice((VOCAB, _log_int(rng, 1000, VOCAB)))
        while tokens * n > MAX_LOGITS:
            tokens = tokens * 2 // 3
        c = _logprobs("", tokens, n, rng.random() < 0.5, rng.choice((0, 1, 1, rng.randint(2, 16))),
                      rng.choice((0, 1, 5, 20, rng.randint(1, 32))), rng.choice((1.0, 1.0, 0.5, 0.01)),
                      rng.choice((0, 0, rng.randint(1, 64))), rng.randint(0, tokens // 4))
    c.pop("name")
    return c


# ------------------------------------------------------------------ inputs
class State:
    """What the program keeps; the library's allocations go with it."""

    def __init__(self, case):
        self.case = case
        self._owned = []
        weakref.finalize(self, State._release, self._owned)

    @staticmethod
    def _release(owned):
        for free, handle in owned:
            free(handle)
        owned.clear()

    def keep(self, free, handle):
        self._owned.append((free, handle))
        return handle


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _hidden(g, rows, dim):
    """Hidden states: normal, with channels of different size."""
    spread = torch.exp(0.5 * torch.randn(dim, generator=g, device="cuda"))
    return (torch.randn(rows, dim, generator=g, device="cuda") * spread).to(torch.bfloat16)


def _int4(g, n, k):
    """packed [n][k/8] and zero points [n/8][k/128] as int32 words, scales bf16; the
    products of unit inputs come out near 1."""
    groups = k // GROUP
    i32 = dict(generator=g, device="cuda", dtype=torch.int32)
    packed = torch.randint(-(1 << 31), (1 << 31) - 1, (n, k // 8), **i32)
    zp = (torch.randint(0, (1 << 31) - 1, (n // 8, groups), **i32) & 0x77777777) + 0x44444444
    scale = (0.5 + torch.rand(n, groups, generator=g, device="cuda")) * (0.15 / math.sqrt(k))
    return packed, scale.to(torch.bfloat16), zp


def _codes(x):
    """Rows of 128-input groups in 8 bits: codes [T][k] int8 and scales [k/128][T] fp32."""
    t, k = x.shape
    v = x.float().view(t, k // GROUP, GROUP)
    top = v.abs().amax(2)
    q = torch.round(v * (127.0 / top.clamp(min=1e-30))[:, :, None]).clamp(-127, 127)
    return q.view(t, k).to(torch.int8), (top / 127.0).t().contiguous()


def _inputs(case, seed):
    """Everything a pass reads, made from the seed alone."""
    g, c = _gen(seed), case
    d, t = {}, case["tokens"]
    if c["op"] == "norm":
        d["h"] = _hidden(g, t, c["dim"])
        d["x"] = _hidden(g, t, c["dim"]) if c["residual"] else None
        d["w"] = (0.3 * torch.randn(c["dim"], generator=g, device="cuda")).to(torch.bfloat16)
    elif c["op"] == "rows":
        d["buffer"] = _hidden(g, t, c["dim"] + c["beside"])
        d["x"] = d["buffer"][:, :c["dim"]]
    elif c["op"] == "linear":
        d["q"], d["scale"] = _codes(_hidden(g, t, c["k"]))
        d["int4"] = _int4(g, c["n"], c["k"])
        d["bias"] = _hidden(g, 1, c["n"])[0] if c["bias"] else None
        width = c["n"] // 2 if c["act"] == "swiglu" else c["n"]
        d["residual"] = _hidden(g, t, width) if c["residual"] else None
    else:
        n = c["n"]
        x = 2.0 * torch.randn(t, n + c["beside"], generator=g, device="cuda")
        likely = torch.randint(0, n, (t, 8), generator=g, device="cuda")
        x.scatter_(1, likely, 6.0 + 5.0 * torch.rand(t, 8, generator=g, device="cuda"))
        if c["allowed"] < 1.0:
            x.masked_fill_(torch.rand(n + c["beside"], generator=g, device="cuda") >= c["allowed"], -math.inf)
        d["buffer"] = x if c["f32"] else x.to(torch.bfloat16)
        d["logits"] = d["buffer"][:, :n]
        # a row's first token is one of the likely ones; rows of padding ask for none (-1)
        asked = torch.randint(0, n, (t, c["asked"]), generator=g, device="cuda")
        if c["asked"]:
            asked[:, 0] = likely[:, 0]
            asked[t - c["pad"]:] = -1
        d["asked"] = asked.to(torch.int32)
    return d


def _order():
    """Place of each of 32 consecutive inputs in a chunk of 8-bit rows as the library holds
    them: inputs 8 w + {0, 4, 1, 5} at 4 w, inputs 8 w + {2, 6, 3, 7} at 16 + 4 w."""
    half = ((0, 4, 1, 5), (2, 6, 3, 7))
    return [8 * w + e for h in half for w in range(4) for e in h]


def prepare(case, seed):
    st = State(dict(case))
    c, d = st.case, _inputs(case, seed)
    st.d, t = d, c["tokens"]
    cuda = dict(device="cuda")
    if c["op"] in ("norm", "rows"):
        st.h = torch.zeros(t, c["dim"], dtype=torch.bfloat16, **cuda)
        st.values = torch.zeros(t, c["dim"], dtype=torch.bfloat16, **cuda)
        st.scale = torch.zeros(c["dim"] // GROUP, t, dtype=torch.float32, **cuda)
        st.q = torch.zeros(t, c["dim"], dtype=torch.int8, **cuda)
    elif c["op"] == "linear":
        width = c["n"] // 2 if c["act"] == "swiglu" else c["n"]
        st.out = torch.zeros(t, width, dtype=torch.float32 if c["f32"] else torch.bfloat16, **cuda)
    else:
        st.lp = torch.zeros(t, c["asked"], dtype=torch.float32, **cuda)
        st.entropy = torch.zeros(t, dtype=torch.float32, **cuda)
        st.ids = torch.zeros(t, c["top_k"], dtype=torch.int32, **cuda)
        st.top = torch.zeros(t, c["top_k"], dtype=torch.float32, **cuda)
    if not own:
        return st
    hip = _hip()
    if c["op"] in ("norm", "rows"):
        st.a8 = hip.a8_over(st.q, st.scale)
    elif c["op"] == "linear":
        at = torch.arange(c["k"], **cuda).view(-1, 32)[:, torch.tensor(_order(), **cuda)].reshape(-1)
        st.q = d["q"][:, at].contiguous()
        st.a8 = hip.a8_over(st.q, d["scale"])
        packed, scale, zp = d["int4"]
        n = packed.shape[0]
        st.w = st.keep(hip.awq_free, hip.awq_alloc_fused(n, c["k"]))
        hip.awq_repack_into(st.w, 0, packed, scale, zp, n)
        st.ws = st.keep(hip.gemm_workspace_free, hip.gemm_workspace_alloc(256 << 20))
        st.act = getattr(hip, "ACT_" + c["act"].upper())
    else:
        size = hip.logprobs_workspace(t, c["n"], c["top_k"])
        st.ws = st.keep(hip.gemm_workspace_free, hip.gemm_workspace_alloc(size))
    return st


# -------------------------------------------------------------- plain forms
def _levels(words, axis):
    """Eight 4-bit levels of each int32 word, lowest first, along `axis`."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    v = (words.unsqueeze(axis + 1) >> shifts.view((8,) + (1,) * (words.dim() - 1 - axis))) & 15
    return v.flatten(axis, axis + 1)


def _dequant(int4):
    """The weights as fp32: (q - zp) s."""
    packed, scale, zp = int4
    n, k = packed.shape[0], packed.shape[1] * 8
    q = _levels(packed, 1).float().view(n, k // GROUP, GROUP)
    z = _levels(zp, 0).float()
    return ((q - z[:, :, None]) * scale.float()[:, :, None]).view(n, k)


def _activate(v, act):
    if act == "none":
        return v
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v * math.sqrt(0.5))
    if act == "gelu_tanh":
        u = math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)
        return v / (1.0 + torch.exp(-2.0 * u))
    half = v.shape[1] // 2
    gate, up = v[:, :half], v[:, half:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _values(y):
    """What 8 bits and a scale a group hold of fp32 rows, and the scales. The quotient is
    formed in 64 bits: in 32, values next to a border between codes fall to either side."""
    t, k = y.shape
    v = y.double().view(t, k // GROUP, GROUP)
    top = v.abs().amax(2)
    q = torch.round(v * (127.0 / top)[:, :, None])
    scale = (top / 127.0).float()
    return (q.float() * scale[:, :, None]).view(t, k).to(torch.bfloat16), scale.t().contiguous()


def _plain_norm(st):
    c, d = st.case, st.d
    h = d["h"]
    if c["residual"]:
        h = (h.float() + d["x"].float()).to(torch.bfloat16)
    v = h.double()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * (1.0 + d["w"].double())
    return (h,) + _values(y)


def _plain_linear(st):
    c, d = st.case, st.d
    t, k = d["q"].shape
    x = (d["q"].float().view(t, k // GROUP, GROUP) * d["scale"].t()[:, :, None]).view(t, k)
    v = x @ _dequant(d["int4"]).t()
    if c["bias"]:
        v = v + d["bias"].float()
    v = _activate(v, c["act"])
    if c["residual"]:
        v = v + d["residual"].float()
    return v if c["f32"] else v.to(torch.bfloat16)


def _top(x, k):
    """Indices of the k largest of each row, the lower index among equals: one 64-bit key
    for each value, its bits in order above, its index reversed below."""
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    key = (bits << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
    return torch.topk(key, k, dim=1, sorted=True).indices


def _plain_logprobs(st):
    c, d = st.case, st.d
    x = d["logits"].float() + 0.0   # -0 counts as 0
    top = x.amax(1, keepdim=True)
    y = x - top
    e = torch.exp(y)
    total = e.sum(1, dtype=torch.float64)
    log = torch.log(total)
    y = torch.where(e > 0.0, y, torch.zeros_like(y))
    entropy = log - (e * y).sum(1, dtype=torch.float64) / total
    base = top.double() + log[:, None]
    ids = _top(x, c["top_k"])
    best = torch.gather(x, 1, ids)
    ids = torch.where(best > -math.inf, ids, -1).to(torch.int32)
    asked = d["asked"].long()
    lp = torch.gather(x, 1, asked.clamp(min=0)).double() - base
    lp = torch.where(asked >= 0, lp, torch.zeros_like(lp))
    return lp.float(), entropy.float(), ids, (best.double() - base).float()


def run(st):
    c, d = st.case, st.d
    t = c["tokens"]
    if not own:
        if c["op"] == "norm":
            return _plain_norm(st)
        if c["op"] == "rows":
            return _values(d["x"].float())
        return _plain_linear(st) if c["op"] == "linear" else _plain_logprobs(st)
    hip = _hip()
    if c["op"] == "norm":
        hip.rmsnorm_a8(st.a8, d["h"], d["w"], t, EPS, residual=d["x"], out=st.h if c["residual"] else None)
        hip.a8_dequant_rows(st.values, st.a8, 0, t)
        return (st.h if c["residual"] else d["h"]), st.values, st.scale
    if c["op"] == "rows":
        hip.quantize_a8(st.a8, d["x"], t)
        hip.a8_dequant_rows(st.values, st.a8, 0, t)
        return st.values, st.scale
    if c["op"] == "linear":
        if c["f32"]:
            hip.linear_w4a8_f32(st.out, st.w, st.a8, t, st.ws)
        else:
            hip.linear_w4a8(st.out, st.w, st.a8, t, st.ws, bias=d["bias"], act=st.act, residual=d["residual"])
        return st.out
    hip.logprobs(st.lp, d["logits"], d["asked"], t, c["n"], st.ws, entropy=st.entropy, top_ids=st.ids,
                 top_logprobs=st.top, top_k=c["top_k"])
    return st.lp, st.entropy, st.ids, st.top


# -------------------------------------------------------------- exact values
def _exact_rows8(y):
    groups = y.reshape(y.shape[0], -1, GROUP)
    step = groups.abs().max(dim=2, keepdim=True).values / 127.0
    return (torch.round(groups / step) * step).reshape(y.shape), step[:, :, 0].T


def _exact_activation(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.sigmoid(math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3))
    if act == "swiglu":
        gate, up = v.chunk(2, dim=1)
        return gate * torch.sigmoid(gate) * up
    return v


def _exact_product(x, int4, r0, r1):
    packed, scale, zp = int4
    n, groups = r1 - r0, packed.shape[1] * 8 // GROUP
    words = packed[r0:r1].to(torch.int64) & 0xFFFFFFFF
    q = torch.stack([(words // 16 ** i) % 16 for i in range(8)], -1).reshape(n, groups, GROUP)
    zw = zp[r0 // 8:r1 // 8].to(torch.int64) & 0xFFFFFFFF
    z = torch.stack([(zw // 16 ** i) % 16 for i in range(8)], 1).reshape(n, groups, 1)
    w = ((q - z).double() * scale[r0:r1].double().reshape(n, groups, 1)).reshape(n, -1)
    return torch.matmul(x, w.t().contiguous())


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "norm":
        h = d["h"].double()
        if c["residual"]:
            h = (h + d["x"].double()).to(torch.bfloat16).double()
        rms = torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / c["dim"] + EPS)
        return (h,) + _exact_rows8((1.0 + d["w"].double()) * h / rms)
    if c["op"] == "rows":
        return _exact_rows8(d["x"].double())
    if c["op"] == "linear":
        x = d["q"].double() * torch.repeat_interleave(d["scale"].double().T, GROUP, dim=1)
        part = 32768
        v = torch.cat([_exact_product(x, d["int4"], r, min(r + part, c["n"])) for r in range(0, c["n"], part)], 1)
        if c["bias"]:
            v += d["bias"].double()
        v = _exact_activation(v, c["act"])
        return v + d["residual"].double() if c["residual"] else v
    x = d["logits"].double()
    lps, entropies, ids, tops = [], [], [], []
    step = max(1, (1 << 25) // c["n"])
    for i in range(0, c["tokens"], step):
        lp = torch.log_softmax(x[i:i + step], 1)
        asked = d["asked"][i:i + step].long()
        some = asked >= 0
        lps.append(torch.where(some, torch.gather(lp, 1, torch.where(some, asked, 0)), 0.0))
        entropies.append(torch.special.entr(torch.exp(lp)).sum(1))
        order = torch.argsort(lp, dim=1, descending=True, stable=True)[:, :c["top_k"]]
        best = torch.gather(lp, 1, order)
        ids.append(torch.where(best > -math.inf, order, -1).to(torch.int32))
        tops.append(best)
    return torch.cat(lps), torch.cat(entropies), torch.cat(ids), torch.cat(tops)


# --------------------------------------------------------------------- work
def work(case):
    c, t = case, case["tokens"]
    if c["op"] in ("norm", "rows"):
        # rows (and the residual's both ways) and the weight; values in 16 bits, scales
        size = 2 if c["op"] == "rows" else 6 if c["residual"] else 2
        return {"bytes": t * c["dim"] * (size + 2) + 4 * t * c["dim"] // GROUP
                + (2 * c["dim"] if c["op"] == "norm" else 0), "flops": 10 * t * c["dim"]}
    if c["op"] == "linear":
        k, n = c["k"], c["n"]
        width = n // 2 if c["act"] == "swiglu" else n
        extra = (2 * n if c["bias"] else 0) + (2 * t * width if c["residual"] else 0)
        return {"bytes": int(n * k * (0.5 + 2.5 / GROUP) + t * k * (1 + 4 / GROUP)
                             + t * width * (4 if c["f32"] else 2) + extra), "flops": 2 * t * n * k}
    return {"bytes": t * c["n"] * (4 if c["f32"] else 2) + 8 * t * (c["asked"] + c["top_k"]) + 4 * t,
            "flops": 8 * t * c["n"]}
