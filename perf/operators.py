"""The operators of a layer of experts and of a dense projection with its
epilogue, as cases that can be timed and compared: the router with its plan, the
W4A16 products grouped by expert, the weighted sum of a token's expert rows, and
the W4A16 product with bias, activation and residual.

    own                   False: run() computes the plain form; True: the library's kernels
    listed()              the cases that stand for the range
    draw(rng)             one more case of the same ranges
    prepare(case, seed)   inputs, weights and buffers that a program has in hand
    run(state)            one pass through one operator, and its outputs
    work(case)            bytes and operations that a pass cannot do without
    exact(case, seed)     the outputs of the same inputs in 64 bits

Weights are INT4 group-128 as a checkpoint holds them (8 levels a word along the
inputs, zero points along the outputs, bf16 scales); activations are normal with
a spread between channels, as hidden states have it; router logits have popular
and unpopular experts.
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
ACTS = ("none", "silu", "gelu", "gelu_tanh", "swiglu")
# (hidden, qkv rows, attention width, intermediate) of the benchmark's layer and of
# its 8-way shard
HIDDEN, QKV, ATTN, INTER = 5120, 7168, 4096, 17408
SHARD_INTER = 2176
MAX_FLOPS = 2.0 * 4096 * 8 * 2048 * 2048   # of the largest grouped case
MAX_FLOPS_DENSE = 2.0 * 4096 * HIDDEN * INTER


def _hip():
    path = os.path.join(ROOT, "qwen38-3090-cuda-server_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import w4a16_hip

    return w4a16_hip


# ------------------------------------------------------------------- cases
def _route(name, tokens, experts, top_k, f32, renorm, pad):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k,
            "f32": f32, "renorm": renorm, "pad": pad}


def _grouped(name, tokens, experts, top_k, k, n, gather, act, bias, pad):
    return {"name": name, "op": "grouped", "tokens": tokens, "experts": experts, "top_k": top_k,
            "k": k, "n": n, "gather": gather, "act": act, "bias": bias, "pad": pad}


def _combine(name, tokens, experts, top_k, dim, residual, pad):
    return {"name": name, "op": "combine", "tokens": tokens, "experts": experts, "top_k": top_k,
            "dim": dim, "residual": residual, "pad": pad}


def _linear(name, tokens, k, n, act, bias, residual):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "act": act,
            "bias": bias, "residual": residual}


def listed():
    return [
        # the router of one decoded token: the smallest call, all latency
        _route("route_token", 1, 64, 8, False, True, 0),
        # the router of a full prompt chunk, fp32 logits, its last rows padding
        _route("route_prompt", 4096, 128, 8, True, False, 96),
        # one decoded token through its experts' gate|up with SwiGLU
        _grouped("experts_up_token", 1, 64, 8, 2048, 2048, True, "swiglu", False, 0),
        # the widest verify block through the experts' down projection: a few rows an expert
        _grouped("experts_down_verify", 16, 64, 8, 1024, 2048, False, "none", False, 0),
        # a chat turn over few wide experts (the eight-way shard's width): tens of rows
        # an expert, ragged
        _grouped("experts_up_chat", 200, 32, 4, HIDDEN, 2 * SHARD_INTER, True, "swiglu", False, 0),
        # the down projection of an odd prompt with expert biases and padded tokens
        _grouped("experts_down_odd", 1001, 32, 4, SHARD_INTER, HIDDEN, False, "none", True, 23),
        # a full prompt chunk through the experts' gate|up with SwiGLU
        _grouped("experts_up_prompt", 4096, 64, 8, 2048, 2048, True, "swiglu", False, 0),
        # expert rows of a verify block back into its hidden states
        _combine("combine_verify", 9, 64, 8, 2048, True, 0),
        # the same for a full prompt chunk
        _combine("combine_prompt", 4096, 64, 8, 2048, True, 96),
        # the qkv projection of one token, with bias
        _linear("linear_qkv_token", 1, HIDDEN, QKV, "none", True, False),
        # the gate|up projection of a verify block (last token and eight drafts)
        _linear("linear_up_verify", 9, HIDDEN, 2 * INTER, "swiglu", False, False),
        # the down projection of a full prompt chunk, added to the hidden states
        _linear("linear_down_prompt", 4096, INTER, HIDDEN, "none", False, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    r = rng.random()
    experts = _log_int(rng, 4, 256)
    top_k = rng.randint(1, min(8, experts))
    if r < 0.2:
        tokens = _log_int(rng, 1, 4096)
        c = _route("", tokens, experts, top_k, rng.random() < 0.5, rng.random() < 0.5,
                   rng.randint(0, tokens // 4))
    elif r < 0.6:
        experts = min(experts, 96)
        top_k = min(top_k, experts)
        k = GROUP * rng.randint(2, 40)
        act = rng.choice(ACTS + ("swiglu", "none"))
        n = 128 * rng.randint(2, 34) if act == "swiglu" else 64 * rng.randint(3, 80)
        tokens = _log_int(rng, 1, 4096)
        while 2.0 * tokens * top_k * k * n > MAX_FLOPS:
            tokens = tokens * 2 // 3
        c = _grouped("", tokens, experts, top_k, k, n, rng.random() < 0.5, act,
                     rng.random() < 0.3, rng.randint(0, tokens // 4))
    elif r < 0.72:
        tokens = _log_int(rng, 1, 4096)
        c = _combine("", tokens, experts, top_k, 8 * rng.randint(16, 256), rng.random() < 0.6,
                     rng.randint(0, tokens // 4))
    else:
        k = rng.choice((HIDDEN, ATTN, SHARD_INTER, INTER, GROUP * rng.randint(1, 60)))
        act = rng.choice(ACTS + ("swiglu", "none"))
        n = 128 * rng.randint(2, 200) if act == "swiglu" else 64 * rng.randint(3, 240)
        tokens = rng.choice((1, rng.randint(2, 16), _log_int(rng, 17, 4096)))
        while 2.0 * tokens * k * n > MAX_FLOPS_DENSE:
            tokens = tokens * 2 // 3
        c = _linear("", tokens, k, n, act, rng.random() < 0.5, rng.random() < 0.5)
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


def _logits(g, c):
    """Router logits; the last `pad` rows belong to no token and choose no expert."""
    t, e = c["tokens"], c["experts"]
    popular = 0.7 * torch.randn(e, generator=g, device="cuda")
    x = 1.5 * torch.randn(t, e, generator=g, device="cuda") + popular
    x[t - c["pad"]:] = -math.inf
    return x


def _choice(g, c):
    """Experts [T][k] of each token (-1: none) and their normalised weights."""
    x = _logits(g, c)
    v, ids = torch.sort(x, dim=1, descending=True)
    v, ids = v[:, :c["top_k"]], ids[:, :c["top_k"]]
    live = v > -math.inf
    e = torch.where(live, torch.exp(v - v[:, :1]), torch.zeros_like(v))
    weights = torch.where(live, e / e.sum(1, keepdim=True), torch.zeros_like(v))
    return torch.where(live, ids, torch.full_like(ids, -1)), weights


def _plan(ids, experts):
    """Pairs (token, slot) by expert, in order: offsets [E + 1], the token at each
    position (-1 behind the last) and each pair's position (-1: none)."""
    t, k = ids.shape
    flat = ids.reshape(-1)
    order = torch.sort(torch.where(flat < 0, experts, flat), stable=True).indices
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.cumsum(counts, 0)
    at = torch.arange(t * k, device=flat.device)
    live = at < offsets[-1]
    tokens = torch.where(live, order // k, -1)
    pos = torch.empty_like(order)
    pos[order] = torch.where(live, at, -1)
    i32 = torch.int32
    return offsets.to(i32), tokens.to(i32), pos.to(i32)


def _inputs(case, seed):
    """Everything a pass reads, made from the seed alone."""
    g, c = _gen(seed), case
    d = {}
    if c["op"] == "route":
        x = _logits(g, c)
        d["logits"] = x if c["f32"] else x.to(torch.bfloat16)
        return d
    if c["op"] in ("grouped", "combine"):
        ids, weights = _choice(g, c)
        d["offsets"], d["tokens"], d["pos"] = _plan(ids, c["experts"])
        pairs = c["tokens"] * c["top_k"]
        if c["op"] == "combine":
            d["weights"] = weights.contiguous()
            d["y"] = _hidden(g, pairs, c["dim"])
            d["residual"] = _hidden(g, c["tokens"], c["dim"]) if c["residual"] else None
            return d
        d["x"] = _hidden(g, c["tokens"] if c["gather"] else pairs, c["k"])
        d["int4"] = _int4(g, c["experts"] * c["n"], c["k"])
        d["bias"] = _hidden(g, 1, c["experts"] * c["n"])[0] if c["bias"] else None
        return d
    d["x"] = _hidden(g, c["tokens"], c["k"])
    d["int4"] = _int4(g, c["n"], c["k"])
    d["bias"] = _hidden(g, 1, c["n"])[0] if c["bias"] else None
    width = c["n"] // 2 if c["act"] == "swiglu" else c["n"]
    d["residual"] = _hidden(g, c["tokens"], width) if c["residual"] else None
    return d


def prepare(case, seed):
    st = State(dict(case))
    c, d = st.case, _inputs(case, seed)
    st.d = d
    if c["op"] == "combine":
        st.out = torch.zeros(c["tokens"], c["dim"], dtype=torch.bfloat16, device="cuda")
    elif c["op"] in ("grouped", "linear"):
        rows = c["tokens"] * c.get("top_k", 1)
        width = c["n"] // 2 if c["act"] == "swiglu" else c["n"]
        st.out = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    else:
        t, k = c["tokens"], c["top_k"]
        i32 = dict(dtype=torch.int32, device="cuda")
        st.ids = torch.zeros(t, k, **i32)
        st.weights = torch.zeros(t, k, dtype=torch.float32, device="cuda")
        st.offsets = torch.zeros(c["experts"] + 1, **i32)
        st.tokens, st.pos = torch.zeros(t * k, **i32), torch.zeros(t * k, **i32)
    if not own:
        return st
    hip = _hip()
    if c["op"] == "route":
        st.plan = hip.expert_plan_over(st.offsets, st.tokens, st.pos)
    elif c["op"] in ("grouped", "combine"):
        st.plan = hip.expert_plan_over(d["offsets"], d["tokens"], d["pos"])
    if "int4" in d:
        packed, scale, zp = d["int4"]
        n = packed.shape[0]
        st.w = st.keep(hip.awq_free, hip.awq_alloc_fused(n, c["k"]))
        hip.awq_repack_into(st.w, 0, packed, scale, zp, n)
        st.ws = st.keep(hip.gemm_workspace_free, hip.gemm_workspace_alloc(256 << 20))
        if c["op"] == "linear":
            st.scratch = st.keep(hip.gemv_scratch_free, hip.gemv_scratch_alloc(c["k"], n, GROUP, 16))
            st.act = getattr(hip, "ACT_" + c["act"].upper())
        else:
            st.act = getattr(hip, "ACT_" + c["act"].upper())
    return st


# -------------------------------------------------------------- plain forms
def _levels(words, axis):
    """Eight 4-bit levels of each int32 word, lowest first, along `axis`."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    v = (words.unsqueeze(axis + 1) >> shifts.view((8,) + (1,) * (words.dim() - 1 - axis))) & 15
    return v.flatten(axis, axis + 1)


def _dequant(int4, r0, r1):
    """Rows [r0, r1) as fp32: (q - zp) s."""
    packed, scale, zp = int4
    k = packed.shape[1] * 8
    q = _levels(packed[r0:r1], 1).float().view(r1 - r0, k // GROUP, GROUP)
    z = _levels(zp[r0 // 8:r1 // 8], 0).float()
    return ((q - z[:, :, None]) * scale[r0:r1].float()[:, :, None]).view(r1 - r0, k)


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


def _plain_route(st):
    c, x = st.case, st.d["logits"].float()
    k = c["top_k"]
    v, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top = v[:, :1]
    e = torch.where(v > -math.inf, torch.exp(v - top), torch.zeros_like(v))
    total = (e[:, :k] if c["renorm"] else e).sum(1, keepdim=True)
    live = v[:, :k] > -math.inf
    weights = torch.where(live, e[:, :k] / total, torch.zeros_like(total))
    ids = torch.where(live, ids[:, :k], -1)
    offsets, tokens, pos = _plan(ids, c["experts"])
    return ids.to(torch.int32), weights, offsets, tokens, pos


def _plain_grouped(st):
    c, d, n = st.case, st.d, st.case["n"]
    out = st.out.clone()
    bounds = d["offsets"].tolist()
    for e in range(c["experts"]):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        x = d["x"][d["tokens"][lo:hi].long()] if c["gather"] else d["x"][lo:hi]
        v = x.float() @ _dequant(d["int4"], e * n, (e + 1) * n).t()
        if c["bias"]:
            v = v + d["bias"][e * n:(e + 1) * n].float()
        out[lo:hi] = _activate(v, c["act"]).to(torch.bfloat16)
    return out


def _plain_combine(st):
    c, d = st.case, st.d
    at = d["pos"].view(c["tokens"], c["top_k"]).long()
    acc = d["residual"].float() if c["residual"] else torch.zeros(
        c["tokens"], c["dim"], device="cuda")
    for j in range(c["top_k"]):
        live = (at[:, j] >= 0)[:, None]
        rows = d["y"][at[:, j].clamp(min=0)].float()
        acc = acc + torch.where(live, d["weights"][:, j:j + 1] * rows, torch.zeros_like(rows))
    return acc.to(torch.bfloat16)


def _plain_linear(st):
    c, d = st.case, st.d
    v = d["x"].float() @ _dequant(d["int4"], 0, c["n"]).t()
    if c["bias"]:
        v = v + d["bias"].float()
    v = _activate(v, c["act"])
    if c["residual"]:
        v = v + d["residual"].float()
    return v.to(torch.bfloat16)


def run(st):
    c, d = st.case, st.d
    if not own:
        return {"route": _plain_route, "grouped": _plain_grouped, "combine": _plain_combine,
                "linear": _plain_linear}[c["op"]](st)
    hip = _hip()
    if c["op"] == "route":
        call = hip.route_experts_f32 if c["f32"] else hip.route_experts
        call(st.ids, st.weights, d["logits"], c["tokens"], c["experts"], c["top_k"], c["renorm"], st.plan)
        return st.ids, st.weights, st.offsets, st.tokens, st.pos
    if c["op"] == "grouped":
        hip.gemm_grouped_w4a16(st.out, st.w, d["x"], st.plan, c["tokens"] * c["top_k"],
                               gather=c["gather"], bias=d["bias"], act=st.act, ws=st.ws)
    elif c["op"] == "combine":
        hip.combine_experts(st.out, d["y"], d["weights"], c["tokens"], c["top_k"], c["dim"], st.plan,
                            residual=d["residual"])
    else:
        hip.linear_epilogue_w4a16(st.out, st.w, d["x"], c["tokens"], st.scratch, st.ws, bias=d["bias"],
                                  act=st.act, residual=d["residual"])
    return st.out


# -------------------------------------------------------------- exact values
def _exact_rows(x, int4, r0, r1, bias):
    packed, scale, zp = int4
    n, groups = r1 - r0, packed.shape[1] * 8 // GROUP
    words = packed[r0:r1].to(torch.int64) & 0xFFFFFFFF
    q = torch.stack([(words // 16 ** i) % 16 for i in range(8)], -1).reshape(n, groups, GROUP)
    zw = zp[r0 // 8:r1 // 8].to(torch.int64) & 0xFFFFFFFF
    z = torch.stack([(zw // 16 ** i) % 16 for i in range(8)], 1).reshape(n, groups, 1)
    w = ((q - z).double() * scale[r0:r1].double().reshape(n, groups, 1)).reshape(n, -1)
    v = torch.matmul(x.double(), w.t().contiguous())
    return v if bias is None else v + bias[r0:r1].double()


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


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "route":
        x, k = d["logits"].double(), c["top_k"]
        t, e = x.shape
        # stable by expert: among equal logits the lower expert comes first
        rank = torch.argsort(-x, dim=1, stable=True)[:, :k]
        v = torch.gather(x, 1, rank)
        live = torch.isfinite(v)
        base = torch.logsumexp(v if c["renorm"] else x, 1, keepdim=True)
        weights = torch.where(live, torch.exp(v - base), torch.zeros_like(v))
        ids = torch.where(live, rank, -1).cpu()
        lists = [[] for _ in range(e)]
        for i, expert in enumerate(ids.flatten().tolist()):
            if expert >= 0:
                lists[expert].append(i)
        pairs = [i for group in lists for i in group]
        offsets = [0]
        for group in lists:
            offsets.append(offsets[-1] + len(group))
        pos = [-1] * (t * k)
        for at, i in enumerate(pairs):
            pos[i] = at
        tokens = [i // k for i in pairs] + [-1] * (t * k - len(pairs))
        i32 = dict(dtype=torch.int32, device="cuda")
        return (ids.to(**i32), weights, torch.tensor(offsets, **i32), torch.tensor(tokens, **i32),
                torch.tensor(pos, **i32))
    if c["op"] == "combine":
        at = d["pos"].reshape(c["tokens"], c["top_k"]).long()
        w = torch.where(at >= 0, d["weights"].double(), 0.0)
        out = torch.matmul(w[:, None, :], d["y"].double()[at.clamp(min=0)])[:, 0]
        return out + d["residual"].double() if c["residual"] else out
    if c["op"] == "grouped":
        n, bounds = c["n"], d["offsets"].cpu()
        width = n // 2 if c["act"] == "swiglu" else n
        out = torch.zeros(c["tokens"] * c["top_k"], width, dtype=torch.float64, device="cuda")
        source = d["tokens"].long() if c["gather"] else torch.arange(out.shape[0], device="cuda")
        for e in range(c["experts"]):
            i = torch.arange(int(bounds[e]), int(bounds[e + 1]), device="cuda")
            if len(i):
                v = _exact_rows(d["x"][source[i]], d["int4"], e * n, (e + 1) * n, d["bias"])
                out[i] = _exact_activation(v, c["act"])
        return out
    out = _exact_activation(_exact_rows(d["x"], d["int4"], 0, c["n"], d["bias"]), c["act"])
    return out + d["residual"].double() if c["residual"] else out


# --------------------------------------------------------------------- work
def work(case):
    c, t = case, case["tokens"]
    if c["op"] == "route":
        pairs = t * c["top_k"]
        size = 4 if c["f32"] else 2
        return {"bytes": t * c["experts"] * size + 16 * pairs + 4 * (c["experts"] + 1),
                "flops": 4 * t * c["experts"]}
    live = t - c.get("pad", 0)
    if c["op"] == "combine":
        rows = live * c["top_k"]
        return {"bytes": 2 * c["dim"] * (rows + t * (2 if c["residual"] else 1)) + 8 * t * c["top_k"],
                "flops": 2 * rows * c["dim"]}
    k, n = c["k"], c["n"]
    width = n // 2 if c["act"] == "swiglu" else n
    weight = n * k * (0.5 + 2.5 / GROUP)
    if c["op"] == "grouped":
        # experts that some token is expected to choose, were all as popular
        used = c["experts"] * (1.0 - (1.0 - c["top_k"] / c["experts"]) ** live)
        rows = live * c["top_k"]
        inputs = live if c["gather"] else rows
        return {"bytes": int(used * (weight + (2 * n if c["bias"] else 0)) + 2 * inputs * k
                             + 2 * rows * width + 4 * rows),
                "flops": 2 * rows * n * k}
    extra = (2 * n if c["bias"] else 0) + (2 * t * width if c["residual"] else 0)
    return {"bytes": int(weight + 2 * t * (k + width) + extra), "flops": 2 * t * n * k}
