"""Cases of the operators that surround the quantized linears of a transformer block.

Three operators: the RMS norm with the residual's addition and a bf16 or E4M3 output, the matrix product with
bias, activation, gate and residual in its epilogue (bf16 operands, or E4M3 with one scale per row), and the
paged FP8 store of keys and values, quantized as it is written and read back in bf16.

``own = False`` computes each in plain torch operations in fp32, rounded once at the end; ``own = True`` calls
the framework.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3_MAX = 448.0
TINY = 1e-12
DEV = "cuda"


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token between two blocks of width 1536: latency
        {"name": "norm_fp8_1x1536", "op": "norm", "rows": 1, "d": 1536, "inner": 1, "gap": 0, "out": "fp8",
         "residual": "bf16"},
        # the pre-norm of a block over a video chunk, its output quantized for the W8A8 product
        {"name": "norm_fp8_15360x1536", "op": "norm", "rows": 15360, "d": 1536, "inner": 1, "gap": 0, "out": "fp8",
         "residual": "bf16"},
        # per-head norm of the queries inside a fused projection's rows (strided view, 12 heads of 128)
        {"name": "norm_heads_7680x12x128", "op": "norm", "rows": 92160, "d": 128, "inner": 12, "gap": 2048,
         "out": "bf16", "residual": "none"},
        # ragged row length with an fp32 residual stream
        {"name": "norm_f32res_4099x2047", "op": "norm", "rows": 4099, "d": 2047, "inner": 1, "gap": 0, "out": "bf16",
         "residual": "fp32"},
        # first linear of the FFN for one token: reading the weight is all there is
        {"name": "linear_1x1536x8960", "op": "linear", "m": 1, "k": 1536, "n": 8960, "type": "bf16",
         "act": "gelu_tanh", "gated": False, "bias": True, "residual": False},
        # second linear of the W8A8 FFN for a small batch of tokens, added to the stream
        {"name": "linear_fp8_24x8960x1536", "op": "linear", "m": 24, "k": 8960, "n": 1536, "type": "fp8",
         "act": "none", "gated": False, "bias": True, "residual": True},
        # gated FFN input of a prompt of odd length
        {"name": "linear_gated_777x1536x4104", "op": "linear", "m": 777, "k": 1536, "n": 4104, "type": "bf16",
         "act": "silu", "gated": True, "bias": False, "residual": False},
        # second linear of the bf16 FFN over a chunk, added to the stream
        {"name": "linear_15360x8960x1536", "op": "linear", "m": 15360, "k": 8960, "n": 1536, "type": "bf16",
         "act": "none", "gated": False, "bias": True, "residual": True},
        # first linear of the W8A8 FFN, gated, over a chunk
        {"name": "linear_fp8_gated_7680x1536x8960", "op": "linear", "m": 7680, "k": 1536, "n": 8960, "type": "fp8",
         "act": "gelu_tanh", "gated": True, "bias": True, "residual": False},
        # a batch of decoded tokens stored, one in eight of the batch's rows padding
        {"name": "store_64x12x128", "op": "store", "tokens": 64, "heads": 12, "d": 128, "page": 16, "spare": 448,
         "padded": True},
        # a video chunk stored
        {"name": "store_7680x12x128", "op": "store", "tokens": 7680, "heads": 12, "d": 128, "page": 64, "spare": 7680,
         "padded": False},
        # the window of four streams read back for bf16 attention, ragged lengths
        {"name": "fetch_4x7680x12x128", "op": "fetch", "batch": 4, "longest": 7680, "heads": 12, "d": 128, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "linear", "linear", "linear", "store", "fetch"])
    if op == "norm":
        d = _log_int(rng, 64, 8960)
        if rng.random() < 0.7:
            d = max(64, d // 8 * 8)
        inner = rng.choice([1, 1, 1, 4, 12]) if d <= 256 else 1
        rows = max(1, min(_log_int(rng, 1, 65536), 30_000_000 // d))
        rows = max(1, rows // inner) * inner
        return {"op": op, "rows": rows, "d": d, "inner": inner,
                "gap": 8 * rng.randrange(0, 300) if d % 8 == 0 and rng.random() < 0.3 else 0,
                "out": rng.choice(["bf16", "fp8"]), "residual": rng.choice(["none", "bf16", "fp32"])}
    if op == "linear":
        gated = rng.random() < 0.4
        m = _log_int(rng, 1, 16384)
        k = max(64, _log_int(rng, 64, 8960) // 16 * 16)
        n = max(64, _log_int(rng, 64, 8960) // 8 * 8)
        most = 420e9 / (2 * k * n * (2 if gated else 1))
        return {"op": op, "m": max(1, min(m, int(most))), "k": k, "n": n, "type": rng.choice(["bf16", "fp8"]),
                "act": rng.choice(["silu", "gelu_tanh", "gelu", "relu"] if gated else
                                  ["none", "none", "gelu_tanh", "silu", "gelu", "relu"]),
                "gated": gated, "bias": rng.random() < 0.6, "residual": rng.random() < 0.5}
    heads, d, page = rng.choice([1, 2, 5, 8, 12, 16]), rng.choice([64, 80, 96, 128, 256]), rng.choice([1, 16, 48, 64])
    if op == "store":
        tokens = max(1, min(_log_int(rng, 1, 16384), 15_000_000 // (heads * d)))
        return {"op": op, "tokens": tokens, "heads": heads, "d": d, "page": page,
                "spare": rng.randrange(0, 2 * tokens + 16), "padded": rng.random() < 0.3}
    batch = _log_int(rng, 1, 32)
    longest = max(1, min(_log_int(rng, 1, 16384), 40_000_000 // (batch * heads * d)))
    return {"op": op, "batch": batch, "longest": longest, "heads": heads, "d": d, "page": page}


# ---------------------------------------------------------------- inputs
def _codes(v):
    """(E4M3 codes, one fp32 scale a row) of fp32 rows."""
    s = (v.abs().amax(-1, keepdim=True) / torch.full((), E4M3_MAX, device=v.device)).clamp_min(TINY)
    return (v / s).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * std

    c = dict(case)
    op = c["op"]
    if op == "norm":
        rows, d, inner, gap = c["rows"], c["d"], c["inner"], c["gap"]
        outer = rows // inner
        # activations of a stream: a few channels far larger than the rest
        x = normal(outer, inner * d + gap)
        x[:, :: 97] *= 8.0
        x = x.to(torch.bfloat16)[:, :inner * d].unflatten(1, (inner, d))
        c["x"] = x if inner > 1 else x[:, 0]
        c["w"] = (1.0 + normal(d, std=0.2)).to(torch.bfloat16)
        shape = c["x"].shape
        c["r"] = {"none": None, "bf16": torch.bfloat16, "fp32": torch.float32}[c["residual"]]
        if c["r"] is not None:
            c["r"] = normal(*shape, std=3.0).to(c["r"])
    elif op == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        wn = 2 * n if c["gated"] else n
        x, w = normal(m, k), normal(wn, k, std=1.0 / math.sqrt(k))
        if c["type"] == "fp8":
            c["x"], c["sx"] = _codes(x)
            c["w"], c["sw"] = _codes(w)
        else:
            c["x"], c["w"] = x.to(torch.bfloat16), w.to(torch.bfloat16)
        c["b"] = normal(wn, std=0.1).to(torch.bfloat16) if c["bias"] else None
        c["r"] = normal(m, n).to(torch.bfloat16) if c["residual"] else None
    else:
        heads, d, page = c["heads"], c["d"], c["page"]
        if op == "store":
            t = c["tokens"]
            pages = -(-(t + c["spare"]) // page)
            # a chunk's tokens fill pages one after another, the pages lie anywhere
            at = torch.randperm(pages, generator=g, device=DEV)
            slots = (at[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:t]
            if c["padded"]:
                slots = torch.where(torch.arange(t, device=DEV) % 8 == 7, -1, slots)
            c["slots"] = slots.contiguous()
            qkv = normal(t, 3, heads, d, std=1.5).to(torch.bfloat16)  # a fused projection's rows
            c["k"], c["v"] = qkv[:, 1], qkv[:, 2]
        else:
            b, longest = c["batch"], c["longest"]
            per = -(-longest // page)
            pages = b * per + 3
            lens = torch.randint(max(1, longest // 3), longest + 1, (b,), generator=g, device=DEV)
            lens[0] = longest
            if b > 2:
                lens[2] = 0
            c["lens"] = lens.to(torch.int32)
            c["table"] = torch.randperm(pages, generator=g, device=DEV)[:b * per].view(b, per).to(torch.int32)
        for name in ("k", "v"):
            q, s = _codes(normal(pages, page, heads, d))
            c[name + "_codes"], c[name + "_scale"] = q, s[..., 0].contiguous()
    return c


# ---------------------------------------------------------------- one pass
def _activate(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(z * -math.sqrt(0.5))
    return z


def run(state):
    op = state["op"]
    if own:
        return _run_own(state, op)
    if op == "norm":
        s, r = state["x"].float(), state["r"]
        out = []
        if r is not None:
            s = s + r
            out = [s.to(r.dtype)]
        v = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + 1e-6) * state["w"].float()
        return [*_codes(v), *out] if state["out"] == "fp8" else [v.to(torch.bfloat16), *out]
    if op == "linear":
        z = torch.matmul(state["x"].float(), state["w"].float().t())
        if state["type"] == "fp8":
            z = z * state["sx"] * state["sw"].t()
        if state["b"] is not None:
            z = z + state["b"]
        if state["gated"]:
            a, u = z.chunk(2, -1)
            z = _activate(a, state["act"]) * u
        else:
            z = _activate(z, state["act"])
        if state["r"] is not None:
            z = z + state["r"]
        return z.to(torch.bfloat16)
    if op == "store":
        slots, k, v = state["slots"], state["k"], state["v"]
        if state["padded"]:
            keep = slots >= 0
            slots, k, v = slots[keep], k[keep], v[keep]
        return [*_store(k, slots, state["k_codes"], state["k_scale"]),
                *_store(v, slots, state["v_codes"], state["v_scale"])]
    table, longest = state["table"].long(), state["longest"]
    used = (torch.arange(longest, device=table.device) < state["lens"][:, None])[..., None, None]
    return [_fetch(state["k_codes"], state["k_scale"], table, longest, used),
            _fetch(state["v_codes"], state["v_scale"], table, longest, used)]


def _store(x, slots, codes, scale):
    q, s = _codes(x.float())
    codes.view(torch.uint8).flatten(0, 1)[slots] = q.view(torch.uint8)
    scale.flatten(0, 1)[slots] = s[..., 0]
    return codes, scale


def _fetch(codes, scale, table, longest, used):
    q = codes.view(torch.uint8)[table].flatten(1, 2)[:, :longest].view(torch.float8_e4m3fn)
    s = scale[table].flatten(1, 2)[:, :longest]
    return torch.where(used, q.float() * s[..., None], torch.zeros((), device=s.device)).to(torch.bfloat16)


def _run_own(state, op):
    from flashvsr_optimizations_b200 import ops
    if op == "norm":
        x, w, r = state["x"], state["w"], state["r"]
        if state["out"] == "fp8":
            return ops.rms_norm_fp8(x, w) if r is None else ops.add_rms_norm_fp8(x, r, w)
        return [ops.rms_norm(x, w)] if r is None else ops.add_rms_norm(x, r, w)
    if op == "linear":
        if state["type"] == "fp8":
            return ops.fp8_scaled_mm_act(state["x"], state["sx"], state["w"], state["sw"], state["b"],
                                         act=state["act"], gated=state["gated"], residual=state["r"])
        return ops.linear_act(state["x"], state["w"], state["b"], act=state["act"], gated=state["gated"],
                              residual=state["r"])
    cache = state["k_codes"], state["k_scale"], state["v_codes"], state["v_scale"]
    if op == "store":
        ops.fp8_cache_write(state["k"], state["v"], state["slots"], *cache)
        return cache
    return ops.fp8_cache_read(*cache, state["table"], state["lens"], state["longest"])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        n, each = case["rows"] * case["d"], {"none": 0, "bf16": 2, "fp32": 4}[case["residual"]]
        wide = 1 if case["out"] == "fp8" else 2
        return {"bytes": n * (2 + 2 * each + wide) + 2 * case["d"] + (4 * case["rows"] if wide == 1 else 0),
                "flops": 6 * n}
    if op == "linear":
        m, k, n, e = case["m"], case["k"], case["n"], 1 if case["type"] == "fp8" else 2
        wn = 2 * n if case["gated"] else n
        return {"bytes": e * (m + wn) * k + (4 * (m + wn) if e == 1 else 0) + (2 * wn if case["bias"] else 0)
                + 2 * m * n * (2 if case["residual"] else 1), "flops": 2 * m * wn * k}
    h, d = case["heads"], case["d"]
    if op == "store":
        t = case["tokens"]
        if case["padded"]:
            t -= t // 8
        return {"bytes": 2 * t * h * (3 * d + 4) + 8 * case["tokens"], "flops": 4 * t * h * d}
    t, longest = case["batch"], case["longest"]
    read = 0.6 * t * longest  # the lengths are drawn between a third of the longest and the longest
    return {"bytes": 2 * h * (read * (d + 4) + t * longest * 2 * d), "flops": 2 * read * h * d}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_codes(v):
    s = torch.maximum(v.abs().amax(-1, keepdim=True) / E4M3_MAX, v.new_full((), TINY))
    return v / s, s


def _exact_store(x, slots, codes, scale):
    rows = slots >= 0
    q, s = _exact_codes(x.double()[rows])
    codes, scale = codes.double(), scale.double()
    codes.flatten(0, 1)[slots[rows]] = q
    scale.flatten(0, 1)[slots[rows]] = s[..., 0]
    return codes, scale


def _exact_activation(a, act):
    if act == "relu":
        return a.clamp_min(0)
    if act == "silu":
        return a * torch.sigmoid(a)
    if act == "gelu_tanh":
        return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    return 0.5 * a * (1 + torch.erf(a / math.sqrt(2))) if act == "gelu" else a


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "norm":
        s = st["x"].double()
        if st["r"] is not None:
            s = s + st["r"].double()
        v = s / torch.sqrt(s.square().sum(-1, keepdim=True) / case["d"] + 1e-6) * st["w"].double()
        first = list(_exact_codes(v)) if case["out"] == "fp8" else [v]
        return first + ([] if st["r"] is None else [s])
    if op == "linear":
        z = st["x"].double() @ st["w"].double().T
        if case["type"] == "fp8":
            z *= st["sx"].double()
            z *= st["sw"].double().T
        if case["bias"]:
            z += st["b"].double()
        h = _exact_activation(z[:, :case["n"]] if case["gated"] else z, case["act"])
        if case["gated"]:
            h = h * z[:, case["n"]:]
        return h + st["r"].double() if case["residual"] else h
    if op == "store":
        return [*_exact_store(st["k"], st["slots"], st["k_codes"], st["k_scale"]),
                *_exact_store(st["v"], st["slots"], st["v_codes"], st["v_scale"])]
    out = []
    for name in ("k", "v"):
        full = st[name + "_codes"].double() * st[name + "_scale"].double()[..., None]
        got = full.new_zeros(case["batch"], case["longest"], case["heads"], case["d"])
        for i, n in enumerate(st["lens"].tolist()):
            got[i, :n] = full[st["table"][i].long()].flatten(0, 1)[:n]
        out.append(got)
    return out
