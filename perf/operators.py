"""The operators of the 8-bit serving path, as measured cases: the KV cache held in 8 bits (quantised as it is written, read
back, attended to by single tokens), the row-quantising layer kernels around the projections (residual add + RMSNorm,
SiLU*mul) and the 8-bit integer projections themselves.

``own`` false computes every operator in its plain form with elementary torch operations in 32 bits (64 where a value can
lie next to a rounding border); ``own`` true makes the calls a serving program makes of ``loongserve_b200``.

Codes.  A row (one head of one token in the cache, one token's activations, one output channel of a weight) is held as codes
and one fp32 scale: amax = max(max|x|, 2^-100); int8: scale = amax/127, code = rint(x * fl32(127/amax)); e4m3: scale =
amax/448, code = e4m3(x * fl32(448/amax)).  The value a code stands for is code * scale.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128                                        # head dim of the attention path
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100


def listed():
    return [
        # one decode step of a batch writes its new tokens' K and V rows of a layer, and they are read back
        {"name": "kv_write_step", "op": "kv_write", "tokens": 64, "kv_heads": 32, "code": "int8", "dtype": "bf16", "pool": 20000},
        # a long prompt's rows of a layer go into the pool at scattered slots
        {"name": "kv_write_prompt", "op": "kv_write", "tokens": 16384, "kv_heads": 32, "code": "e4m3", "dtype": "bf16", "pool": 32768},
        # a layer's rows of cached requests come back as 16-bit rows (hand-over to an instance that holds them so)
        {"name": "kv_read_back", "op": "kv_read", "tokens": 65535, "kv_heads": 8, "code": "int8", "dtype": "f16", "pool": 100003},
        # one short conversation: latency of a single layer call
        {"name": "decode_one_short", "op": "decode", "batch": 1, "min_len": 513, "max_len": 513, "q_heads": 32, "kv_heads": 8,
         "code": "int8", "dtype": "bf16"},
        # an ordinary serving batch with as many kv heads as q heads, ragged lengths
        {"name": "decode_batch", "op": "decode", "batch": 32, "min_len": 1024, "max_len": 16384, "q_heads": 32, "kv_heads": 32,
         "code": "int8", "dtype": "bf16"},
        # two very long contexts, grouped heads, e4m3 codes
        {"name": "decode_long_grouped", "op": "decode", "batch": 2, "min_len": 200001, "max_len": 262144, "q_heads": 32, "kv_heads": 8,
         "code": "e4m3", "dtype": "f16"},
        # decode step: residual add and norm, 16-bit output (the last norm before the logits)
        {"name": "norm_step", "op": "norm", "tokens": 64, "hidden": 4096, "dtype": "bf16", "quant": False},
        # prompt: residual add and norm with the 8-bit rows that the projection reads
        {"name": "norm_prompt_q8", "op": "norm", "tokens": 16384, "hidden": 4096, "dtype": "bf16", "quant": True},
        # decode step of a ragged batch: gate/up product of the FFN into 8-bit rows
        {"name": "silu_step", "op": "silu", "tokens": 33, "ffn": 11008, "dtype": "f16"},
        # the same for a prompt
        {"name": "silu_prompt", "op": "silu", "tokens": 8192, "ffn": 11008, "dtype": "bf16"},
        # decode step: the FFN's down projection for a batch (weights are what is read)
        {"name": "mm_step", "op": "mm", "tokens": 64, "in": 11008, "out": 4096, "dtype": "bf16"},
        # prompt: the FFN's gate and up projection
        {"name": "mm_prompt", "op": "mm", "tokens": 16384, "in": 4096, "out": 22016, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv_write", "kv_read", "decode", "decode", "norm", "silu", "mm", "mm"])
    dtype = rng.choice(["bf16", "f16"])
    code = rng.choice(["int8", "e4m3"])
    if op in ("kv_write", "kv_read"):
        heads = rng.choice([1, 2, 4, 8, 16, 32])
        n = _log_int(rng, 1, 16384 * 32 // max(heads, 8))
        return {"op": op, "tokens": n, "kv_heads": heads, "code": code, "dtype": dtype, "pool": n + _log_int(rng, 1, 20000)}
    if op == "decode":
        heads = rng.choice([1, 2, 4, 8, 32])
        group = rng.choice([1, 2, 4, 5, 8, 16]) if heads < 8 else rng.choice([1, 2, 4])
        batch = _log_int(rng, 1, 96)
        top = _log_int(rng, 1, min(200000, 32 * 16384 * 32 // (batch * max(heads, 4))))
        return {"op": op, "batch": batch, "min_len": rng.randint(0 if batch > 1 else 1, top), "max_len": top, "q_heads": heads * group,
                "kv_heads": heads, "code": code, "dtype": dtype}
    if op == "norm":
        hidden = 8 * _log_int(rng, 16, 1400)
        return {"op": op, "tokens": _log_int(rng, 1, 16384 * 4096 // hidden), "hidden": hidden, "dtype": dtype, "quant": rng.random() < 0.6}
    if op == "silu":
        ffn = 8 * _log_int(rng, 16, 1800)
        return {"op": op, "tokens": _log_int(rng, 1, 8192 * 8192 // ffn), "ffn": ffn, "dtype": dtype}
    k = 16 * _log_int(rng, 8, 700)
    n = _log_int(rng, 100, 22016)
    return {"op": "mm", "tokens": _log_int(rng, 1, min(16384, 16384 * 4096 // k)), "in": k, "out": n, "dtype": dtype}


# ---------------------------------------------------------------------------------------------- plain quantisation
def _amax(x):
    """max|x| of the last dimension in fp32, not below 2^-100."""
    return x.abs().amax(-1, keepdim=True).float().clamp_min(TINY)


def _codes(x, inv, code):
    """Codes of x (fp32) by the fp32 factor inv: the product goes to the nearest code, ties to the even one."""
    if code == "int8":                          # in 64 bits: a product of 24-bit numbers is exact there, so no border is missed
        return torch.round(x.double() * inv.double()).to(torch.int8)
    return (x * inv).to(torch.float8_e4m3fn)


def _quantise(x, code):
    a = _amax(x)
    return _codes(x.float(), TOP[code] / a, code), (a / TOP[code]).squeeze(-1)


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _pool_views(rows, heads2, code):
    """A pool whose row keeps a token whole: heads2 * D codes, then heads2 fp32 scales."""
    width = (heads2 * (D + 4) + 15) // 16 * 16
    raw = torch.zeros(rows, width, dtype=torch.uint8, device=DEV)
    codes = raw[:, :heads2 * D].view(CODES[code]).unflatten(1, (heads2, D))
    scales = raw[:, heads2 * D:heads2 * (D + 4)].view(torch.float32)
    return raw, codes, scales


def _rows_like_kv(g, n, heads2, dtype):
    """K and V rows as a projection leaves them: heads of different size, a few large channels, tokens of different size."""
    x = torch.randn(n, heads2, D, generator=g, device=DEV, dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn(1, heads2, 1, generator=g, device=DEV))
    x *= torch.exp(0.2 * torch.randn(n, 1, 1, generator=g, device=DEV))
    x[:, :, :2] *= 3.0
    return x.to(dtype)


def _fill_pool(g, codes, scales, code, dtype):
    for a in range(0, codes.shape[0], 16384):
        x = _rows_like_kv(g, min(16384, codes.shape[0] - a), codes.shape[1], dtype)
        c, s = _quantise(x, code)
        codes[a:a + 16384].copy_(c)
        scales[a:a + 16384].copy_(s)


def prepare(case, seed):
    g, op, dt = _gen(seed), case["op"], TYPES[case["dtype"]]
    s = {"case": case}
    if op in ("kv_write", "kv_read"):
        h2 = 2 * case["kv_heads"]
        s["raw"], s["codes"], s["scales"] = _pool_views(case["pool"], h2, case["code"])
        s["slots"] = torch.randperm(case["pool"], generator=g, device=DEV)[:case["tokens"]]
        if op == "kv_write":
            s["kv"] = _rows_like_kv(g, case["tokens"], h2, dt)
        else:
            _fill_pool(g, s["codes"], s["scales"], case["code"], dt)
    elif op == "decode":
        b, hq, hkv, top = case["batch"], case["q_heads"], case["kv_heads"], case["max_len"]
        lens = torch.randint(case["min_len"], top + 1, (b,), generator=g, device=DEV)
        lens[0] = top
        total = int(lens.sum())
        s["raw"], s["codes"], s["scales"] = _pool_views(total + 3, 2 * hkv, case["code"])
        _fill_pool(g, s["codes"], s["scales"], case["code"], dt)
        s["table"] = torch.full((b + 1, top + 2), 2147483647, dtype=torch.int32, device=DEV)
        perm = torch.randperm(total + 3, generator=g, device=DEV).to(torch.int32)
        s["rows"] = torch.randperm(b + 1, generator=g, device=DEV)[:b].to(torch.int32)
        at = 0
        for i, n in enumerate(lens.tolist()):
            s["table"][int(s["rows"][i]), :n] = perm[at:at + n]
            at += n
        s["lens"] = lens.to(torch.int32)
        s["q"] = (1.5 * torch.randn(b, hq, D, generator=g, device=DEV)).to(dt)
    elif op == "norm":
        t, h = case["tokens"], case["hidden"]
        s["x"] = torch.randn(t, h, generator=g, device=DEV).to(dt)
        s["residual"] = (2.0 * torch.randn(t, h, generator=g, device=DEV)).to(dt)
        s["weight"] = (1.0 + 0.1 * torch.randn(h, generator=g, device=DEV)).to(dt)
        s["eps"] = 1e-5
    elif op == "silu":
        s["io"] = (1.5 * torch.randn(case["tokens"], 2 * case["ffn"], generator=g, device=DEV)).to(dt)
    else:
        t, k, n = case["tokens"], case["in"], case["out"]
        s["a"], s["a_scale"] = _quantise(torch.randn(t, k, generator=g, device=DEV), "int8")
        s["w"], s["w_scale"] = _quantise(0.02 * torch.randn(n, k, generator=g, device=DEV), "int8")
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return _RUN[state["case"]["op"]](state)


def _run_kv_write(s):
    if own:
        from loongserve_b200 import kv_ops
        kv_ops.destindex_copy_quantize_kv(s["kv"], s["slots"], s["codes"], s["scales"])
        back = kv_ops.gather_dequantize_kv(s["codes"], s["scales"], s["slots"], s["kv"].dtype)
    else:
        c, sc = _quantise(s["kv"], s["case"]["code"])
        s["codes"].view(torch.uint8)[s["slots"]] = c.view(torch.uint8)
        s["scales"][s["slots"]] = sc
        back = _read(s, s["kv"].dtype)
    return {"values": back, "scales": s["scales"]}


def _read(s, dtype):
    c = s["codes"].view(torch.uint8)[s["slots"]].view(s["codes"].dtype)
    return (c.float() * s["scales"][s["slots"]].unsqueeze(-1)).to(dtype)


def _run_kv_read(s):
    dtype = TYPES[s["case"]["dtype"]]
    if own:
        from loongserve_b200 import kv_ops
        return kv_ops.gather_dequantize_kv(s["codes"], s["scales"], s["slots"], dtype)
    return _read(s, dtype)


def _run_decode(s):
    hkv, top = s["case"]["kv_heads"], s["case"]["max_len"]
    codes, scales = s["codes"], s["scales"]
    if own:
        from loongserve_b200 import flash_decoding
        return flash_decoding.token_decode_attention_q8(
            s["q"], codes[:, :hkv], scales[:, :hkv], codes[:, hkv:], scales[:, hkv:], s["table"], s["rows"], s["lens"], top)
    b, hq = s["q"].shape[:2]
    mask = torch.arange(top, device=DEV)[None] >= s["lens"][:, None]                       # [b, top]: past the request's end
    slots = s["table"][s["rows"].long()][:, :top].long().masked_fill(mask, 0)
    kv = codes.view(torch.uint8)[slots].view(codes.dtype).float() * scales[slots].unsqueeze(-1)        # [b, top, 2*hkv, D]
    k, v = kv[:, :, :hkv].permute(0, 2, 1, 3), kv[:, :, hkv:].permute(0, 2, 1, 3)          # [b, hkv, top, D]
    q = s["q"].float().view(b, hkv, hq // hkv, D)
    x = (q @ k.transpose(-1, -2)) * (D ** -0.5)
    x = x.masked_fill(mask[:, None, None], -math.inf)
    top_x = x.amax(-1, keepdim=True)
    at = torch.where(torch.isinf(top_x), torch.zeros_like(top_x), top_x)
    p = torch.exp(x - at)
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (at + torch.log(total)).view(b, hq)
    return o.reshape(b, hq, D).to(s["q"].dtype), lse


def _values(codes, scale, dtype):
    return (codes.float() * scale.unsqueeze(-1)).to(dtype)


def _run_norm(s):
    quant, dt = s["case"]["quant"], s["x"].dtype
    if own:
        from loongserve_b200 import layer_ops
        if not quant:
            return {"out": layer_ops.add_rms_norm(s["x"], s["residual"], s["weight"], s["eps"]), "residual": s["residual"]}
        codes, scale = layer_ops.add_rms_norm_quant(s["x"], s["residual"], s["weight"], s["eps"])
        return {"out": layer_ops.dequantize_rows(codes, scale, dt), "scale": scale, "residual": s["residual"]}
    t = s["x"].float() + s["residual"].float()
    s["residual"].copy_(t.to(dt))
    y = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    if not quant:
        return {"out": y.to(dt), "residual": s["residual"]}
    codes, scale = _quantise(y, "int8")
    return {"out": _values(codes, scale, dt), "scale": scale, "residual": s["residual"]}


def _run_silu(s):
    dt, f = s["io"].dtype, s["case"]["ffn"]
    if own:
        from loongserve_b200 import layer_ops
        codes, scale = layer_ops.silu_and_mul_quant(s["io"])
        return {"out": layer_ops.dequantize_rows(codes, scale, dt), "scale": scale}
    gate, up = s["io"][:, :f].float(), s["io"][:, f:].float()
    codes, scale = _quantise(gate / (1 + torch.exp(-gate)) * up, "int8")
    return {"out": _values(codes, scale, dt), "scale": scale}


def _run_mm(s):
    dt = TYPES[s["case"]["dtype"]]
    if own:
        from loongserve_b200 import layer_ops
        return layer_ops.mm_w8a8(s["a"], s["a_scale"], s["w"], s["w_scale"], out_dtype=dt)
    acc = torch.mm(s["a"].float(), s["w"].float().t())
    return (acc * s["a_scale"][:, None] * s["w_scale"][None]).to(dt)


_RUN = {"kv_write": _run_kv_write, "kv_read": _run_kv_read, "decode": _run_decode, "norm": _run_norm, "silu": _run_silu, "mm": _run_mm}


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Inputs read once, outputs written once (the 8-bit rows of a kv_write, norm or silu pass are what it leaves to the next
    operator: they count as written where the pool keeps them, and the 16-bit values that come back count as written)."""
    op = case["op"]
    if op == "kv_write":
        e = case["tokens"] * 2 * case["kv_heads"]
        return {"bytes": e * (2 * D + D + 4 + 2 * D) + 8 * case["tokens"], "flops": 4 * e * D}
    if op == "kv_read":
        e = case["tokens"] * 2 * case["kv_heads"]
        return {"bytes": e * (D + 4 + 2 * D) + 8 * case["tokens"], "flops": e * D}
    if op == "decode":
        tokens = case["max_len"] + (case["batch"] - 1) * (case["min_len"] + case["max_len"]) // 2
        io = case["batch"] * case["q_heads"] * (4 * D + 4)
        return {"bytes": tokens * (2 * case["kv_heads"] * (D + 4) + 4) + io, "flops": 4 * tokens * case["q_heads"] * D}
    if op == "norm":
        e = case["tokens"] * case["hidden"]
        return {"bytes": 8 * e + 2 * case["hidden"] + (4 * case["tokens"] if case["quant"] else 0), "flops": 5 * e}
    if op == "silu":
        e = case["tokens"] * case["ffn"]
        return {"bytes": 6 * e + 4 * case["tokens"], "flops": 6 * e}
    t, k, n = case["tokens"], case["in"], case["out"]
    return {"bytes": t * k + n * k + 2 * t * n + 4 * (t + n), "flops": 2 * t * k * n}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_rows(x, code):
    """(values, scales) of rows held in 8 bits, x in 64 bits."""
    scale = x.abs().amax(-1, keepdim=True).clamp_min(TINY) / TOP[code]
    t = x / scale
    if code == "int8":
        c = torch.round(t)
    else:                                       # nearest multiple of the binade's step: 3 mantissa bits, smallest step 2^-9
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** -6))) - 3)
        c = torch.round(t / step) * step
    return c * scale, scale.squeeze(-1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "kv_write":
        values = torch.empty(s["kv"].shape, dtype=torch.float64, device=DEV)
        scales = s["scales"].double()
        for a in range(0, case["tokens"], 2048):
            values[a:a + 2048], scales[s["slots"][a:a + 2048]] = _exact_rows(s["kv"][a:a + 2048].double(), case["code"])
        return {"values": values, "scales": scales}
    if op == "kv_read":
        c = s["codes"].view(torch.uint8)[s["slots"]].view(s["codes"].dtype).double()
        return c * s["scales"][s["slots"]].double()[..., None]
    if op == "decode":
        hkv, b, hq = case["kv_heads"], case["batch"], case["q_heads"]
        o = torch.zeros(b, hq, D, dtype=torch.float64, device=DEV)
        lse = torch.full((b, hq), -math.inf, dtype=torch.float64, device=DEV)
        for i, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            slots = s["table"][int(s["rows"][i]), :n].long()
            for h in range(hkv):
                k = s["codes"][:, h].view(torch.uint8)[slots].view(s["codes"].dtype).double() * s["scales"][slots, h].double()[:, None]
                v = s["codes"][:, hkv + h].view(torch.uint8)[slots].view(s["codes"].dtype).double() * s["scales"][slots, hkv + h].double()[:, None]
                heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                x = torch.einsum("gd,nd->gn", s["q"][i, heads].double(), k) / math.sqrt(D)
                lse[i, heads] = torch.logsumexp(x, -1)
                o[i, heads] = torch.einsum("gn,nd->gd", torch.softmax(x, -1), v)
        return o, lse
    if op == "norm":
        t = s["x"].double() + s["residual"].double()
        y = t / torch.sqrt(t.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"].double()
        if not case["quant"]:
            return {"out": y, "residual": t}
        values, scale = _exact_rows(y, "int8")
        return {"out": values, "scale": scale, "residual": t}
    if op == "silu":
        gate, up = s["io"].double().chunk(2, -1)
        values, scale = _exact_rows(gate * torch.sigmoid(gate) * up, "int8")
        return {"out": values, "scale": scale}
    out = torch.empty(case["tokens"], case["out"], dtype=torch.float64, device=DEV)
    w = s["w"].double() * s["w_scale"].double()[:, None]
    for a in range(0, case["tokens"], 2048):
        out[a:a + 2048] = (s["a"][a:a + 2048].double() * s["a_scale"][a:a + 2048].double()[:, None]) @ w.t()
    return out
