"""The measured cases of the KV-cache operators: writing a quantised cache and reading it back, decode attention over caches of
ragged lengths, and decode attention of a batch that shares a prompt.

`run` computes a case either in its plain form (elementary torch operations in fp32, rounded once) or, where `own` is true,
through the library's entry points (include/diopi/functions_b200.h). Caches are [batch, kv heads, capacity, dim], int8 with
one fp32 scale per row (`quant`) or in the model's type.
"""
import math

import torch

own = False

DEV = "cuda:0"
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases ---------------------------------------------------------------------------------------------------------------
def _cache(name, dtype, B, S, Hq, Hkv, D, rot, L, interleaved=False, idle=0):
    c = dict(op="cache", dtype=dtype, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, rot=rot, L=L, interleaved=interleaved, idle=idle)
    return dict(c, name=name) if name else c


def _decode(name, dtype, B, Hq, Hkv, D, L, lo, hi, quant=True, idle=0):
    c = dict(op="decode", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, lo=lo, hi=hi, quant=quant, idle=idle)
    return dict(c, name=name) if name else c


def _prefix(name, dtype, B, Hq, Hkv, D, P, L, lo, hi, quant=True, idle=0):
    c = dict(op="prefix", dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, D=D, P=P, L=L, lo=lo, hi=hi, quant=quant, idle=idle)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of one sequence, a small model: pure latency
        _cache("cache-step-1", "bf16", 1, 1, 8, 8, 64, 64, 512),
        # the decode step of a 32-head layer at batch 64, sequences at different positions
        _cache("cache-step-64", "bf16", 64, 1, 32, 32, 128, 128, 4096),
        # eight prompts of 2048 tokens written at once (the prefill of the same layer)
        _cache("cache-prompt-16k", "bf16", 8, 2048, 32, 32, 128, 128, 2112),
        # a chunk of odd length into the middle of the cache, grouped heads, half of the head rotated in interleaved pairs
        _cache("cache-chunk-odd", "fp16", 5, 333, 64, 8, 128, 64, 1500, interleaved=True, idle=1),
        # one short sequence of a small model: latency
        _decode("decode-1-short", "bf16", 1, 8, 8, 64, 512, 300, 300),
        # batch 64 at 4096 keys, every head with its own keys: the largest read
        _decode("decode-64x4096", "bf16", 64, 32, 32, 128, 4096, 4096, 4096),
        # a serving batch: grouped heads, lengths from one token to the whole capacity, idle slots in between
        _decode("decode-ragged", "fp16", 48, 64, 8, 128, 16384, 1, 16384, idle=4),
        # one long document, grouped heads: the keys have to be spread over the whole GPU
        _decode("decode-long-1", "bf16", 1, 64, 8, 128, 131072, 131071, 131071),
        # the cache kept in the model's type, ragged odd lengths
        _decode("decode-model-type", "bf16", 16, 32, 32, 128, 4096, 17, 3999, quant=False),
        # three short answers behind a short prompt: latency
        _prefix("prefix-3-short", "bf16", 3, 8, 8, 64, 97, 64, 1, 33),
        # 64 answers behind one prompt of 4096 tokens, every head with its own keys
        _prefix("prefix-64", "bf16", 64, 32, 32, 128, 4096, 1024, 1, 1024),
        # 256 answers behind a document of 32768 tokens, grouped heads: bound by the products over the prefix
        _prefix("prefix-256", "bf16", 256, 64, 8, 128, 32768, 1024, 16, 1024),
    ]


_HEADS = ((8, 8), (32, 32), (64, 8), (32, 8), (16, 1), (24, 8), (8, 4), (10, 2), (48, 2), (7, 1))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("cache", "decode", "decode", "prefix", "prefix"))
    dtype = rng.choice(("bf16", "fp16"))
    Hq, Hkv = rng.choice(_HEADS)
    D = rng.choice((64, 128, 128))
    if op == "cache":
        tokens = _log(rng, 1, max(1, (16384 * 96) // (Hq + 2 * Hkv)))
        B = min(_log(rng, 1, 128), tokens)
        S = rng.choice((1, max(1, tokens // B)))
        L = S + _log(rng, 1, 2048)
        return _cache(None, dtype, B, S, Hq, Hkv, D, rng.choice((D, D, D // 2, D // 4)), L, rng.random() < 0.5, rng.choice((0, 0, B // 5)))
    quant = rng.random() < 0.7
    B = _log(rng, 1, 256)
    most = (1 << 30) // (1 if quant else 2) // (B * Hkv * D)
    if op == "decode":
        L = _log(rng, 1, min(most, 131072))
        hi = _log(rng, 1, L)
        return _decode(None, dtype, B, Hq, Hkv, D, L, _log(rng, 1, hi), hi, quant, rng.choice((0, 0, B // 5)))
    L = _log(rng, 1, min(most, 4096))
    hi = _log(rng, 1, L)
    P = _log(rng, 1, min(65536, (256 * 64 * 128 * 32768) // (B * Hq * D)))
    return _prefix(None, dtype, B, Hq, Hkv, D, P, L, _log(rng, 1, hi), hi, quant, rng.choice((0, 0, B // 5)))


def _lengths(case):
    """Lengths of the batch's sequences: evenly spread from lo to hi, the first `idle` ones empty. Their order is the seed's."""
    B, lo, hi, idle = case["B"], case["lo"], case["hi"], case["idle"]
    n = B - idle
    return [0] * idle + [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def work(case):
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    if case["op"] == "cache":
        t = (B - case["idle"]) * case["S"]
        q, kv, rows = t * Hq * D, 2 * t * Hkv * D, 2 * t * Hkv
        # in: q / k / v in two bytes; out: q, codes and scales; the read-back reads codes and scales and writes two bytes each
        return {"bytes": 2 * (q + kv) + 2 * q + (kv + 4 * rows) + (kv + 4 * rows) + 2 * kv, "flops": 3 * q + 7 * kv}
    keys = sum(_lengths(case))
    row = (D + 4) if case["quant"] else 2 * D
    shared = case.get("P", 0)
    return {"bytes": 2 * keys * Hkv * row + 2 * shared * Hkv * 2 * D + 2 * 2 * B * Hq * D + 4 * B * Hq,
            "flops": 4 * Hq * D * (keys + B * shared)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _codes(shape, g):
    """An int8 cache as a writer leaves it: rows of normal values at different magnitudes, codes up to +-127, a scale per row."""
    codes = torch.empty(shape, dtype=torch.int8, device=DEV)
    for b in range(shape[0]):
        x = torch.randn(shape[1:], generator=g, device=DEV, dtype=torch.float16)
        x.mul_(127.0 / x.abs().amax(-1, keepdim=True))
        codes[b] = x.round_().to(torch.int8)
    scale = torch.exp(torch.randn(shape[:-1], generator=g, device=DEV) * 0.3) * 0.02
    return codes, scale


def prepare(case, seed):
    g = _generator(seed)
    dt = _TYPES[case["dtype"]]
    B, Hq, Hkv, D, L = (case[k] for k in ("B", "Hq", "Hkv", "D", "L"))
    order = torch.randperm(B, generator=g, device=DEV)
    if case["op"] == "cache":
        S, rot = case["S"], case["rot"]
        qkv = torch.randn((B, S, (Hq + 2 * Hkv) * D), generator=g, device=DEV).to(dt)
        inv = 1.0 / 10000.0 ** (torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
        angle = torch.outer(torch.arange(L, device=DEV, dtype=torch.float64), inv)
        start = torch.tensor([-1] * case["idle"] + [(L - S) - (L - S) * i // max(1, B - case["idle"] - 1) for i in range(B - case["idle"])], device=DEV)[order]
        return {"case": case, "qkv": qkv, "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float(), "positions": start,
                "q_out": torch.zeros((B, S, Hq, D), dtype=dt, device=DEV),
                "k_cache": torch.zeros((B, Hkv, L, D), dtype=torch.int8, device=DEV), "k_scale": torch.zeros((B, Hkv, L), device=DEV),
                "v_cache": torch.zeros((B, Hkv, L, D), dtype=torch.int8, device=DEV), "v_scale": torch.zeros((B, Hkv, L), device=DEV),
                "k_back": torch.zeros((B, S, Hkv, D), dtype=dt, device=DEV), "v_back": torch.zeros((B, S, Hkv, D), dtype=dt, device=DEV)}
    s = {"case": case, "q": torch.randn((B, Hq, D), generator=g, device=DEV).to(dt), "lengths": torch.tensor(_lengths(case), device=DEV)[order]}
    if case["quant"]:
        s["k_cache"], s["k_scale"] = _codes((B, Hkv, L, D), g)
        s["v_cache"], s["v_scale"] = _codes((B, Hkv, L, D), g)
    else:
        s["k_cache"], s["v_cache"] = (torch.randn((B, Hkv, L, D), generator=g, device=DEV, dtype=dt) for _ in range(2))
        s["k_scale"] = s["v_scale"] = None
    if case["op"] == "prefix":
        s["prefix_k"], s["prefix_v"] = (torch.randn((case["P"], Hkv, D), generator=g, device=DEV, dtype=dt) for _ in range(2))
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, rot, interleaved):
    """x [B, S, H, D] in fp32, cos / sin [B, S, 1, rot / 2]: the first `rot` values of a head in pairs, the others as they are."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)
    a, b = r[..., : rot // 2], r[..., rot // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)


def _quantise(x):
    scale = x.abs().amax(-1) / 127.0
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x / safe.unsqueeze(-1)).clamp(-127, 127), scale


def _plain_cache(s):
    c = s["case"]
    B, S, Hq, Hkv, D, L, rot = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "L", "rot"))
    slot = s["positions"][:, None] + torch.arange(S, device=DEV)
    valid = (s["positions"][:, None] >= 0) & (slot < L)
    slot = slot.clamp(0, L - 1)
    x = s["qkv"].float().view(B, S, Hq + 2 * Hkv, D)
    cos, sin = s["cos"][slot].unsqueeze(2), s["sin"][slot].unsqueeze(2)
    rotated = _rotate(x[:, :, : Hq + Hkv], cos, sin, rot, c["interleaved"])
    live = valid[:, :, None, None]
    s["q_out"].copy_(torch.where(live, rotated[:, :, :Hq].to(s["q_out"].dtype), s["q_out"]))
    rows = torch.arange(B, device=DEV)[:, None].expand(B, S)
    for new, codes, scales, back in ((rotated[:, :, Hq:], "k_cache", "k_scale", "k_back"), (x[:, :, Hq + Hkv:], "v_cache", "v_scale", "v_back")):
        code, scale = _quantise(new)
        s[codes][rows, :, slot] = torch.where(live, code.to(torch.int8), s[codes][rows, :, slot])
        s[scales][rows, :, slot] = torch.where(live[..., 0], scale, s[scales][rows, :, slot])
        got = s[codes][rows, :, slot].float() * s[scales][rows, :, slot].unsqueeze(-1)
        s[back].copy_(torch.where(live, got.to(s[back].dtype), s[back]))
    return {k: s[k] for k in ("q_out", "k_scale", "v_scale", "k_back", "v_back")}


def _plain_attention(s):
    c = s["case"]
    B, Hq, Hkv, D, L = (c[k] for k in ("B", "Hq", "Hkv", "D", "L"))
    g = Hq // Hkv
    q = s["q"].float().view(B, Hkv, g, D)
    k, v = s["k_cache"].float(), s["v_cache"].float()
    if c["quant"]:
        k.mul_(s["k_scale"].unsqueeze(-1))
        v.mul_(s["v_scale"].unsqueeze(-1))
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)
    del k
    unseen = torch.arange(L, device=DEV) >= s["lengths"][:, None, None, None]
    score.masked_fill_(unseen, -math.inf)
    top = score.amax(-1, keepdim=True)
    if "prefix_k" in s:
        P = c["P"]
        rows = q.permute(1, 0, 2, 3).reshape(Hkv, B * g, D)
        shared = torch.matmul(rows, s["prefix_k"].float().permute(1, 2, 0)) / math.sqrt(D)          # [Hkv, B g, P]
        top = torch.maximum(top, shared.amax(-1).view(Hkv, B, g, 1).transpose(0, 1))
    base = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = score.sub_(base).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v)
    del v, p, score
    if "prefix_k" in s:
        p = shared.view(Hkv, B, g, P).sub_(base.transpose(0, 1)).exp_()
        total = total + p.sum(-1, keepdim=True).transpose(0, 1)
        out = out + torch.matmul(p.view(Hkv, B * g, P), s["prefix_v"].float().transpose(0, 1)).view(Hkv, B, g, D).transpose(0, 1)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = base + torch.log(total)
    return {"out": out.to(s["q"].dtype).view(B, Hq, D), "lse": lse.view(B, Hq)}


# ---- the library's entry points --------------------------------------------------------------------------------------------------
_lib = None


def _library():
    """The operator binding and a context on torch's current stream, as a serving loop keeps them."""
    global _lib
    if _lib is None:
        import __graft_entry__ as entry
        diopi = entry.load_package().diopi
        _lib = diopi, diopi.Context()
    return _lib


def _own_cache(s):
    diopi, ctx = _library()
    cache = (s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"])
    diopi.diopiB200RopeQuantAppendKV(ctx, s["q_out"], s["qkv"], s["cos"], s["sin"], s["positions"], *cache, s["case"]["interleaved"])
    diopi.diopiB200DequantKV(ctx, s["k_back"], s["v_back"], *cache, s["positions"])
    return {k: s[k] for k in ("q_out", "k_scale", "v_scale", "k_back", "v_back")}


def _own_attention(s):
    diopi, ctx = _library()
    q = s["q"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    cache = (s["k_cache"], s["k_scale"], s["v_cache"], s["v_scale"], s["lengths"], 1.0 / math.sqrt(q.shape[2]))
    if "prefix_k" in s:
        diopi.diopiB200SharedPrefixAttention(ctx, out, lse, q, s["prefix_k"], s["prefix_v"], *cache)
    else:
        diopi.diopiB200CachedAttention(ctx, out, lse, q, *cache)
    ctx.release_workspace()
    return {"out": out, "lse": lse}


def run(state):
    if state["case"]["op"] == "cache":
        return _own_cache(state) if own else _plain_cache(state)
    return _own_attention(state) if own else _plain_attention(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_cache(case, s):
    B, S, Hq, Hkv, D, L, rot = (case[k] for k in ("B", "S", "Hq", "Hkv", "D", "L", "rot"))
    half = rot // 2
    out = {k: s[k].double() for k in ("q_out", "k_scale", "v_scale", "k_back", "v_back")}
    first = torch.arange(half, device=DEV)
    i, j = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + half)
    for b, start in enumerate(s["positions"].tolist()):
        if start < 0:
            continue
        n = min(S, L - start)
        x = s["qkv"][b, :n].double().view(n, Hq + 2 * Hkv, D)
        z = torch.polar(torch.ones((n, 1, half), dtype=torch.float64, device=DEV),
                        torch.atan2(s["sin"][start:start + n].double(), s["cos"][start:start + n].double()).unsqueeze(1))
        z = z * torch.hypot(s["sin"][start:start + n].double(), s["cos"][start:start + n].double()).unsqueeze(1)
        y = x.clone()
        turned = torch.complex(x[..., i], x[..., j])[:, : Hq + Hkv] * z
        y[:, : Hq + Hkv, i], y[:, : Hq + Hkv, j] = turned.real, turned.imag
        out["q_out"][b, :n] = y[:, :Hq]
        for at, scales, back in ((Hq, "k_scale", "k_back"), (Hq + Hkv, "v_scale", "v_back")):
            rows = y[:, at:at + Hkv]
            step = rows.abs().max(-1).values / 127
            out[scales][b, :, start:start + n] = step.T
            whole = torch.round(rows / torch.where(step == 0, 1.0, step).unsqueeze(-1))
            out[back][b, :n] = whole * step.unsqueeze(-1)
    return out


def _exact_attention(case, s):
    B, Hq, Hkv, D = (case[k] for k in ("B", "Hq", "Hkv", "D"))
    g = Hq // Hkv
    out = torch.zeros((B, Hkv, g, D), dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hkv, g), -math.inf, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(B, Hkv, g, D)
    pk = pv = None
    if case["op"] == "prefix":
        pk, pv = s["prefix_k"].double().transpose(0, 1).contiguous(), s["prefix_v"].double().transpose(0, 1).contiguous()
    for b, n in enumerate(s["lengths"].tolist()):
        k, v = s["k_cache"][b, :, :n].double(), s["v_cache"][b, :, :n].double()
        if case["quant"]:
            k, v = k * s["k_scale"][b, :, :n, None].double(), v * s["v_scale"][b, :, :n, None].double()
        score = q[b] @ k.transpose(1, 2)
        if pk is not None:
            score = torch.cat([q[b] @ pk.transpose(1, 2), score], dim=-1)
        if score.shape[-1] == 0:
            continue
        score = score * D ** -0.5
        lse[b] = torch.logsumexp(score, dim=-1)
        p = torch.exp(score - lse[b].unsqueeze(-1))
        if pk is None:
            out[b] = p @ v
        else:
            out[b] = p[..., : pk.shape[1]] @ pv + p[..., pk.shape[1]:] @ v
    return {"out": out.view(B, Hq, D), "lse": lse.view(B, Hq)}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_cache(case, s) if case["op"] == "cache" else _exact_attention(case, s)
