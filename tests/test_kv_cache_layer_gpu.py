"""The decoder layer over an int8 cache: chunks of a prompt, ragged decode steps, a shared prompt, one captured step replayed for many
tokens - the cache operators as they are used together, against the layer's formulas in plain fp32 on the CPU."""
import math

import pytest
import torch

from oracle import llama_cpu

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def _layer(L, heads, kv_heads, d, layout="half", seed=3):
    cfg = llama_cpu.LayerConfig(hidden=512, heads=heads, kv_heads=kv_heads, head_dim=d, ffn=1376, eps=1e-6, rope_layout=layout)
    w = llama_cpu.make_weights(cfg, seed=seed)
    return cfg, llama_cpu.round_weights(w, BF), L.DecoderLayer(cfg, w, dtype=BF, device=DEV)


def _quantised(y):
    """A row as the int8 cache holds it."""
    scale = y.abs().amax(-1, keepdim=True) / 127
    return torch.round(y / scale.clamp_min(1e-30)) * scale


def _token(cfg, w, x, keys, vals, place):
    """One token of one sequence in fp32: x [hidden], keys / vals [n, Hkv, D] lists of cached rows (appended to)."""
    d, hq, hk = cfg.head_dim, cfg.heads, cfg.kv_heads
    hn = llama_cpu.rms_norm(x[None], w["attention_norm"], cfg.eps)
    cos, sin = llama_cpu.rope_tables(d, torch.tensor([place]))
    def turn(t, h):
        return llama_cpu.rotary(cfg, t.view(1, h, d), cos, sin).view(h, d)
    q, k = turn(hn @ w["wq"].T, hq), turn(hn @ w["wk"].T, hk)
    keys.append(_quantised(k))
    vals.append(_quantised((hn @ w["wv"].T).view(hk, d)))
    kk, vv = (torch.stack(t).repeat_interleave(hq // hk, dim=1) for t in (keys, vals))
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, kk) / math.sqrt(d), -1)
    h = x + (torch.einsum("hn,nhd->hd", p, vv).reshape(1, -1) @ w["wo"].T)[0]
    hn = llama_cpu.rms_norm(h[None], w["ffn_norm"], cfg.eps)
    return h + ((torch.nn.functional.silu(hn @ w["w1"].T) * (hn @ w["w3"].T)) @ w["w2"].T)[0]


def _near(got, want):
    """The layer bound against fp32 that the other layer tests use, 1e-2 and 2e-2, plus what a code that falls the other way moves: the
    bf16 rounding of a projection can move a row's values by a step of 1 / 127 of its maximum, 1 / 254 on average over keys."""
    got = got.float().cpu()
    rel = ((got - want).norm() / want.norm()).item()
    assert (got - want).abs().max().item() <= 3e-2 and rel <= 1e-2 + 1 / 254, ((got - want).abs().max().item(), rel)


@pytest.mark.parametrize("heads,kv_heads,d,layout", [(8, 8, 64, "interleaved"), (4, 2, 128, "half")])
def test_ragged_decode_steps(pkg, heads, kv_heads, d, layout):
    """Sequences that start at different times, one idle throughout."""
    from dipu_b200 import layer as L
    cfg, w, lay = _layer(L, heads, kv_heads, d, layout)
    B, steps = 5, 9
    begin = [0, 3, 99, 1, 6]          # the step at which a sequence starts; 99: idle
    cache = L.QuantKVCache(B, kv_heads, 16, d, DEV)
    xs = torch.randn((steps, B, 512), generator=torch.Generator().manual_seed(1)).mul(0.5).to(BF)
    keys, vals = [[] for _ in range(B)], [[] for _ in range(B)]
    for t in range(steps):
        pos = torch.tensor([t - s if t >= s else -1 for s in begin], device=DEV)
        y = lay.decode_cached(xs[t].to(DEV), cache, pos, pos + 1)
        torch.cuda.synchronize()
        for b in range(B):
            if t >= begin[b]:
                _near(y[b], _token(cfg, w, xs[t, b].float(), keys[b], vals[b], t - begin[b]))
    assert (cache.k[2] == 0).all() and (cache.k_scale[2] == 0).all() and pkg.diopi.gemm_status() == 0


def test_chunked_prompt_then_decode_behind_a_shared_prompt(pkg):
    """A shared prompt, two chunks of every sequence's own prompt, decode steps from one captured graph."""
    from dipu_b200 import layer as L
    cfg, w, lay = _layer(L, 4, 2, 128)
    B, P, chunks, steps = 3, 37, (20, 13), 4
    g = torch.Generator().manual_seed(2)
    xp = torch.randn((P, 512), generator=g).mul(0.5).to(BF)
    xs = torch.randn((B, sum(chunks) + steps, 512), generator=g).mul(0.5).to(BF)
    stream = torch.cuda.ExternalStream(pkg.devapis.getDefaultStream(0), device=DEV)
    torch.cuda.synchronize()
    got = torch.zeros_like(xs, dtype=torch.float32)
    with torch.cuda.stream(stream):
        prefix = lay.prefix_kv(xp.to(DEV))
        cache = L.QuantKVCache(B, 2, 64, 128, DEV)
        at = 0
        for n in chunks:
            y = lay.prefill_cached(xs[:, at:at + n].reshape(B * n, 512).to(DEV), B, n, cache, at, prefix)
            got[:, at:at + n] = y.view(B, n, 512).float().cpu()
            at += n
        pos = torch.full((B,), at, device=DEV)
        lens = pos + 1
        x = xs[:, at].to(DEV)
        got[:, at] = lay.decode_cached(x, cache, pos, lens, prefix).float().cpu()
        replay, out = lay.capture_decode_cached(x, cache, pos, lens, prefix, stream.cuda_stream)
        for t in range(at + 1, at + steps):
            x.copy_(xs[:, t])
            pos.add_(1)
            lens.add_(1)
            replay()
            got[:, t] = out.float().cpu()
        pkg.devapis.graphDestroy(replay.graph)
    torch.cuda.synchronize()
    assert pkg.diopi.gemm_status() == 0
    pk, pv = (t.float().cpu() for t in prefix)
    cos, sin = llama_cpu.rope_tables(128, torch.arange(P))
    hn = llama_cpu.rms_norm(xp.float(), w["attention_norm"], cfg.eps)
    want_k = llama_cpu.rotary(cfg, (hn @ w["wk"].T).view(P, 2, 128), cos, sin)
    assert ((pk - want_k).norm() / want_k.norm()).item() <= 1e-2
    for b in range(B):
        keys, vals = list(pk), list(pv)
        for t in range(xs.shape[1]):
            _near(got[b, t], _token(cfg, w, xs[b, t].float(), keys, vals, P + t))


def test_more_sequences_than_the_fused_tail_serves(pkg):
    """Above 128 rows the feed-forward block runs op by op; the same rows give the same result either way."""
    from dipu_b200 import layer as L
    cfg, w, lay = _layer(L, 4, 4, 128)
    x = torch.randn((130, 512), generator=torch.Generator().manual_seed(5)).mul(0.5).to(BF)
    pos = torch.zeros(130, dtype=torch.int64, device=DEV)
    y = lay.decode_cached(x.to(DEV), L.QuantKVCache(130, 4, 4, 128, DEV), pos, pos + 1)
    torch.cuda.synchronize()
    for b in (0, 64, 129):
        _near(y[b], _token(cfg, w, x[b].float(), [], [], 0))


def test_layer_refuses(pkg):
    from dipu_b200 import layer as L
    _, _, lay = _layer(L, 8, 8, 64)
    with pytest.raises(AssertionError, match="head dim 128"):
        lay.prefill_cached(torch.zeros(4, 512, dtype=BF, device=DEV), 2, 2, L.QuantKVCache(2, 8, 8, 64, DEV))
    _, _, lay = _layer(L, 4, 2, 128)
    with pytest.raises(AssertionError, match="of a cache of 8"):
        lay.prefill_cached(torch.zeros(18, 512, dtype=BF, device=DEV), 2, 9, L.QuantKVCache(2, 2, 8, 128, DEV))
