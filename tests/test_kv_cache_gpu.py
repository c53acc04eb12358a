"""The int8 key / value cache and decode attention over ragged caches, with and without a shared prompt, against plain 64-bit
restatements of their formulas.

Tolerances. u = eps / 2 is half a step of the type (bf16 2^-8, fp16 2^-11 relative).
Rotation: two products and a sum in fp32, each off by at most 2^-24 relative to |a| + |b| (|cos|, |sin| <= 1): 3 * 2^-24 (|a| + |b|).
Codes: |y - code * scale| <= 0.5 scale, plus 127 * 2^-22 of a step for the roundings of 127 / max|y|, y and the scale.
Attention: a probability is rounded once to the operand type of the second product (u relative; fp16 for int8 caches, with a floor
of 2^-24 of the largest value for probabilities that are subnormal there), scores carry the fp32 sums' D * 2^-24 relative to
scale * sum |q k| (doubled: the maximum is subtracted), exp2 and the fp32 sums 2^-20, and the result is rounded once:
  |error| <= u_p A + A (2 D 2^-24 S + 2^-20) + n 2^-24 max|v| + u |out|,   A = sum p |v| / sum p,  S = max_j scale sum |q k_j|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -11}


def _randn(shape, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _tables(rows, rot):
    inv = 1.0 / 10000.0 ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.outer(torch.arange(rows, dtype=torch.float64), inv)
    return torch.cos(a).float(), torch.sin(a).float()


def _rotate(x, cos, sin, rot, interleaved):
    """x [..., D] float64, cos / sin [..., rot / 2]: rotated values, and |a| + |b| of every value's pair."""
    y, mag = x.clone(), x.abs()
    half = rot // 2
    i = torch.arange(half) * 2 if interleaved else torch.arange(half)
    j = i + 1 if interleaved else i + half
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * cos - b * sin, b * cos + a * sin
    mag = mag.clone()
    mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return y, mag


class Cache:
    """A cache on the device whose storage is wider than its views, filled with a pattern that must survive."""

    def __init__(self, B, Hkv, L, D, pad=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        def codes():
            return torch.randint(-127, 128, (B, Hkv, L + pad, D), generator=g, dtype=torch.int8).to(DEV)
        def scales():
            return torch.rand((B, Hkv, L + pad), generator=g).to(DEV)
        self.full = [codes(), scales(), codes(), scales()]
        self.before = [t.clone() for t in self.full]
        self.k, self.ks, self.v, self.vs = (t[:, :, :L] for t in self.full)
        self.args = (self.k, self.ks, self.v, self.vs)


def _check_write(pkg, ctx, B, S, Hq, Hkv, D, rot, L, inter, dtype, positions, seed=1, x=None, table_rows=None, two_d=False, pad=0):
    C = (Hq + 2 * Hkv) * D
    x = _randn((B, S, C), seed, dtype) if x is None else x
    rows = table_rows or L
    cos, sin = _tables(rows, rot) if rot else (None, None)
    cache = Cache(B, Hkv, L, D, pad, seed)
    q = torch.full((B, S, Hq, D), 7.0, dtype=dtype, device=DEV) if Hq else None
    pos = torch.tensor(positions, dtype=torch.int64, device=DEV)
    xd, qd = x.to(DEV), q
    if two_d:
        xd, qd = xd[:, 0], q[:, 0]
    pkg.diopi.diopiB200RopeQuantAppendKV(ctx, qd, xd, cos.to(DEV) if rot else None, sin.to(DEV) if rot else None, pos, *cache.args, inter)
    torch.cuda.synchronize()
    want = [t.clone().cpu() for t in cache.before]
    got = [t.cpu() for t in cache.full]
    xs = x.double().view(B, S, Hq + 2 * Hkv, D)
    for b in range(B):
        for s in range(S):
            slot = positions[b] + s
            if positions[b] < 0 or slot >= L or (rot and slot >= rows):
                if Hq:
                    assert (q[b, s] == 7.0).all()
                continue
            y, mag = xs[b, s], xs[b, s].abs()
            if rot:
                yr, mr = _rotate(y[:Hq + Hkv], cos[slot].double(), sin[slot].double(), rot, inter)
                y, mag = torch.cat([yr, y[Hq + Hkv:]]), torch.cat([mr, mag[Hq + Hkv:]])
            if Hq:
                err = (q[b, s].cpu().double() - y[:Hq]).abs()
                assert (err <= HALF[dtype] * y[:Hq].abs() + 4 * 2.0 ** -24 * mag[:Hq] + 2.0 ** -25).all()
            for i, at in ((0, Hq), (2, Hq + Hkv)):
                rows_y, rows_m = y[at:at + Hkv], mag[at:at + Hkv]
                code, scale = got[i][b, :, slot].double(), got[i + 1][b, :, slot].double()
                top = rows_y.abs().amax(-1)
                assert ((scale - top / 127).abs() <= 2.0 ** -22 * rows_m.amax(-1) / 127 + 2.0 ** -149).all()
                assert (code.abs() <= 127).all() and ((code.abs().amax(-1) == 127) | (top < 1e-35)).all()
                err = (code * scale[:, None] - rows_y).abs()
                assert (err <= (0.5 + 127 * 2.0 ** -22) * scale[:, None] + 4 * 2.0 ** -24 * rows_m + 2.0 ** -149 * 127).all()
                want[i][b, :, slot], want[i + 1][b, :, slot] = got[i][b, :, slot], got[i + 1][b, :, slot]
    for g, w in zip(got, want):
        assert torch.equal(g, w)   # no other slot changed
    return cache, pos, q


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,L,inter", [
    (1, 1, 8, 8, 64, 64, 40, False), (3, 1, 4, 2, 128, 128, 33, True), (2, 7, 5, 1, 128, 64, 19, False), (2, 5, 3, 3, 64, 32, 9, True),
    (4, 2, 2, 1, 128, 16, 6, False), (2, 3, 0, 2, 64, 64, 8, False), (2, 3, 4, 2, 128, 0, 8, False), (1, 200, 6, 2, 128, 32, 256, True)])
def test_write(pkg, ctx, dtype, B, S, Hq, Hkv, D, rot, L, inter):
    g = torch.Generator().manual_seed(B * 100 + S)
    positions = torch.randint(0, L - S + 1, (B,), generator=g).tolist()
    cache, pos, _ = _check_write(pkg, ctx, B, S, Hq, Hkv, D, rot, L, inter, dtype, positions, pad=3)
    k, v = (torch.full((B, S, Hkv, D), 3.0, dtype=dtype, device=DEV) for _ in range(2))
    pkg.diopi.diopiB200DequantKV(ctx, k, v, *cache.args, pos)
    torch.cuda.synchronize()
    for b in range(B):
        sl = slice(positions[b], positions[b] + S)
        for out, c, s in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):   # an fp32 product rounded once: bit for bit
            assert torch.equal(out[b], (c[b, :, sl].float() * s[b, :, sl, None]).to(dtype).transpose(0, 1))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot,L,inter", [(2, 300, 97, 9, 128, 128, 310, False), (3, 200, 65, 23, 64, 32, 205, True), (1, 520, 96, 16, 128, 64, 530, True),
                                                      (2, 400, 0, 42, 64, 16, 402, False)])
def test_write_many_rows(pkg, ctx, dtype, B, S, Hq, Hkv, D, rot, L, inter):
    """From 65536 rows on a thread takes 16 values."""
    assert B * S * (Hq + 2 * Hkv) >= 65536
    _check_write(pkg, ctx, B, S, Hq, Hkv, D, rot, L, inter, dtype, [3, L - S, -1][:B] if B > 1 else [7], pad=1)


def test_write_one_token_two_dimensional(pkg, ctx):
    _check_write(pkg, ctx, 5, 1, 4, 2, 128, 128, 12, False, BF, [3, 11, 0, 7, 7], two_d=True)


def test_write_idle_and_past_the_end(pkg, ctx):
    """Negative positions are idle; tokens behind the cache or the tables are skipped, also for positions near 2^63."""
    _check_write(pkg, ctx, 6, 4, 3, 1, 64, 64, 10, False, BF, [-1, 8, 10, 2 ** 62, -2 ** 62, 0])
    _check_write(pkg, ctx, 3, 4, 3, 1, 64, 64, 10, True, FP, [2 ** 63 - 1, 5, -2 ** 63], table_rows=7)


def test_write_rows_of_zeros_and_tiny_rows(pkg, ctx):
    x = _randn((2, 4, 4 * 64), 3, BF)
    x[0, 0] = 0
    x[0, 1] *= 1e-31
    x[0, 2] *= 1e-36
    x[0, 3] = 0
    x[0, 3, ::5] = 9.2e-41      # the smallest bf16 magnitude: its scale underflows to zero
    x[1, 0] *= 1e35
    x[1, 1, 1:] = 0
    cache, _, _ = _check_write(pkg, ctx, 2, 4, 2, 1, 64, 0, 4, False, BF, [0, 0], x=x)
    assert (cache.ks[0, :, 0] == 0).all() and (cache.k[0, :, 0] == 0).all()


def test_write_rows_that_are_not_finite_read_back_as_nan(pkg, ctx):
    x = _randn((4, 1, 4 * 128), 3, FP)
    x[0, 0, 2 * 128 + 5] = math.inf       # in k
    x[1, 0, 2 * 128 + 127] = math.nan
    x[2, 0, 3 * 128] = -math.inf          # in v
    cos, sin = (t.to(DEV) for t in _tables(4, 128))
    cache = Cache(4, 1, 4, 128)
    q = torch.empty(4, 1, 2, 128, dtype=FP, device=DEV)
    pos = torch.zeros(4, dtype=torch.int64, device=DEV)
    pkg.diopi.diopiB200RopeQuantAppendKV(ctx, q, x.to(DEV), cos, sin, pos, *cache.args, False)
    k, v = (torch.empty(4, 1, 1, 128, dtype=FP, device=DEV) for _ in range(2))
    pkg.diopi.diopiB200DequantKV(ctx, k, v, *cache.args, None)
    torch.cuda.synchronize()
    assert [bool(t.isnan().all()) for t in k] == [True, True, False, False] and [bool(t.isnan().all()) for t in v] == [False, False, True, False]
    assert not k[2:].isnan().any() and not v[3].isnan().any() and not v[:2].isnan().any()


def test_read_back_windows(pkg, ctx):
    """No positions: the first slots; a window that leaves the cache keeps what the outputs held; strided outputs."""
    cache = Cache(3, 2, 9, 64, pad=2)
    buf = torch.full((2, 3, 5, 2, 128), 5.0, dtype=BF, device=DEV)
    k, v = buf[0, ..., :64], buf[1, ..., 64:]
    pos = torch.tensor([6, -1, 2], device=DEV)
    pkg.diopi.diopiB200DequantKV(ctx, k, v, *cache.args, pos)
    torch.cuda.synchronize()
    for out, c, s in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        full = (c.float() * s[..., None]).to(BF).transpose(1, 2)
        assert torch.equal(out[0, :3], full[0, 6:]) and (out[0, 3:] == 5).all() and (out[1] == 5).all() and torch.equal(out[2], full[2, 2:7])
    assert (buf[0, ..., 64:] == 5).all() and (buf[1, ..., :64] == 5).all()
    pkg.diopi.diopiB200DequantKV(ctx, k, v, *cache.args, None)
    torch.cuda.synchronize()
    assert torch.equal(k, (cache.k.float() * cache.ks[..., None]).to(BF).transpose(1, 2)[:, :5])


# ---- attention -----------------------------------------------------------------------------------------------------------------
def _reference(q, k, v, scale):
    """q [g, D], k / v [n, D] float64: out, lse, and the two sums of the tolerance."""
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.full((q.shape[0],), -math.inf, dtype=torch.float64), torch.zeros_like(q), torch.zeros(q.shape[0], 1)
    s = scale * (q @ k.T)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    return p @ v, lse, p @ v.abs(), (scale * (q.abs() @ k.abs().T)).amax(-1, keepdim=True)


def _attend(pkg, ctx, dtype, B, Hq, Hkv, D, L, lengths, quant, P=None, seed=0, qscale=1.0, kscale=None, views=False, scale=None, heads_first=False, poison=True):
    """Runs the operator on random inputs and holds out and lse to the 64-bit formula. Slots behind a sequence's length hold NaN."""
    scale = D ** -0.5 if scale is None else scale
    q = _randn((B, Hq, D), seed + 1, dtype, qscale)
    if quant:
        g = torch.Generator().manual_seed(seed)
        kc, vc = (torch.randint(-127, 128, (B, Hkv, L, D), generator=g, dtype=torch.int8) for _ in range(2))
        ks, vs = (torch.exp(torch.randn((B, Hkv, L), generator=g) * 0.5) * 0.012 for _ in range(2))
        if kscale is not None:
            ks = ks * kscale(L)
        k, v = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    else:
        kc, vc = (_randn((B, Hkv, L, D), seed + 2 + i, dtype) for i in range(2))
        if kscale is not None:
            kc = (kc * kscale(L)[:, None]).to(dtype)
        ks = vs = None
        k, v = kc.double(), vc.double()
    pk, pv = (_randn((P, Hkv, D), seed + 5 + i, dtype) for i in range(2)) if P is not None else (None, None)
    dev = [None if t is None else t.to(DEV) for t in (q, kc, ks, vc, vs, pk, pv)]
    n = [min(max(x, 0), L) for x in lengths]
    if poison:
        for b in range(B):   # what lies behind a sequence must not matter
            for t in (dev[2], dev[4]) if quant else (dev[1], dev[3]):
                t[b, :, n[b]:] = math.nan
    out = torch.full((B, Hq, D), math.nan, dtype=dtype, device=DEV)
    if views:   # q and out as slices of wider buffers, caches with other pitches and order
        wide = torch.zeros((B, Hq + 2, D + 8), dtype=dtype, device=DEV)
        wide[:, 1:-1, :D] = dev[0]
        dev[0] = wide[:, 1:-1, :D]
        out = torch.full((B, Hq + 1, D + 16), math.nan, dtype=dtype, device=DEV)[:, 1:, 16:]
        dev[1], dev[3] = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dev[1], dev[3]))
    if heads_first and P is not None:
        dev[5], dev[6] = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in dev[5:7])
    lse = torch.full((B, Hq), math.nan, device=DEV)
    lens = torch.tensor(lengths, dtype=torch.int64, device=DEV)
    if P is None:
        pkg.diopi.diopiB200CachedAttention(ctx, out, lse, dev[0], *dev[1:5], lens, scale)
    else:
        pkg.diopi.diopiB200SharedPrefixAttention(ctx, out, lse, dev[0], dev[5], dev[6], *dev[1:5], lens, scale)
    torch.cuda.synchronize()
    ctx.release_workspace()
    assert pkg.diopi.gemm_status() == 0
    got, got_lse = out.cpu().double(), lse.cpu().double()
    grp = Hq // Hkv
    for b in range(B):
        for h in range(Hkv):
            kk, vv = k[b, h, :n[b]], v[b, h, :n[b]]
            if P is not None:
                kk, vv = torch.cat([pk[:, h].double(), kk]), torch.cat([pv[:, h].double(), vv])
            rows = slice(h * grp, (h + 1) * grp)
            want, wlse, A, S = _reference(q[b, rows].double(), kk, vv, scale)
            if kk.shape[0] == 0:
                assert (got[b, rows] == 0).all() and (got_lse[b, rows] == -math.inf).all()
                continue
            up = 2.0 ** -11 if quant and not P else HALF[dtype]
            slack = 2 * D * 2.0 ** -24 * S + 2.0 ** -20
            tol = (up + slack) * A + kk.shape[0] * 2.0 ** -24 * vv.abs().max() + HALF[dtype] * want.abs()
            err = (got[b, rows] - want).abs()
            assert (err <= tol).all(), (b, h, n[b], (err / tol).max().item())
            lerr = (got_lse[b, rows] - wlse).abs()
            assert (lerr <= slack[:, 0] + 2.0 ** -22 * wlse.abs()).all(), (b, h, n[b], lerr.max().item())
    return out, lse


HEADS = [(8, 8, 64), (4, 4, 128), (8, 1, 128), (16, 2, 64), (7, 1, 128), (32, 2, 128), (12, 4, 64), (48, 2, 128), (9, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("quant,dtype", [(True, BF), (True, FP), (False, BF), (False, FP)])
def test_cached_attention(pkg, ctx, quant, dtype, Hq, Hkv, D):
    """Lengths around the tile sizes, one token, none, and values outside [0, L], in one batch."""
    _attend(pkg, ctx, dtype, 14, Hq, Hkv, D, 300, [300, 0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 257, 10 ** 12, -5], quant)


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("B,Hq,Hkv,L,lo", [(1, 8, 1, 9001, 9001), (2, 2, 2, 5000, 1), (3, 40, 8, 2049, 2000), (1, 1, 1, 20000, 19999), (40, 8, 4, 700, 1), (700, 2, 1, 530, 0)])
def test_cached_attention_long_and_uneven(pkg, ctx, quant, B, Hq, Hkv, L, lo):
    g = torch.Generator().manual_seed(L)
    _attend(pkg, ctx, BF, B, Hq, Hkv, 128, L, torch.randint(lo, L + 1, (B,), generator=g).tolist(), quant)


@pytest.mark.parametrize("quant", [True, False])
def test_cached_attention_all_empty_and_no_capacity(pkg, ctx, quant):
    _attend(pkg, ctx, BF, 3, 4, 2, 64, 20, [0, 0, 0], quant)
    _attend(pkg, ctx, BF, 2, 4, 2, 64, 0, [0, 5], quant)
    _attend(pkg, ctx, BF, 0, 4, 2, 64, 4, [], quant)


@pytest.mark.parametrize("quant", [True, False])
def test_cached_attention_views(pkg, ctx, quant):
    _attend(pkg, ctx, BF, 3, 8, 2, 128, 200, [200, 77, 3], quant, views=True)


@pytest.mark.parametrize("quant,dtype", [(True, BF), (True, FP), (False, BF)])
def test_cached_attention_growing_scores(pkg, ctx, quant, dtype):
    """Scores that grow along the keys make the running maximum move all the time; ones that fall never move it."""
    _attend(pkg, ctx, dtype, 2, 4, 2, 128, 600, [600, 333], quant, kscale=lambda n: torch.linspace(0.1, 12.0, n))
    _attend(pkg, ctx, dtype, 2, 4, 2, 128, 600, [600, 333], quant, kscale=lambda n: torch.linspace(12.0, 0.1, n))


def test_cached_attention_query_magnitudes(pkg, ctx):
    """Queries far outside and far below fp16's range (the int8 path multiplies in fp16)."""
    for mag in (1e-20, 1e-6, 1e5, 1e12, 1e30):
        _attend(pkg, ctx, BF, 2, 4, 2, 128, 90, [90, 31], True, qscale=mag, scale=128 ** -0.5 / mag)


@pytest.mark.parametrize("quant", [True, False])
def test_cached_attention_not_finite(pkg, ctx, quant):
    """A NaN among the visible keys makes that head's output NaN and no other; an empty sequence ignores its query."""
    B, H, D, L = 3, 2, 64, 70
    q = _randn((B, H, D), 1, BF).to(DEV)
    q[2] = math.nan
    if quant:
        kc, vc = (torch.randint(-127, 128, (B, H, L, D), dtype=torch.int8, device=DEV) for _ in range(2))
        ks, vs = (torch.rand(B, H, L, device=DEV) * 0.01 for _ in range(2))
        ks[0, 1, 30] = math.nan
        vs[1, 0, 69] = math.nan
    else:
        kc, vc = (_randn((B, H, L, D), 2 + i, BF).to(DEV) for i in range(2))
        ks = vs = None
        kc[0, 1, 30, 5] = math.nan
        vc[1, 0, 69] = math.nan
    out, lse = torch.empty_like(q), torch.empty(B, H, device=DEV)
    pkg.diopi.diopiB200CachedAttention(ctx, out, lse, q, kc, ks, vc, vs, torch.tensor([70, 70, 0], device=DEV), 0.125)
    torch.cuda.synchronize()
    ctx.release_workspace()
    assert out[0, 1].isnan().all() and out[1, 0].isnan().all()
    assert not out[0, 0].isnan().any() and not out[1, 1].isnan().any()
    assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_cached_attention_beyond_32_bit_offsets(pkg, ctx):
    """Sequences whose rows lie more than 2^31 elements apart."""
    pitch = 2 ** 31 + 4096
    B, H, L, D = 2, 2, 96, 64
    store = [torch.zeros(pitch + H * L * D, dtype=torch.int8, device=DEV) for _ in range(2)]
    kc, vc = (t.as_strided((B, H, L, D), (pitch, L * D, D, 1)) for t in store)
    small = [torch.randint(-127, 128, (B, H, L, D), dtype=torch.int8, device=DEV) for _ in range(2)]
    kc.copy_(small[0])
    vc.copy_(small[1])
    ks, vs = (torch.rand(B, H, L, device=DEV) * 0.01 for _ in range(2))
    q = _randn((B, 4, D), 1, BF).to(DEV)
    lens = torch.tensor([96, 95], device=DEV)
    outs = []
    for a, b in ((kc, vc), small):
        out = torch.empty_like(q)
        pkg.diopi.diopiB200CachedAttention(ctx, out, None, q, a, ks, b, vs, lens, 0.125)
        outs.append(out)
    x = _randn((B, (4 + 2 * H) * D), 9, BF).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(L, D))
    for a, b in ((kc, vc), small):
        pkg.diopi.diopiB200RopeQuantAppendKV(ctx, torch.empty_like(q), x, cos, sin, lens - 1, a, ks, b, vs, False)
    torch.cuda.synchronize()
    ctx.release_workspace()
    assert torch.equal(*outs) and torch.equal(kc, small[0]) and torch.equal(vc, small[1])


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("P", [1, 127, 128, 300])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_shared_prefix(pkg, ctx, dtype, P, Hq, Hkv, D):
    _attend(pkg, ctx, dtype, 5, Hq, Hkv, D, 70, [70, 0, 1, 33, 64], quant=(P != 127), P=P, heads_first=P == 300)


@pytest.mark.parametrize("quant", [True, False])
def test_shared_prefix_ranges_across_pairs(pkg, ctx, quant):
    """More (key head, 256 query rows) pairs than half the SMs, and than all of them: a CTA's range of blocks crosses from one pair into
    the next, and from pairs with two row tiles into the last one of a head, which has one."""
    _attend(pkg, ctx, BF, 550, 32, 16, 64, 8, [i % 9 for i in range(550)], quant, P=2560)
    _attend(pkg, ctx, FP, 275, 128, 32, 64, 8, [i % 9 for i in range(275)], quant, P=200)
    _attend(pkg, ctx, BF, 265, 80, 80, 128, 8, [i % 9 for i in range(265)], quant, P=300)


@pytest.mark.parametrize("B,Hq,Hkv,D,P", [(70, 8, 4, 128, 500), (300, 2, 2, 64, 130), (33, 16, 1, 128, 1025), (129, 2, 1, 128, 64), (2, 2, 2, 128, 9000)])
@pytest.mark.parametrize("quant", [True, False])
def test_shared_prefix_many_rows(pkg, ctx, quant, B, Hq, Hkv, D, P):
    g = torch.Generator().manual_seed(B)
    _attend(pkg, ctx, BF, B, Hq, Hkv, D, 40, torch.randint(0, 41, (B,), generator=g).tolist(), quant, P=P)


@pytest.mark.parametrize("quant", [True, False])
def test_shared_prefix_without_own_keys_or_without_prefix(pkg, ctx, quant):
    _attend(pkg, ctx, BF, 3, 4, 2, 128, 16, [0, 0, 0], quant, P=200)
    _attend(pkg, ctx, BF, 3, 4, 2, 128, 0, [0, 0, 0], quant, P=200)
    _attend(pkg, ctx, BF, 3, 4, 2, 128, 16, [0, 16, 5], quant, P=0)
    _attend(pkg, ctx, BF, 2, 4, 2, 128, 0, [0, 0], quant, P=0)


def test_shared_prefix_equals_one_cache(pkg, ctx):
    """The prompt as a prefix and the prompt written in front of every sequence's cache are the same attention."""
    B, Hq, Hkv, D, P, n = 6, 8, 2, 128, 150, 50
    q = _randn((B, Hq, D), 1, FP).to(DEV)
    pk, pv = (_randn((P, Hkv, D), 2 + i, FP).to(DEV) for i in range(2))
    k, v = (_randn((B, Hkv, n, D), 4 + i, FP).to(DEV) for i in range(2))
    kk, vv = (torch.cat([a.transpose(0, 1).expand(B, Hkv, P, D), b], 2) for a, b in ((pk, k), (pv, v)))
    lens = torch.tensor([50, 0, 1, 17, 32, 49], device=DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    pkg.diopi.diopiB200SharedPrefixAttention(ctx, a, None, q, pk, pv, k, None, v, None, lens, 0.1)
    pkg.diopi.diopiB200CachedAttention(ctx, b, None, q, kk, None, vv, None, lens + P, 0.1)
    torch.cuda.synchronize()
    ctx.release_workspace()
    # each is off its exact value by u (A + |out|) with A <= max|v|
    assert ((a.double() - b.double()).abs() <= 2 * (2.0 ** -11 * (vv.abs().max().double() + a.double().abs()) + 2.0 ** -14)).all()


@pytest.mark.parametrize("P", [None, 260])
def test_same_bits_every_time_and_on_another_stream(pkg, diopi, P):
    outs = []
    for i in range(3):
        stream = torch.cuda.Stream() if i == 2 else torch.cuda.current_stream()
        c = diopi.Context(stream=stream.cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            outs.append(_attend(pkg, c, BF, 5, 8, 2, 128, 900, [900, 5, 640, 0, 77], True, P=P))
    for o, l in outs[1:]:
        assert torch.equal(o, outs[0][0]) and torch.equal(l, outs[0][1])


@pytest.mark.parametrize("P", [None, 200])
def test_step_replayed_from_a_graph(pkg, diopi, P):
    """A captured write + attention follows positions and lengths that change between replays; two graphs with contexts of their own
    replay on two streams at once."""
    B, Hq, Hkv, D, L = 6, 8, 2, 128, 700
    cos, sin = (t.to(DEV) for t in _tables(L, D))
    pk, pv = (_randn((P, Hkv, D), 7 + i, BF).to(DEV) for i in range(2)) if P else (None, None)

    class Step:
        def __init__(self, seed):
            self.x = _randn((B, (Hq + 2 * Hkv) * D), seed, BF).to(DEV)
            self.cache = Cache(B, Hkv, L, D, seed=seed)
            self.cache.ks.mul_(0.01)
            self.pos = torch.zeros(B, dtype=torch.int64, device=DEV)
            self.len = torch.zeros(B, dtype=torch.int64, device=DEV)
            self.q = torch.zeros(B, Hq, D, dtype=BF, device=DEV)
            self.out = torch.zeros(B, Hq, D, dtype=BF, device=DEV)
            self.lse = torch.zeros(B, Hq, device=DEV)

        def at(self, places):
            self.pos.copy_(torch.tensor(places))
            self.len.copy_(torch.tensor(places) + 1)

        def run(self, ctx):
            diopi.diopiB200RopeQuantAppendKV(ctx, self.q, self.x, cos, sin, self.pos, *self.cache.args, False)
            if P:
                diopi.diopiB200SharedPrefixAttention(ctx, self.out, self.lse, self.q, pk, pv, *self.cache.args, self.len, 0.09)
            else:
                diopi.diopiB200CachedAttention(ctx, self.out, self.lse, self.q, *self.cache.args, self.len, 0.09)

    graphs = []
    for i in range(2):
        stream = torch.cuda.ExternalStream(pkg.devapis.getStreamFromPool(0), device=DEV)
        step = Step(20 + i)
        ctx = diopi.Context(stream=stream.cuda_stream, device=0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step.run(ctx)      # warm-up outside the capture
            stream.synchronize()
            ctx.release_workspace()
            pkg.devapis.graphBeginCapture(ctx.stream)
            step.run(ctx)
            graph = pkg.devapis.graphEndCapture(ctx.stream)
        graphs.append((step, stream, ctx, graph))
    eager = diopi.Context()
    for places in ([699, 0, 3, 320, -1, 77], [5, 640, 64, 63, 62, 1]):
        torch.cuda.synchronize()
        for step, _, _, _ in graphs:
            step.at(places)
        torch.cuda.synchronize()
        for _ in range(3):
            for _, _, ctx, graph in graphs:
                pkg.devapis.graphLaunch(graph, ctx.stream)
        torch.cuda.synchronize()
        for step, _, _, _ in graphs:
            got = step.out.clone(), step.lse.clone()
            step.out.zero_()
            step.run(eager)
            torch.cuda.synchronize()
            eager.release_workspace()
            assert torch.equal(step.out, got[0]) and torch.equal(step.lse, got[1])
    for _, _, _, graph in graphs:
        pkg.devapis.graphDestroy(graph)
