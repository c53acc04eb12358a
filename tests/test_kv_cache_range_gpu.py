"""The ends of the value range in the operators on key / value caches: rows near the largest bf16, probabilities far below the
largest one, value rows of very different magnitudes, infinities among the values.

Tolerance of the attention (u = eps / 2, half a step of a type; p the exact softmax, A = sum p |v|, n the keys of a part). A probability is
held for the second product
  over int8 rows              as fp16, its products p vs lifted so that a column's largest one lies at 2^6 or more: relative 2^-11 (bf16
                              results), 2^-22 (fp16 results: two terms), and 2^-25 / 2^6 of the largest product where it is subnormal
  over rows in bf16           in two terms, 2^-16, bf16 having fp32's range
  over rows in fp16           in two terms, 2^-22, the largest one lifted to 2^7: 2^-25 / 2^7 of the largest probability
  over a shared prompt        in one term, 2^-8 (bf16) or 2^-11 (fp16, and 2^-32 of the largest probability).
Scores carry the fp32 sums' D 2^-24 relative to S = scale sum |q k|, in numerator and denominator, exponentials and sums 2^-20; the
second product's fp32 sums 2^-22 A for each of a warp's n / 16 steps and the 64 of the joins; the result is rounded once.
"""
import math

import pytest
import torch

from test_kv_cache_gpu import BF, DEV, FP, HALF, _check_write, _randn

pytestmark = pytest.mark.gpu


# ---- the writer ------------------------------------------------------------------------------------------------------------------
def _huge(shape, seed):
    """Rows whose largest magnitudes lie between 2^125 and the largest bf16 (2^128 less one part in 256)."""
    x = _randn(shape, seed).clamp(-3, 3)
    top = torch.exp2(torch.linspace(125.0, 127.9, shape[-2]))[:, None]
    return (x / x.abs().amax(-1, keepdim=True) * top).to(BF)


@pytest.mark.parametrize("B,S", [(2, 3), (2, 1400)])
def test_write_rows_near_the_largest_bf16(pkg, ctx, B, S):
    """Both thread widths; without a rotation (which may leave fp32's range)."""
    Hq, Hkv, D = 4, 10, 64
    x = _huge((B, S, Hq + 2 * Hkv, D), 5).view(B, S, (Hq + 2 * Hkv) * D)
    assert (B * S * (Hq + 2 * Hkv) >= 65536) == (S > 3)
    cache, _, _ = _check_write(pkg, ctx, B, S, Hq, Hkv, D, 0, S, False, BF, [0] * B, x=x)
    k, v = (torch.empty(B, S, Hkv, D, dtype=BF, device=DEV) for _ in range(2))
    pkg.diopi.diopiB200DequantKV(ctx, k, v, *cache.args, None)
    torch.cuda.synchronize()
    for out, c, s in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        assert torch.equal(out, (c.float() * s[..., None]).to(BF).transpose(1, 2))


@pytest.mark.parametrize("inter", [False, True])
def test_write_rotated_rows_near_the_largest_bf16(pkg, ctx, inter):
    x = _huge((2, 3, 4 + 2 * 10, 128), 6) * 0.5
    _check_write(pkg, ctx, 2, 3, 4, 10, 128, 128, 9, inter, BF, [2, 5], x=x.view(2, 3, -1))


def test_write_without_key_heads(pkg, ctx):
    """A rank or a model part that only turns queries: no key heads, an empty cache."""
    _check_write(pkg, ctx, 2, 3, 4, 0, 64, 64, 8, False, BF, [1, 4])
    _check_write(pkg, ctx, 2, 3, 4, 0, 128, 64, 8, True, FP, [-1, 6])


# ---- attention --------------------------------------------------------------------------------------------------------------------
def _run(pkg, ctx, q, cache, lengths, scale, prefix=None):
    out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device=DEV)
    lens = torch.tensor(lengths, dtype=torch.int64, device=DEV)
    if prefix is None:
        pkg.diopi.diopiB200CachedAttention(ctx, out, lse, q, *cache, lens, scale)
    else:
        pkg.diopi.diopiB200SharedPrefixAttention(ctx, out, lse, q, *prefix, *cache, lens, scale)
    torch.cuda.synchronize()
    ctx.release_workspace()
    assert pkg.diopi.gemm_status() == 0
    return out, lse


def _exact(q, cache, b, h, n, scale, prefix=None):
    """In 64 bits for the query heads of key head h of sequence b: scores [g, keys], k, v, value scales of the own keys."""
    kc, ks, vc, vs = cache
    k, v = kc[b, h, :n].double(), vc[b, h, :n].double()
    if ks is not None:
        k, v = k * ks[b, h, :n, None].double(), v * vs[b, h, :n, None].double()
    if prefix is not None:
        k, v = torch.cat([prefix[0][:, h].double(), k]), torch.cat([prefix[1][:, h].double(), v])
    g = q.shape[1] // kc.shape[1]
    rows = q[b, h * g:(h + 1) * g].double()
    return rows, k, v, scale * (rows @ k.T)


def _hold(pkg, ctx, q, cache, lengths, scale, prefix=None, sequences=None):
    out, lse = _run(pkg, ctx, q, cache, lengths, scale, prefix)
    dtype, (B, Hq, D), Hkv, quant = q.dtype, q.shape, cache[0].shape[1], cache[1] is not None
    P, g = 0 if prefix is None else prefix[0].shape[0], Hq // Hkv
    for b in range(B) if sequences is None else sequences:
        n = lengths[b]
        for h in range(Hkv):
            rows, k, v, s = _exact(q, cache, b, h, n, scale, prefix)
            if k.shape[0] == 0:
                assert (out[b, h * g:(h + 1) * g] == 0).all()
                continue
            wlse = torch.logsumexp(s, -1)
            p = torch.exp(s - wlse[:, None])
            want, A = p @ v, p @ v.abs()
            S = (scale * (rows.abs() @ k.abs().T)).amax(-1, keepdim=True)
            slack = 2 * D * 2.0 ** -24 * S + 2.0 ** -20
            tol = slack * A + (k.shape[0] / 16 + 64) * 2.0 ** -22 * A + HALF[dtype] * want.abs() + (2.0 ** -25 if dtype is FP else 0.0)
            if P:
                tol = tol + HALF[dtype] * (p[:, :P] @ v[:P].abs())
                if dtype is FP:
                    tol = tol + P * 2.0 ** -32 * p[:, :P].amax(-1, keepdim=True) * v[:P].abs().amax(0)
            if n:
                po, vo = p[:, P:], v[P:]
                two = dtype is FP or not quant
                tol = tol + ((2.0 ** -16 if dtype is BF and not quant else 2.0 ** -22) if two else 2.0 ** -11) * (po @ vo.abs())
                if quant:
                    tol = tol + n * 2.0 ** -31 * 127 * (po * cache[3][b, h, :n].double().abs()).amax(-1, keepdim=True)
                elif dtype is FP:
                    tol = tol + n * 2.0 ** -32 * po.amax(-1, keepdim=True) * vo.abs().amax(0)
            err = (out[b, h * g:(h + 1) * g].double() - want).abs()
            assert (err <= tol).all(), (b, h, n, (err / tol).max().item())
            lerr = (lse[b, h * g:(h + 1) * g].double() - wlse).abs()
            assert (lerr <= slack[:, 0] + 2.0 ** -22 * wlse.abs()).all(), (b, h, n, lerr.max().item())
    return out


def _codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(DEV)


def _scales(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.exp(torch.randn(shape, generator=g) * 0.5) * 0.012).to(DEV)


def _cache(quant, dtype, B, Hkv, L, D, seed=3):
    if quant:
        return [_codes((B, Hkv, L, D), seed), _scales((B, Hkv, L), seed + 1), _codes((B, Hkv, L, D), seed + 2), _scales((B, Hkv, L), seed + 3)]
    return [_randn((B, Hkv, L, D), seed, dtype).to(DEV), None, _randn((B, Hkv, L, D), seed + 2, dtype).to(DEV), None]


KINDS = [(True, BF), (True, FP), (False, BF), (False, FP)]


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (14, 2, 64), (16, 1, 128), (24, 1, 128)])
@pytest.mark.parametrize("quant,dtype", KINDS)
def test_probabilities_in_two_terms(pkg, ctx, quant, dtype, Hq, Hkv, D):
    """Whole segments and pieces, held to the bound of two terms."""
    for L, lengths in ((300, [300, 0, 1, 77]), (900, [900, 640, 17, 65])):
        _hold(pkg, ctx, _randn((4, Hq, D), 1, dtype).to(DEV), _cache(quant, dtype, 4, Hkv, L, D), lengths, D ** -0.5)


def _two_groups(quant, dtype, B, n):
    """Sequence b: even keys have score 0, odd ones 8 t = -(b + 1) / 16; the values of the two groups cancel, and all keys of a group
    have the same probability, so that its rounding does not average out. q, cache, t."""
    D = 64
    q = torch.ones((B, 1, D), dtype=dtype, device=DEV)
    odd = torch.arange(n, device=DEV) % 2 == 1
    t = -(torch.arange(B, device=DEV) + 1) / 128.0
    if quant:
        k, v = (torch.full((B, 1, n, D), 64, dtype=torch.int8, device=DEV) for _ in range(2))
        v[:, :, odd] = -37
        ks = torch.where(odd, t[:, None, None] / 64, torch.zeros((), device=DEV))
        vs = torch.where(odd, 0.01 * 64 / 37 * torch.exp(-8 * t)[:, None, None], torch.full((), 0.01, device=DEV))
        return q, [k, ks, v, vs], t
    k = torch.where(odd[None, None, :, None], t[:, None, None, None], torch.zeros((), device=DEV)).expand(B, 1, n, D)
    v = torch.where(odd[None, None, :, None], -torch.exp(-8 * t)[:, None, None, None], torch.ones((), device=DEV)).expand(B, 1, n, D)
    return q, [k.to(dtype).contiguous(), None, v.to(dtype).contiguous(), None], t


@pytest.mark.parametrize("quant,dtype", [(True, FP), (False, BF), (False, FP)])
@pytest.mark.parametrize("n", [256, 600])
def test_one_term_would_show(pkg, ctx, quant, dtype, n):
    q, cache, _ = _two_groups(quant, dtype, 12, n)
    _hold(pkg, ctx, q, cache, [n] * 12, 0.125)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("quant", [True, False])
def test_probabilities_behind_a_prompt(pkg, ctx, quant, dtype):
    prefix = [_randn((300, 2, 128), 8 + i, dtype).to(DEV) for i in range(2)]
    _hold(pkg, ctx, _randn((3, 8, 128), 1, dtype).to(DEV), _cache(quant, dtype, 3, 2, 600, 128), [600, 0, 33], 128 ** -0.5, prefix)


def _towards(q, nats, scale):
    """A key row along the first query head of every key head, whose score is about `nats`; the other rows of q are made equal to it."""
    return q.float() * (nats / (scale * q.float().pow(2).sum(-1, keepdim=True)))


def _sink_case(quant, dtype, n, nats, at, vscale, D=128):
    """One key head and query head: every key has score 0 but those `at`, `nats` above; their value rows are `vscale` times the others'.
    The values are positive and the small probabilities alike, so that their roundings do not cancel."""
    scale = D ** -0.5
    q = _randn((1, 1, D), 1, dtype).to(DEV)
    row = _towards(q[0, 0], nats, scale)
    cache = _cache(quant, dtype, 1, 1, n, D)
    cache[0].zero_()
    cache[2].abs_()
    if quant:
        cache[3].fill_(0.012)
        step = row.abs().max() / 127
        cache[0][0, 0, at] = torch.round(row / step).to(torch.int8)
        cache[1][0, 0, at] = step
        cache[3][0, 0, at] *= vscale
    else:
        cache[0][0, 0, at] = row.to(dtype)
        cache[2][0, 0, at] *= vscale
    return q, cache, [n], scale


@pytest.mark.parametrize("quant,dtype", KINDS)
@pytest.mark.parametrize("at", [0, 1500, 2900])
@pytest.mark.parametrize("nats", [12.0, 15.0])
def test_many_keys_behind_sink_keys(pkg, ctx, quant, dtype, at, nats):
    """A sink in each quarter of a unit of 64 keys holds most of the weight and has a tiny value row: the result is the sum of the other,
    small, probabilities. 640 sequences read the same cache, so that whole sequences fall to one CTA."""
    q, cache, lengths, scale = _sink_case(quant, dtype, 3000, nats, [at, at + 16, at + 32, at + 48], 1e-6 if quant or dtype is BF else 1e-3)
    cache = [None if t is None else t.expand(640, *t.shape[1:]) for t in cache]
    _hold(pkg, ctx, q.expand(640, 1, 128), cache, lengths * 640, scale, sequences=(0, 319, 639))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("at", [0, 300, 999])
@pytest.mark.parametrize("nats,vscale", [(-40.0, 1e6), (-60.0, 1e5), (-20.0, 1e6), (60.0, 1e-7)])
def test_one_value_row_of_another_magnitude(pkg, ctx, dtype, at, nats, vscale):
    """The magnitude of a value row whose key has no weight must not cost the others their bits."""
    _hold(pkg, ctx, *_sink_case(True, dtype, 1000, nats, [at], vscale))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("L", [400, 900])
def test_query_heads_that_see_values_of_different_magnitudes(pkg, ctx, dtype, L):
    """Two query heads share a key head; each looks at its own half of the keys, whose values are 10^6 apart."""
    D, scale = 64, 64 ** -0.5
    q = torch.zeros((1, 2, D), device=DEV)
    q[0, 0, :32], q[0, 1, 32:] = 1.0, 1.0
    cache = _cache(True, dtype, 1, 1, L, D)
    half = torch.arange(L, device=DEV) % 2 == 0
    cache[0][0, 0] = torch.where(half[:, None] == (torch.arange(D, device=DEV) < 32), 100, -100).to(torch.int8)
    cache[1].fill_(0.03)
    cache[3][0, 0] *= torch.where(half, 1e-3, 1e3)
    _hold(pkg, ctx, q.to(dtype), cache, [L], scale)


@pytest.mark.parametrize("mag", [1e-34, 1e-20, 1e20, 1e33])
def test_value_rows_of_any_magnitude(pkg, ctx, mag):
    cache = _cache(True, BF, 2, 2, 700, 128)
    cache[3] *= mag
    _hold(pkg, ctx, _randn((2, 4, 128), 1, BF).to(DEV), cache, [700, 333], 128 ** -0.5)


def test_value_rows_near_the_largest_bf16(pkg, ctx):
    """One key of that size: its weight times its row stays in range, as does a score that grows towards it."""
    cache = _cache(True, BF, 1, 1, 600, 128)
    cache[0][:] = torch.linspace(0, 100, 600, device=DEV).to(torch.int8)[:, None]
    cache[1].fill_(0.01)
    cache[3].fill_(1e30)
    cache[3][0, 0, 599] = 3.3e38 / 127
    q = torch.full((1, 2, 128), 0.5, dtype=BF, device=DEV)
    _hold(pkg, ctx, q, cache, [600], 0.1)


def test_value_magnitudes_that_grow_and_fall(pkg, ctx):
    for dtype in (BF, FP):
        for flip in (False, True):
            cache = _cache(True, dtype, 2, 2, 700, 64)
            ramp = torch.logspace(-3, 3, 700, device=DEV)
            cache[3] *= ramp.flip(0) if flip else ramp
            _hold(pkg, ctx, _randn((2, 4, 64), 1, dtype).to(DEV), cache, [700, 401], 0.125)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("at", [0, 700, 1499])
def test_many_prompt_rows_behind_a_sink_row(pkg, ctx, dtype, at):
    """160 key heads, so that a CTA takes all rows of one, or most of them."""
    H = 160
    q, cache, _, scale = _sink_case(False, dtype, 1500, 15.0, [at], 1e-3)
    prefix = [t[0, 0, :, None].expand(1500, H, 128).contiguous() for t in (cache[0], cache[2])]
    own = _cache(True, dtype, 1, 1, 40, 128)
    own[0].zero_()
    for n in (0, 40):
        _hold(pkg, ctx, q.expand(1, H, 128), [t.expand(1, H, *t.shape[2:]) for t in own], [n], scale, prefix)


# ---- infinities among the values ----------------------------------------------------------------------------------------------------
def _same(out, want):
    """Infinities and NaN where the definition has them; the rest is the other tests' business."""
    assert torch.equal(out.isnan(), want.isnan()), (int(out.isnan().sum()), int(want.isnan().sum()))
    assert torch.equal(out.double().nan_to_num(0, 1e300, -1e300).abs() == 1e300, want.nan_to_num(0, 1e300, -1e300).abs() == 1e300)
    inf = want.isinf()
    assert torch.equal(out[inf].double(), want[inf])
    err = (out[~inf & ~want.isnan()].double() - want[~inf & ~want.isnan()]).abs()
    assert (err <= 0.02 * (1 + want[~inf & ~want.isnan()].abs())).all()


@pytest.mark.parametrize("quant,dtype", KINDS)
@pytest.mark.parametrize("L", [130, 700])
@pytest.mark.parametrize("P", [0, 150])
def test_infinite_values(pkg, ctx, quant, dtype, L, P):
    """An infinity in a visible value row gives an infinity of its sign (NaN beside one of the other sign), also at the last key of a
    ragged sequence and at a key of hardly any weight; one behind the sequence gives nothing."""
    B, Hq, Hkv, D = 3, 6, 2, 128
    q = _randn((B, Hq, D), 1, dtype).to(DEV)
    cache = _cache(quant, dtype, B, Hkv, L, D)
    lengths = [L, 77, 3]
    if quant:
        cache[3] *= 0.2
        cache[3][0, 0, 5] = math.inf
        cache[3][1, 1, 76] = math.inf
        cache[3][2, :, 3:] = math.inf
    else:
        v = cache[2]
        v[0, 0, 5, 7] = v[0, 0, L - 1, 9] = math.inf
        v[0, 0, 11, 20] = -math.inf
        v[0, 1, 2, 3], v[0, 1, 60, 3] = math.inf, -math.inf
        v[1, 0, 76, 1] = v[1, 1, 30, 2] = -math.inf
        v[2, :, 3:] = math.inf
        cache[0][1, 1, 30] = _towards(q[1, 3], -60.0, D ** -0.5).to(dtype)
    prefix = None
    if P:
        prefix = [_randn((P, Hkv, D), 8 + i, dtype).to(DEV) for i in range(2)]
        prefix[1][P - 1, 0, 40], prefix[1][3, 1, 50] = math.inf, -math.inf
        prefix[0][3, 1] = _towards(q[2, 4], -60.0, D ** -0.5).to(dtype)
    out, lse = _run(pkg, ctx, q, cache, lengths, D ** -0.5, prefix)
    g = Hq // Hkv
    for b in range(B):
        for h in range(Hkv):
            _, _, v, s = _exact(q, cache, b, h, lengths[b], D ** -0.5, prefix)
            p = torch.softmax(s, -1)
            want = (p[:, :, None] * v[None]).sum(1)
            _same(out[b, h * g:(h + 1) * g], want)
    assert lse.isfinite().all()


@pytest.mark.parametrize("quant", [True, False])
@pytest.mark.parametrize("L", [300, 900])
@pytest.mark.parametrize("P", [0, 150])
def test_sums_of_values_near_the_largest_bf16(pkg, ctx, quant, L, P):
    """Their sum leaves fp32 before it is divided; the result does not."""
    cache = _cache(quant, BF, 2, 2, L, 128)
    if quant:
        cache[3].fill_(3.3e38 / 127)
    else:
        cache[2][:] = (cache[2].float().clamp(-3, 3) * 1.1e38).to(BF)
    prefix = [_randn((P, 2, 128), 8 + i, BF).to(DEV) for i in range(2)] if P else None
    out = _hold(pkg, ctx, _randn((2, 4, 128), 1, BF).to(DEV), cache, [L, L // 2], 128 ** -0.5, prefix)
    assert out.isfinite().all()
