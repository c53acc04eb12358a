"""The ends of the value range in the operators on key / value caches: rows near the largest bf16."""
import pytest
import torch

from test_kv_cache_gpu import BF, DEV, FP, _check_write, _randn

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
