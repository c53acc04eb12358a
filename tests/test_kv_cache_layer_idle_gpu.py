"""Idle sequences and places past the cache in the decode step behind a shared prompt: nothing that the step did not write shows."""
import math

import pytest
import torch

from test_kv_cache_layer_gpu import BF, DEV, _layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("behind_prompt", [True, False])
def test_sequences_that_are_not_written_take_nothing_from_old_memory(pkg, captured, behind_prompt):
    """Fresh memory holds NaN here. Sequence 1 is idle, sequence 2 past its cache: the same, finite, rows whatever was in memory."""
    from dipu_b200 import layer as L
    _, _, lay = _layer(L, 4, 2, 128)
    g = torch.Generator().manual_seed(4)
    x = torch.randn((4, 512), generator=g).mul(0.5).to(BF).to(DEV)
    prompt = torch.randn((21, 512), generator=g).mul(0.5).to(BF).to(DEV)
    pos, lens = torch.tensor([3, -1, 8, 0], device=DEV), torch.tensor([4, 0, 8, 1], device=DEV)
    stream = torch.cuda.ExternalStream(pkg.devapis.getDefaultStream(0), device=DEV)
    torch.cuda.synchronize()
    empty, got = lay._empty, []
    with torch.cuda.stream(stream):
        prefix = lay.prefix_kv(prompt) if behind_prompt else None
        lay.decode_cached(x, L.QuantKVCache(4, 2, 8, 128, DEV), pos, lens, prefix)
        for fill in (math.nan, 3.0):
            def poisoned(*shape, dtype=None):
                t = empty(*shape, dtype=dtype)
                return t.fill_(fill) if t.is_floating_point() else t
            cache = L.QuantKVCache(4, 2, 8, 128, DEV)
            lay._empty = poisoned
            if captured:
                replay, out = lay.capture_decode_cached(x, cache, pos, lens, prefix, stream.cuda_stream)
                replay()
                got.append(out.clone())
                pkg.devapis.syncStream(stream.cuda_stream)
                pkg.devapis.graphDestroy(replay.graph)
            else:
                got.append(lay.decode_cached(x, cache, pos, lens, prefix).clone())
            lay._empty = empty
    torch.cuda.synchronize()
    assert got[0].isfinite().all() and torch.equal(got[0], got[1])
