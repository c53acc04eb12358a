"""The angle tables of the decoder layer over an int8 cache, which a serving loop asks for with every prompt length."""
import pytest
import torch

from oracle import llama_cpu


@pytest.fixture()
def lay(pkg):
    from dipu_b200 import layer as L
    cfg = llama_cpu.LayerConfig(hidden=256, heads=2, kv_heads=2, head_dim=128, ffn=320, eps=1e-6)
    return L.DecoderLayer(cfg, llama_cpu.make_weights(cfg, seed=1), device="cpu")


class _Cache:
    capacity = 96


def _prompt(n):
    return (torch.empty(n, 2, 128), torch.empty(n, 2, 128))


def _bytes(value, seen):
    """Bytes of all tensor memory that an object's containers hold, each storage once."""
    if isinstance(value, torch.Tensor):
        s = value.untyped_storage()
        n = 0 if s.data_ptr() in seen else s.nbytes()
        seen.add(s.data_ptr())
        return n
    if isinstance(value, dict):
        return sum(_bytes(v, seen) for v in value.values())
    if isinstance(value, (list, tuple)):
        return sum(_bytes(v, seen) for v in value)
    return 0


def test_tables_do_not_grow_with_the_number_of_prompt_lengths(lay):
    first = _bytes(vars(lay), set())
    for n in list(range(1, 300)) + list(range(299, 0, -1)):
        lay._cached_tables(_Cache, _prompt(n))
    # cos and sin for the 395 positions in use, float32 [positions, 64]: four times that leaves room for growing in steps
    assert _bytes(vars(lay), set()) - first <= 4 * 2 * 395 * 64 * 4


def test_tables_hold_the_positions_behind_the_prompt(lay):
    from dipu_b200 import layer as L
    kept = []
    for n in (0, 7, 300, 1, 299):
        cos, sin = lay._cached_tables(_Cache, _prompt(n) if n else None)
        want = L.rope_tables(128, torch.arange(n, n + 96), lay.rope_base, "cpu")
        assert torch.equal(cos, want[0]) and torch.equal(sin, want[1])
        for t in (cos, sin):
            assert t.is_contiguous() and t.data_ptr() % 16 == 0
        kept.append((cos, cos.clone()))
    assert all(torch.equal(a, b) for a, b in kept)   # a captured step goes on reading the table it was captured with


def test_a_capture_that_fails_leaves_the_layer_as_it_was(lay, monkeypatch):
    """An error inside the step ends the capture, which may fail in turn; later calls must not go on keeping their temporaries."""
    from dipu_b200 import layer as L

    class StepError(Exception):
        pass

    def step(*args):
        raise StepError

    ended = []

    def end(stream):
        ended.append(stream)
        raise RuntimeError("the capture was invalidated")

    monkeypatch.setattr(L.devapis, "graphBeginCapture", lambda stream: None)
    monkeypatch.setattr(L.devapis, "graphEndCapture", end)
    monkeypatch.setattr(lay, "decode_cached", step)
    with pytest.raises((StepError, RuntimeError)):
        lay.capture_decode_cached(None, _Cache, None, None, stream=0)
    assert ended and lay._keep is None
