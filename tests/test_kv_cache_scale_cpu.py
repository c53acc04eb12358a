"""A softmax scale that single precision cannot hold is refused like one that is not a number."""
import pytest

from test_kv_cache_cpu import _attention_args, _prefix_args, _refused


@pytest.mark.parametrize("scale", [1e39, 3e38, 1e-46, 1e-39])
@pytest.mark.parametrize("entry,args", [("diopiB200CachedAttention", _attention_args), ("diopiB200SharedPrefixAttention", _prefix_args)])
def test_scales_out_of_single_precision(diopi, entry, args, scale):
    """It is used times log2(e), as a normal float32."""
    _refused(diopi, entry, {**args(), "scale": scale}, "scale leaves float32's range")
