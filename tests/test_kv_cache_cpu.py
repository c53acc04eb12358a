"""What the operators on key / value caches refuse. The checks come before any device work, so the handles here describe host memory
as if it were the device's and no GPU is needed."""
import ctypes

import pytest
import torch

BF, FP, F32, I8, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int64


def _handle(diopi, t):
    """A handle for a host tensor that claims to be a device tensor (unless it is marked as the host's)."""
    h = diopi.Handle(t)
    if not getattr(t, "on_host", False):
        diopi._host.minihostFreeTensor(ctypes.c_void_p(h.ptr))
        shape, stride = ((ctypes.c_int64 * t.dim())(*v) for v in (t.shape, t.stride()))
        h.ptr = diopi._host.minihostMakeTensor(ctypes.c_void_p(t.data_ptr()), t.dim(), shape, stride, diopi.DTYPE[t.dtype], 1, getattr(t, "device_index", 0))
    return h


def _aligned(shape, dtype):
    n = 1
    for s in shape:
        n *= s
    raw = torch.zeros(n * dtype.itemsize + 64, dtype=torch.uint8)
    off = -raw.data_ptr() % 64
    return raw[off:off + n * dtype.itemsize].view(dtype).view(shape)


B, S, HQ, HKV, D, L, P = 2, 3, 4, 2, 64, 16, 8


def _write_args():
    return {"q_out": _aligned((B, S, HQ, D), BF), "qkv": _aligned((B, S, (HQ + 2 * HKV) * D), BF), "cos": _aligned((L, D // 2), F32),
            "sin": _aligned((L, D // 2), F32), "positions": _aligned((B,), I64), "k_cache": _aligned((B, HKV, L, D), I8),
            "k_scale": _aligned((B, HKV, L), F32), "v_cache": _aligned((B, HKV, L, D), I8), "v_scale": _aligned((B, HKV, L), F32), "interleaved": False}


def _attention_args(quant=True):
    t = I8 if quant else BF
    scales = [_aligned((B, HKV, L), F32) for _ in range(2)] if quant else [None, None]
    return {"out": _aligned((B, HQ, D), BF), "softmax_lse": _aligned((B, HQ), F32), "q": _aligned((B, HQ, D), BF), "k_cache": _aligned((B, HKV, L, D), t),
            "k_scale": scales[0], "v_cache": _aligned((B, HKV, L, D), t), "v_scale": scales[1], "lengths": _aligned((B,), I64), "scale": 0.1}


def _prefix_args(quant=True):
    a = _attention_args(quant)
    return {**{k: a[k] for k in ("out", "softmax_lse", "q")}, "prefix_k": _aligned((P, HKV, D), BF), "prefix_v": _aligned((P, HKV, D), BF),
            **{k: a[k] for k in ("k_cache", "k_scale", "v_cache", "v_scale", "lengths", "scale")}}


def _dequant_args():
    a = _write_args()
    return {"k_out": _aligned((B, S, HKV, D), BF), "v_out": _aligned((B, S, HKV, D), BF), "k_cache": a["k_cache"], "k_scale": a["k_scale"],
            "v_cache": a["v_cache"], "v_scale": a["v_scale"], "positions": a["positions"]}


def _host(t):
    t.on_host = True
    return t


def _elsewhere(t):
    t.device_index = 1
    return t


def _off(t):
    """The same shape, one element off its alignment."""
    raw = _aligned((t.numel() + 1,), t.dtype)
    return raw[1:].view(t.shape)


def _refused(diopi, name, args, match):
    ctx = diopi.Context()
    handles = [_handle(diopi, a) if isinstance(a, torch.Tensor) else a for a in args.values()]
    with pytest.raises(diopi.DiopiError, match=match):
        getattr(diopi, name)(ctx, *handles)


_WRITE = [
    ({"k_cache": _aligned((B, HKV, L, D), BF), "v_cache": _aligned((B, HKV, L, D), BF)}, "int8 codes"),
    ({"k_scale": _aligned((B, HKV, L), FP)}, "scales must be float32"),
    ({"v_scale": _aligned((B, HKV, L + 1), F32)}, "scales must be float32"),
    ({"v_cache": _aligned((B, HKV, L + 1, D), I8)}, "same shape"),
    ({"k_cache": _off(_aligned((B, HKV, L, D), I8))}, "16-byte aligned"),
    ({"k_cache": _aligned((B, 1, L, D), I8).expand(B, HKV, L, D)}, "not shared"),
    ({"k_scale": _aligned((B, HKV, L, 2), F32)[..., 0]}, "neighbours"),
    ({"k_cache": _aligned((B, HKV, L, 2 * D), I8)[..., ::2]}, "contiguous"),
    ({"qkv": _aligned((B, S, (HQ + 2 * HKV) * D), F32)}, "bfloat16 or float16|qkv's dtype"),
    ({"qkv": _aligned((B, S, (HQ + HKV) * D), BF)}, "columns"),
    ({"q_out": _aligned((B, S, HQ, D), FP)}, "qkv's dtype"),
    ({"q_out": _aligned((B, S, HQ, 2 * D), BF)[..., ::2]}, "contiguous"),
    ({"q_out": _aligned((B, 1, HQ, D), BF).expand(B, S, HQ, D)}, "pitches"),
    ({"q_out": _aligned((B, HQ, D), BF)}, "q_out must be"),
    ({"positions": _aligned((B,), torch.int32)}, "positions must be"),
    ({"positions": _aligned((B + 1,), I64)}, "positions must be"),
    ({"positions": _host(_aligned((B,), I64))}, "positions must be"),
    ({"cos": None}, "go together"),
    ({"cos": _aligned((L, D), F32), "sin": _aligned((L, D), F32)}, "rotated part"),
    ({"cos": _aligned((L, 3), F32), "sin": _aligned((L, 3), F32)}, "rotated part"),
    ({"cos": _aligned((L, D // 2), BF), "sin": _aligned((L, D // 2), BF)}, "float32 tables"),
    ({"sin": _aligned((L + 1, D // 2), F32)}, "float32 tables"),
    ({"k_cache": _aligned((B, HKV, L, 32), I8), "v_cache": _aligned((B, HKV, L, 32), I8)}, "head dim 64 or 128"),
    ({"k_scale": _host(_aligned((B, HKV, L), F32))}, "live on the device"),
    ({"v_scale": _elsewhere(_aligned((B, HKV, L), F32))}, "one device"),
    ({"positions": _elsewhere(_aligned((B,), I64))}, "one device"),
]


@pytest.mark.parametrize("change,match", _WRITE)
def test_write_refuses(diopi, change, match):
    _refused(diopi, "diopiB200RopeQuantAppendKV", {**_write_args(), **change}, match)


@pytest.mark.parametrize("change,match", [
    ({"k_out": _aligned((B, S, HKV, D), F32), "v_out": _aligned((B, S, HKV, D), F32)}, "bfloat16 or float16"),
    ({"v_out": _aligned((B, S + 1, HKV, D), BF)}, "same shape"),
    ({"k_out": _aligned((B, S, HKV + 1, D), BF), "v_out": _aligned((B, S, HKV + 1, D), BF)}, "outputs must be"),
    ({"k_out": _aligned((B, L + 1, HKV, D), BF), "v_out": _aligned((B, L + 1, HKV, D), BF), "positions": None}, "slots asked"),
    ({"k_out": _aligned((1, S, HKV, D), BF).expand(B, S, HKV, D)}, "pitches"),
    ({"positions": _aligned((2 * B,), I64)[::2]}, "positions must be"),
    ({"k_out": _elsewhere(_aligned((B, S, HKV, D), BF))}, "one device"),
])
def test_read_back_refuses(diopi, change, match):
    _refused(diopi, "diopiB200DequantKV", {**_dequant_args(), **change}, match)


_ATTENTION = [
    ({"q": _aligned((B, HQ, D), F32), "out": _aligned((B, HQ, D), F32)}, "bfloat16 or float16"),
    ({"out": _aligned((B, HQ, D), FP)}, "one dtype"),
    ({"out": _aligned((B, HQ + 2, D), BF)}, "q's shape"),
    ({"out": _aligned((1, HQ, D), BF).expand(B, HQ, D)}, "pitches"),
    ({"q": _aligned((B, HQ, D + 4), BF)[..., :D]}, "pitches"),
    ({"q": _off(_aligned((B, HQ, D), BF))}, "aligned"),
    ({"q": _aligned((B, 3, D), BF), "out": _aligned((B, 3, D), BF), "softmax_lse": None}, "cannot share"),
    ({"q": _aligned((B, HQ, 32), BF), "out": _aligned((B, HQ, 32), BF)}, "head dim"),
    ({"q": _aligned((B + 1, HQ, D), BF), "out": _aligned((B + 1, HQ, D), BF)}, "batch"),
    ({"k_scale": None}, "go together"),
    ({"k_scale": None, "v_scale": None}, "without scales"),
    ({"k_cache": _aligned((B, HKV, L, D), BF), "v_cache": _aligned((B, HKV, L, D), BF)}, "int8 codes"),
    ({"lengths": _aligned((B,), torch.int32)}, "lengths must be"),
    ({"lengths": _host(_aligned((B,), I64))}, "lengths must be"),
    ({"scale": 0.0}, "scale must be positive"),
    ({"scale": float("nan")}, "scale must be positive"),
    ({"scale": float("inf")}, "scale must be positive"),
    ({"softmax_lse": _aligned((B, HQ), BF)}, "softmax_lse"),
    ({"softmax_lse": _aligned((B, 1), F32).expand(B, HQ)}, "softmax_lse"),
    ({"q": _host(_aligned((B, HQ, D), BF))}, "device"),
    ({"v_cache": _elsewhere(_aligned((B, HKV, L, D), I8))}, "one device"),
    ({"softmax_lse": _elsewhere(_aligned((B, HQ), F32))}, "one device"),
]


@pytest.mark.parametrize("entry", ["diopiB200CachedAttention", "diopiB200SharedPrefixAttention"])
@pytest.mark.parametrize("change,match", _ATTENTION)
def test_attention_refuses(diopi, entry, change, match):
    args = _attention_args() if entry == "diopiB200CachedAttention" else _prefix_args()
    _refused(diopi, entry, {**args, **change}, match)


def test_write_and_read_back_refuse_one_tensor_for_k_and_v(diopi):
    a = _write_args()
    _refused(diopi, "diopiB200RopeQuantAppendKV", {**a, "v_cache": a["k_cache"]}, "of their own")
    _refused(diopi, "diopiB200RopeQuantAppendKV", {**a, "v_scale": a["k_scale"]}, "of their own")
    d = _dequant_args()
    _refused(diopi, "diopiB200DequantKV", {**d, "v_out": d["k_out"]}, "two tensors")


def test_attention_refuses_out_that_is_q(diopi):
    a = _attention_args()
    _refused(diopi, "diopiB200CachedAttention", {**a, "out": a["q"]}, "out must not be q")


@pytest.mark.parametrize("change,match", [
    ({"k_cache": _aligned((B, HKV, L, D), FP), "v_cache": _aligned((B, HKV, L, D), FP)}, "q's dtype"),
    ({"k_cache": _off(_aligned((B, HKV, L, D), BF))}, "aligned"),
    ({"v_cache": _aligned((B, HKV, L + 1, D), BF)}, "same shape"),
    ({"k_cache": _aligned((B, HKV, L, D + 4), BF)[..., :D]}, "pitches"),
])
def test_attention_over_the_models_type_refuses(diopi, change, match):
    _refused(diopi, "diopiB200CachedAttention", {**_attention_args(False), **change}, match)


@pytest.mark.parametrize("change,match", [
    ({"prefix_k": None}, "are needed"),
    ({"prefix_v": _aligned((P + 1, HKV, D), BF)}, "prefix_k and prefix_v must be"),
    ({"prefix_k": _aligned((P, HKV + 1, D), BF), "prefix_v": _aligned((P, HKV + 1, D), BF)}, "prefix_k and prefix_v must be"),
    ({"prefix_k": _aligned((P, HKV, D), FP)}, "q's dtype"),
    ({"prefix_k": _aligned((P, 1, D), BF).expand(P, HKV, D)}, "pitches"),
    ({"prefix_k": _aligned((P, HKV, 2 * D), BF)[..., ::2]}, "contiguous"),
    ({"prefix_v": _host(_aligned((P, HKV, D), BF))}, "device"),
    ({"prefix_v": _aligned((P * HKV * 3 * D,), BF).as_strided((P, HKV, D), (2 * D + 24, D, 1))}, "multiple of the other"),
])
def test_prefix_refuses(diopi, change, match):
    _refused(diopi, "diopiB200SharedPrefixAttention", {**_prefix_args(), **change}, match)


def test_binding_arguments(diopi):
    """The binding passes what it is given, and raises for what it cannot pass, with handles and with tensors alike."""
    ctx = diopi.Context()
    a = _attention_args()
    with pytest.raises(diopi.DiopiError, match="must live on the device"):   # host tensors, described as such
        diopi.diopiB200CachedAttention(ctx, *a.values())
    with pytest.raises(TypeError, match="expects 9 arguments"):
        diopi.diopiB200CachedAttention(ctx, *list(a.values())[:-1])
    with pytest.raises(diopi.DiopiError, match="no diopi counterpart"):
        diopi.diopiB200CachedAttention(ctx, *{**a, "q": torch.zeros(1, dtype=torch.complex64)}.values())
    sparse = torch.zeros(2, 2).to_sparse()
    with pytest.raises(diopi.DiopiError):   # no strides
        diopi.diopiB200CachedAttention(ctx, *{**a, "q": sparse}.values())
    with pytest.raises(diopi.DiopiError, match="tensor handle is NULL"):
        diopi.diopiB200CachedAttention(ctx, *{**a, "q": None}.values())
    with pytest.raises((TypeError, ValueError)):
        diopi.diopiB200CachedAttention(ctx, *{**a, "scale": "x"}.values())
    with pytest.raises(AttributeError):
        diopi.diopiB200CachedAttention(ctx, *{**a, "q": 3}.values())
    big = [_handle(diopi, x) if isinstance(x, torch.Tensor) else x for x in a.values()]
    with pytest.raises(diopi.DiopiError, match="scale must be positive, got -0.25"):
        diopi.diopiB200CachedAttention(ctx, *big[:-1], -0.25)
