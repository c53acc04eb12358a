// Attention of one new token per sequence over caches of ragged lengths, with or without a prompt that the batch shares.
//
//   diopiB200CachedAttention        softmax(scale * q K_b^T) V_b, K_b / V_b the first lengths[b] rows of sequence b's cache, which is
//                                   int8 codes with one scale per row (kv_cache.cu) or holds the model's type
//   diopiB200SharedPrefixAttention  the same over the rows of a prompt [P, Hkv, D], stored once, and then the sequence's own rows
//
// One warp per key, one CTA per (sequence, query head): the lanes hold D / 32 values each, every warp keeps a running maximum, sum
// and output, and the four warps are merged through shared memory at the end.
#include <cmath>

#include "device_utils.cuh"
#include "diopi/functions_b200.h"
#include "kv_cache.h"

namespace b200 {
namespace {

struct CachedAttnParams {
    const void* q;
    void* out;
    float* lse;                    // optional [B, Hq]
    int64_t q_sb, q_sh, o_sb, o_sh, lse_sb, lse_sh;
    const void* k;
    const void* v;
    const float* ks;               // NULL: caches in the model's type
    const float* vs;
    int64_t k_sb, k_sh, k_sl, v_sb, v_sh, v_sl, ks_sb, ks_sh, vs_sb, vs_sh;
    const int64_t* lengths;
    int64_t L;
    const void* pk;                // shared rows [P, Hkv, D]
    const void* pv;
    int64_t P, pk_sp, pk_sh, pv_sp, pv_sh;
    int B, Hq, Hkv, group;
    float scale_log2;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) cached_attention_kernel(const CachedAttnParams p) {
    constexpr int N = D / 32;
    __shared__ float red[4][D + 2];
    const int h = blockIdx.x, b = blockIdx.y, hk = h / p.group;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t len = min(max(p.lengths[b], int64_t(0)), p.L);
    float q[N], acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = to_f32(static_cast<const T*>(p.q)[b * p.q_sb + h * p.q_sh + lane * N + i]) * p.scale_log2;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t j = warp; j < p.P + len; j += 4) {
        float kf[N], vf[N], vscale = 1.f, kscale = 1.f;
        const int64_t r = j - p.P;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t e = lane * N + i;
            if (r < 0) {
                kf[i] = to_f32(static_cast<const T*>(p.pk)[j * p.pk_sp + hk * p.pk_sh + e]);
                vf[i] = to_f32(static_cast<const T*>(p.pv)[j * p.pv_sp + hk * p.pv_sh + e]);
            } else if (p.ks != nullptr) {
                kf[i] = static_cast<float>(static_cast<const int8_t*>(p.k)[b * p.k_sb + hk * p.k_sh + r * p.k_sl + e]);
                vf[i] = static_cast<float>(static_cast<const int8_t*>(p.v)[b * p.v_sb + hk * p.v_sh + r * p.v_sl + e]);
            } else {
                kf[i] = to_f32(static_cast<const T*>(p.k)[b * p.k_sb + hk * p.k_sh + r * p.k_sl + e]);
                vf[i] = to_f32(static_cast<const T*>(p.v)[b * p.v_sb + hk * p.v_sh + r * p.v_sl + e]);
            }
        }
        if (r >= 0 && p.ks != nullptr) {
            kscale = p.ks[b * p.ks_sb + hk * p.ks_sh + r];
            vscale = p.vs[b * p.vs_sb + hk * p.vs_sh + r];
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(q[i], kf[i], s);
        s = warp_sum(s) * kscale;
        const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.f : m_new;
        const float f = m == -INFINITY ? 0.f : exp2f(m - base), e = exp2f(s - base);
        m = m_new;
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = acc[i] * f + e * vscale * vf[i];
    }
    if (lane == 0) {
        red[warp][0] = m;
        red[warp][1] = l;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) red[warp][2 + lane * N + i] = acc[i];
    __syncthreads();
    float mm = -INFINITY;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, red[w][0]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    for (int w = 0; w < 4; ++w) ll += red[w][1] * exp2f(red[w][0] - base);
    for (int c = threadIdx.x; c < D; c += 128) {
        float a = 0.f;
        for (int w = 0; w < 4; ++w) a += red[w][2 + c] * exp2f(red[w][0] - base);
        static_cast<T*>(p.out)[b * p.o_sb + h * p.o_sh + c] = from_f32<T>(ll == 0.f ? 0.f : a / ll);
    }
    if (threadIdx.x == 0 && p.lse != nullptr) p.lse[b * p.lse_sb + h * p.lse_sh] = ll == 0.f ? -INFINITY : (base + log2f(ll)) * 0.6931471805599453f;
}

// What both entry points take, checked and gathered. `prefix_k` NULL: no shared rows.
diopiError_t cached_attention(const char* name, diopiContextHandle_t ctx, diopiTensorHandle_t out, diopiTensorHandle_t softmax_lse, diopiConstTensorHandle_t q,
                              diopiConstTensorHandle_t prefix_k, diopiConstTensorHandle_t prefix_v, diopiConstTensorHandle_t k_cache,
                              diopiConstTensorHandle_t k_scale, diopiConstTensorHandle_t v_cache, diopiConstTensorHandle_t v_scale,
                              diopiConstTensorHandle_t lengths, double scale) {
    B200_VIEW(vo, out);
    B200_VIEW(vq, q);
    B200_VIEW(vk, k_cache);
    B200_VIEW(vv, v_cache);
    B200_VIEW(vn, lengths);
    TensorView vl, vks, vvs, vpk, vpv;
    if (softmax_lse && !make_view(softmax_lse, &vl, "softmax_lse")) return diopiErrorOccurred;
    B200_CHECK((k_scale == nullptr) == (v_scale == nullptr), "%s: k_scale and v_scale go together", name);
    B200_CHECK(vq.ndim == 3 && vo.ndim == 3 && vk.ndim == 4 && vv.ndim == 4, "%s: q and out must be [batch, heads, dim], caches [batch, kv heads, capacity, dim]", name);
    const int64_t B = vq.shape[0], Hq = vq.shape[1], D = vq.shape[2], Hkv = vk.shape[1], L = vk.shape[2];
    for (int d = 0; d < 3; ++d) B200_CHECK(vo.shape[d] == vq.shape[d], "%s: out must have q's shape", name);
    B200_CHECK((vq.dtype == diopi_dtype_bfloat16 || vq.dtype == diopi_dtype_float16) && vo.dtype == vq.dtype, "%s: q and out must be bfloat16 or float16 of one dtype", name);
    B200_CHECK(D == 64 || D == 128, "%s: head dim 64 or 128, got %lld", name, (long long)D);
    B200_CHECK(vk.shape[0] == B && vk.shape[3] == D, "%s: the caches' batch and head dim must match q", name);
    B200_CHECK(Hkv > 0 && Hq % Hkv == 0, "%s: %lld query heads cannot share %lld key heads", name, (long long)Hq, (long long)Hkv);
    B200_CHECK(vq.device == diopi_device && vo.device == diopi_device, "%s: operands must live on the device", name);
    B200_CHECK(vq.aligned(16) && vo.aligned(16) && kv_rows_fit(vq, 8, false) && kv_rows_fit(vo, 8, true),
               "%s: q and out need contiguous 16-byte aligned rows and pitches that are multiples of 8", name);
    B200_CHECK(vq.numel == 0 || vo.data != vq.data, "%s: out must not be q", name);
    if (k_scale) {
        if (!make_view(k_scale, &vks, "k_scale") || !make_view(v_scale, &vvs, "v_scale")) return diopiErrorOccurred;
        if (diopiError_t e = kv_cache_check(name, vk, vks, vv, vvs, false); e != diopiSuccess) return e;
    } else {
        for (int d = 0; d < 4; ++d) B200_CHECK(vk.shape[d] == vv.shape[d], "%s: k and v caches must have the same shape", name);
        B200_CHECK(vk.dtype == vq.dtype && vv.dtype == vq.dtype, "%s: caches without scales must have q's dtype, got %s and %s", name, dtype_name(vk.dtype), dtype_name(vv.dtype));
        B200_CHECK(vk.device == diopi_device && vv.device == diopi_device, "%s: operands must live on the device", name);
        B200_CHECK(vk.aligned(16) && vv.aligned(16) && kv_rows_fit(vk, 8, false) && kv_rows_fit(vv, 8, false),
                   "%s: cache rows must be contiguous, 16-byte aligned, with pitches that are multiples of 8", name);
    }
    B200_CHECK(vn.dtype == diopi_dtype_int64 && vn.ndim == 1 && vn.shape[0] == B && vn.is_contiguous() && vn.device == diopi_device,
               "%s: lengths must be a dense int64 tensor [batch] on the device", name);
    B200_CHECK(std::isfinite(scale) && scale > 0.0, "%s: scale must be positive, got %g", name, scale);
    if (softmax_lse) {
        B200_CHECK(vl.dtype == diopi_dtype_float32 && vl.ndim == 2 && vl.shape[0] == B && vl.shape[1] == Hq && vl.device == diopi_device,
                   "%s: softmax_lse must be float32 [batch, heads]", name);
        for (int d = 0; d < 2; ++d) B200_CHECK(vl.shape[d] <= 1 || vl.stride[d] > 0, "%s: softmax_lse must not share elements", name);
    }
    int64_t P = 0;
    if (prefix_k) {
        if (!make_view(prefix_k, &vpk, "prefix_k") || !make_view(prefix_v, &vpv, "prefix_v")) return diopiErrorOccurred;
        B200_CHECK(vpk.ndim == 3 && vpv.ndim == 3 && vpk.shape[1] == Hkv && vpk.shape[2] == D && vpk.shape[0] == vpv.shape[0] && vpk.shape[1] == vpv.shape[1] &&
                       vpk.shape[2] == vpv.shape[2],
                   "%s: prefix_k and prefix_v must be [tokens, kv heads, dim]", name);
        B200_CHECK(vpk.dtype == vq.dtype && vpv.dtype == vq.dtype && vpk.device == diopi_device && vpv.device == diopi_device, "%s: the prefix must have q's dtype and device", name);
        B200_CHECK(vpk.aligned(16) && vpv.aligned(16) && kv_rows_fit(vpk, 8, true) && kv_rows_fit(vpv, 8, true),
                   "%s: prefix rows must be contiguous, 16-byte aligned, with positive pitches that are multiples of 8", name);
        P = vpk.shape[0];
    }
    B200_CHECK(P < (1ll << 30) && L < (1ll << 30), "%s: sequence too long", name);
    B200_CHECK(B < (1 << 24) && Hq < 65536, "%s: too many sequences or heads", name);
    if (vq.numel == 0) return diopiSuccess;
    CachedAttnParams p = {};
    p.q = vq.data; p.out = vo.data;
    p.q_sb = vq.stride[0]; p.q_sh = vq.stride[1]; p.o_sb = vo.stride[0]; p.o_sh = vo.stride[1];
    if (softmax_lse) {
        p.lse = static_cast<float*>(vl.data); p.lse_sb = vl.stride[0]; p.lse_sh = vl.stride[1];
    }
    p.k = vk.data; p.v = vv.data;
    p.k_sb = vk.stride[0]; p.k_sh = vk.stride[1]; p.k_sl = vk.stride[2];
    p.v_sb = vv.stride[0]; p.v_sh = vv.stride[1]; p.v_sl = vv.stride[2];
    if (k_scale) {
        p.ks = static_cast<const float*>(vks.data); p.vs = static_cast<const float*>(vvs.data);
        p.ks_sb = vks.stride[0]; p.ks_sh = vks.stride[1]; p.vs_sb = vvs.stride[0]; p.vs_sh = vvs.stride[1];
    }
    p.lengths = static_cast<const int64_t*>(vn.data); p.L = L;
    if (P > 0) {
        p.pk = vpk.data; p.pv = vpv.data; p.P = P;
        p.pk_sp = vpk.stride[0]; p.pk_sh = vpk.stride[1]; p.pv_sp = vpv.stride[0]; p.pv_sh = vpv.stride[1];
    }
    p.B = static_cast<int>(B); p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv); p.group = static_cast<int>(Hq / Hkv);
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    cudaStream_t stream = stream_of(ctx);
    B200_CHECK(B < 65536, "%s: too many sequences", name);
    const dim3 grid(static_cast<unsigned>(Hq), static_cast<unsigned>(B));
    if (vq.dtype == diopi_dtype_bfloat16) {
        if (D == 128) cached_attention_kernel<bf16, 128><<<grid, 128, 0, stream>>>(p); else cached_attention_kernel<bf16, 64><<<grid, 128, 0, stream>>>(p);
    } else {
        if (D == 128) cached_attention_kernel<fp16, 128><<<grid, 128, 0, stream>>>(p); else cached_attention_kernel<fp16, 64><<<grid, 128, 0, stream>>>(p);
    }
    B200_LAUNCH_CHECK(name);
    return diopiSuccess;
}

}  // namespace
}  // namespace b200

extern "C" {

DIOPI_API diopiError_t diopiB200CachedAttention(diopiContextHandle_t ctx, diopiTensorHandle_t out, diopiTensorHandle_t softmax_lse, diopiConstTensorHandle_t q,
                                                diopiConstTensorHandle_t k_cache, diopiConstTensorHandle_t k_scale, diopiConstTensorHandle_t v_cache,
                                                diopiConstTensorHandle_t v_scale, diopiConstTensorHandle_t lengths, double scale) {
    return b200::cached_attention("diopiB200CachedAttention", ctx, out, softmax_lse, q, nullptr, nullptr, k_cache, k_scale, v_cache, v_scale, lengths, scale);
}

DIOPI_API diopiError_t diopiB200SharedPrefixAttention(diopiContextHandle_t ctx, diopiTensorHandle_t out, diopiTensorHandle_t softmax_lse, diopiConstTensorHandle_t q,
                                                      diopiConstTensorHandle_t prefix_k, diopiConstTensorHandle_t prefix_v, diopiConstTensorHandle_t k_cache,
                                                      diopiConstTensorHandle_t k_scale, diopiConstTensorHandle_t v_cache, diopiConstTensorHandle_t v_scale,
                                                      diopiConstTensorHandle_t lengths, double scale) {
    const char* name = "diopiB200SharedPrefixAttention";
    B200_CHECK(prefix_k != nullptr && prefix_v != nullptr, "%s: prefix_k and prefix_v are needed", name);
    return b200::cached_attention(name, ctx, out, softmax_lse, q, prefix_k, prefix_v, k_cache, k_scale, v_cache, v_scale, lengths, scale);
}

}  // extern "C"
