// Attention of the whole batch's query rows over the rows of a prompt that the sequences share: the pieces that
// attention_cached.cu joins with those of the sequences' own keys. One warp per key, one CTA per (sequence, query head).
#include <cmath>

#include "attention_cached.h"
#include "device_utils.cuh"

namespace b200 {
namespace {

struct PrefixParams {
    const void* q;
    const void* k;
    const void* v;
    int64_t q_sb, q_sh, k_sp, k_sh, v_sp, v_sh, P, rows;
    int group;
    float scale_log2;
    float* o;
    float2* ml;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) prefix_kernel(const PrefixParams p) {
    constexpr int N = D / 32;
    __shared__ float red[4][D + 2];
    const int h = blockIdx.x, hk = h / p.group;
    const int64_t b = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float q[N], acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = to_f32(static_cast<const T*>(p.q)[b * p.q_sb + h * p.q_sh + lane * N + i]) * p.scale_log2;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t j = warp; j < p.P; j += 4) {
        float s = 0.f, vf[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s = fmaf(q[i], to_f32(static_cast<const T*>(p.k)[j * p.k_sp + hk * p.k_sh + lane * N + i]), s);
            vf[i] = to_f32(static_cast<const T*>(p.v)[j * p.v_sp + hk * p.v_sh + lane * N + i]);
        }
        s = warp_sum(s);
        const float m_new = fmaxf(m, s), base = m_new == -INFINITY ? 0.f : m_new;
        const float f = m == -INFINITY ? 0.f : exp2f(m - base), e = exp2f(s - base);
        m = m_new;
        l = l * f + e;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = acc[i] * f + e * vf[i];
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
    const int64_t row = hk * p.rows + b * p.group + (h - hk * p.group);
    for (int c = threadIdx.x; c < D; c += 128) {
        float a = 0.f;
        for (int w = 0; w < 4; ++w) a += red[w][2 + c] * exp2f(red[w][0] - base);
        p.o[row * D + c] = a;
    }
    if (threadIdx.x == 0) {
        float l_all = 0.f;
        for (int w = 0; w < 4; ++w) l_all += red[w][1] * exp2f(red[w][0] - base);
        p.ml[row] = make_float2(mm, l_all);
    }
}

}  // namespace

diopiError_t prefix_attention(const char* name, diopiContextHandle_t ctx, const TensorView& q, const TensorView& k, const TensorView& v, float scale_log2,
                              PrefixParts* parts, cudaStream_t stream) {
    const int64_t B = q.shape[0], Hq = q.shape[1], D = q.shape[2], Hkv = k.shape[1];
    B200_CHECK(B < 65536, "%s: too many sequences", name);
    PrefixParams p = {};
    p.q = q.data; p.k = k.data; p.v = v.data;
    p.q_sb = q.stride[0]; p.q_sh = q.stride[1];
    p.k_sp = k.stride[0]; p.k_sh = k.stride[1]; p.v_sp = v.stride[0]; p.v_sh = v.stride[1];
    p.P = k.shape[0]; p.group = static_cast<int>(Hq / Hkv); p.rows = B * p.group;
    p.scale_log2 = scale_log2;
    diopiTensorHandle_t ws = nullptr;
    void* ptr = nullptr;
    B200_CHECK(diopiRequireBuffer(ctx, &ws, B * Hq * (D * 4 + 8), diopi_device) == diopiSuccess && ws != nullptr, "%s: workspace allocation failed", name);
    B200_CHECK(diopiGetTensorData(ws, &ptr) == diopiSuccess && ptr != nullptr, "%s: workspace has no data pointer", name);
    p.o = static_cast<float*>(ptr);
    p.ml = reinterpret_cast<float2*>(p.o + B * Hq * D);
    const dim3 grid(static_cast<unsigned>(Hq), static_cast<unsigned>(B));
    if (q.dtype == diopi_dtype_bfloat16) {
        if (D == 128) prefix_kernel<bf16, 128><<<grid, 128, 0, stream>>>(p); else prefix_kernel<bf16, 64><<<grid, 128, 0, stream>>>(p);
    } else {
        if (D == 128) prefix_kernel<fp16, 128><<<grid, 128, 0, stream>>>(p); else prefix_kernel<fp16, 64><<<grid, 128, 0, stream>>>(p);
    }
    B200_LAUNCH_CHECK(name);
    parts->o = p.o; parts->ml = p.ml; parts->rows = p.rows; parts->splits = 1;
    return diopiSuccess;
}

}  // namespace b200
