// The quantised key / value cache: rows of a head kept as int8 codes with one fp32 scale per (sequence, head, slot).
//
//   diopiB200RopeQuantAppendKV  from the output of ONE q/k/v projection: rotated q -> q_out; rotated k and v -> codes and
//                               scales at the sequences' own positions
//   diopiB200DequantKV          codes * scales of a window of slots, back in the model's type
//
// A row y (D values, fp32; k after the rotation, which is not rounded in between) is stored as
//   scale = max|y| / 127,   code = rint(y / scale) in [-127, 127],   so |y - code * scale| <= 0.5 scale.
// A row of zeros has scale 0 and codes 0; a row that holds an infinity or a NaN has scale NaN, so that it reads back as NaN
// rather than as finite numbers. Symmetric codes need no offset, and one scale per row factors out of q . k and of p * v.
#include "copy.h"
#include "device_utils.cuh"
#include "diopi/functions_b200.h"
#include "kv_cache.h"

namespace b200 {
namespace {

struct AppendParams {
    const void* qkv;
    int64_t x_sb, x_ss;            // element pitches between sequences and tokens
    void* q_out;
    int64_t q_sb, q_ss, q_sh;
    int8_t* k_cache;
    int8_t* v_cache;
    float* k_scale;
    float* v_scale;
    int64_t k_sb, k_sh, k_sl, v_sb, v_sh, v_sl;      // cache pitches (bytes = elements)
    int64_t ks_sb, ks_sh, vs_sb, vs_sh;              // scale pitches; slots are neighbours
    const float* cos_t;
    const float* sin_t;            // [table_rows, rot / 2]
    const int64_t* positions;
    int64_t S, L, table_rows, items;
    int Hq, Hkv, rot;
};

// One thread of a row: 8 values in two groups of four. Half-split layout: values 4c .. 4c+3 of the first half of the rotated part
// and their partners; the part behind it, interleaved pairs and v rows: 8 neighbours.
template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_quant_append_kernel(const AppendParams p) {
    constexpr int LANES = D / 8;   // threads per row
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
    const int c = threadIdx.x % LANES;
    const int heads = p.Hq + 2 * p.Hkv;
    const bool live = item < p.items;
    grid_launch_dependents();   // the attention that follows may set itself up meanwhile
    const int64_t token = live ? item / heads : 0;
    const int h = live ? static_cast<int>(item - token * heads) : 0;
    const int64_t b = token / p.S, s = token - b * p.S;
    const int64_t start = live ? p.positions[b] : -1;
    const int64_t slot = start + s;
    const bool write = start >= 0 && start < p.L && slot < p.L && (p.rot == 0 || slot < p.table_rows);

    const bool rotate = h < p.Hq + p.Hkv && c < p.rot / 8;
    const int lo = (!INTERLEAVED && rotate) ? 4 * c : 8 * c;
    const int hi = (!INTERLEAVED && rotate) ? p.rot / 2 + 4 * c : 8 * c + 4;
    float2 y[4];   // values lo, lo+1 | lo+2, lo+3 | hi, hi+1 | hi+2, hi+3
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = make_float2(0.f, 0.f);
    if (write) {
        const T* src = static_cast<const T*>(p.qkv) + b * p.x_sb + s * p.x_ss + static_cast<int64_t>(h) * D;
        const uint2 wa = __ldcs(reinterpret_cast<const uint2*>(src + lo)), wb = __ldcs(reinterpret_cast<const uint2*>(src + hi));
        y[0] = Pair<T>::widen(wa.x); y[1] = Pair<T>::widen(wa.y);
        y[2] = Pair<T>::widen(wb.x); y[3] = Pair<T>::widen(wb.y);
        if (rotate) {
            const float4 cs = *reinterpret_cast<const float4*>(p.cos_t + slot * (p.rot / 2) + 4 * c);
            const float4 sn = *reinterpret_cast<const float4*>(p.sin_t + slot * (p.rot / 2) + 4 * c);
            if (INTERLEAVED) {
                const float cc[4] = {cs.x, cs.y, cs.z, cs.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = make_float2(fmaf(y[i].y, -ss[i], y[i].x * cc[i]), fmaf(y[i].x, ss[i], y[i].y * cc[i]));
            } else {
                const float2 cc[2] = {make_float2(cs.x, cs.y), make_float2(cs.z, cs.w)}, ss[2] = {make_float2(sn.x, sn.y), make_float2(sn.z, sn.w)};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 a = y[i], bb = y[2 + i];
                    y[i] = fma2(bb, make_float2(-ss[i].x, -ss[i].y), mul2(a, cc[i]));
                    y[2 + i] = fma2(a, ss[i], mul2(bb, cc[i]));
                }
            }
        }
    }
    // Largest magnitude of the row. Compared as bit patterns: infinities and NaN are the largest, and none gets lost.
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, max(__float_as_uint(y[i].x) & 0x7fffffffu, __float_as_uint(y[i].y) & 0x7fffffffu));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!write) return;
    if (h < p.Hq) {
        T* dst = static_cast<T*>(p.q_out) + b * p.q_sb + s * p.q_ss + static_cast<int64_t>(h) * p.q_sh;
        *reinterpret_cast<uint2*>(dst + lo) = make_uint2(Pair<T>::narrow(y[0]), Pair<T>::narrow(y[1]));
        *reinterpret_cast<uint2*>(dst + hi) = make_uint2(Pair<T>::narrow(y[2]), Pair<T>::narrow(y[3]));
        return;
    }
    const bool is_k = h < p.Hq + p.Hkv;
    const int64_t hk = is_k ? h - p.Hq : h - p.Hq - p.Hkv;
    const float amax = __uint_as_float(top);
    const bool finite = top < 0x7f800000u;
    const float scale = finite ? amax / 127.f : __uint_as_float(0x7fc00000u);
    uint32_t code[8];
    if (amax > 1e-30f && finite) {
        // y * (127 / max|y|) + 1.5 * 2^23, rounded once to nearest even: the low byte of the sum is the code. Where the product is
        // within 2^-12 of a tie the quotient itself decides (the product is within 127 * 2^-22 of it): a row's values are few
        // bits long, so half of the largest one, code 63.5, is no rare value.
        const float r = 127.f / amax;
        float off = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = (i & 1) ? y[i >> 1].y : y[i >> 1].x, s = fmaf(x, r, 12582912.f);
            code[i] = __float_as_uint(s);
            off = fmaxf(off, fabsf(fmaf(x, r, 12582912.f - s)));
        }
        if (off > 0.5f - 0x1p-12f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) code[i] = static_cast<uint32_t>(__float2int_rn(((i & 1) ? y[i >> 1].y : y[i >> 1].x) / scale));
        }
    } else {
        // rows so small that 127 / max|y| may overflow, rows of zeros (also those whose scale underflows to zero), rows that are not finite
        const bool zero = !finite || scale == 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            code[2 * i] = zero ? 0u : static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(y[i].x / scale, -127.f), 127.f)));
            code[2 * i + 1] = zero ? 0u : static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(y[i].y / scale, -127.f), 127.f)));
        }
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        w[i] = __byte_perm(__byte_perm(code[4 * i], code[4 * i + 1], 0x0040), __byte_perm(code[4 * i + 2], code[4 * i + 3], 0x0040), 0x5410);
    int8_t* dst = is_k ? p.k_cache + b * p.k_sb + hk * p.k_sh + slot * p.k_sl : p.v_cache + b * p.v_sb + hk * p.v_sh + slot * p.v_sl;
    *reinterpret_cast<uint32_t*>(dst + lo) = w[0];
    *reinterpret_cast<uint32_t*>(dst + hi) = w[1];
    if (c == 0) {
        float* sc = is_k ? p.k_scale + b * p.ks_sb + hk * p.ks_sh + slot : p.v_scale + b * p.vs_sb + hk * p.vs_sh + slot;
        *sc = scale;
    }
}

struct DequantParams {
    const int8_t* cache[2];
    const float* scale[2];
    void* out[2];
    int64_t c_sb[2], c_sh[2], c_sl[2], s_sb[2], s_sh[2], o_sb[2], o_ss[2], o_sh[2];
    const int64_t* positions;      // optional
    int64_t S, L, items;
    int Hkv;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) dequant_kernel(const DequantParams p) {
    constexpr int LANES = D / 8;
    const int which = blockIdx.y;  // 0: k, 1: v
    const int64_t item = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LANES;
    if (item >= p.items) return;
    const int c = threadIdx.x % LANES;
    const int64_t token = item / p.Hkv;
    const int64_t h = item - token * p.Hkv;
    const int64_t b = token / p.S, s = token - b * p.S;
    const int64_t start = p.positions != nullptr ? p.positions[b] : 0;
    if (start < 0 || start >= p.L || start + s >= p.L) return;
    const int64_t slot = start + s;
    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(p.cache[which] + b * p.c_sb[which] + h * p.c_sh[which] + slot * p.c_sl[which] + 8 * c));
    const float scale = p.scale[which][b * p.s_sb[which] + h * p.s_sh[which] + slot];
    const uint32_t words[2] = {w.x, w.y};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = words[i >> 1] >> ((i & 1) * 16);
        const float2 v = make_float2(static_cast<float>(static_cast<int8_t>(u & 0xff)), static_cast<float>(static_cast<int8_t>((u >> 8) & 0xff)));
        o[i] = Pair<T>::narrow(mul2(v, make_float2(scale, scale)));
    }
    T* dst = static_cast<T*>(p.out[which]) + b * p.o_sb[which] + s * p.o_ss[which] + h * p.o_sh[which] + 8 * c;
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
}

bool model_type(diopiDtype_t t) { return t == diopi_dtype_bfloat16 || t == diopi_dtype_float16; }

}  // namespace

bool kv_rows_fit(const TensorView& t, int64_t multiple, bool written) {
    if (t.numel == 0) return true;
    if (t.shape[t.ndim - 1] != 1 && t.stride[t.ndim - 1] != 1) return false;
    for (int d = 0; d + 1 < t.ndim; ++d) {
        if (t.shape[d] == 1) continue;
        if (t.stride[d] < 0 || t.stride[d] % multiple != 0 || (written && t.stride[d] == 0)) return false;
    }
    return true;
}

diopiError_t kv_cache_check(const char* name, const TensorView& k, const TensorView& ks, const TensorView& v, const TensorView& vs, bool written) {
    B200_CHECK(k.ndim == 4 && v.ndim == 4, "%s: caches must be [batch, kv heads, capacity, dim]", name);
    for (int d = 0; d < 4; ++d) B200_CHECK(k.shape[d] == v.shape[d], "%s: k and v caches must have the same shape", name);
    B200_CHECK(k.dtype == diopi_dtype_int8 && v.dtype == diopi_dtype_int8, "%s: quantised caches hold int8 codes, got %s and %s", name, dtype_name(k.dtype),
               dtype_name(v.dtype));
    B200_CHECK(ks.dtype == diopi_dtype_float32 && vs.dtype == diopi_dtype_float32 && ks.ndim == 3 && vs.ndim == 3, "%s: scales must be float32 [batch, kv heads, capacity]", name);
    for (int d = 0; d < 3; ++d) B200_CHECK(ks.shape[d] == k.shape[d] && vs.shape[d] == k.shape[d], "%s: scales must be float32 [batch, kv heads, capacity]", name);
    B200_CHECK(k.device == diopi_device && v.device == diopi_device && ks.device == diopi_device && vs.device == diopi_device, "%s: operands must live on the device", name);
    B200_CHECK(k.aligned(16) && v.aligned(16) && kv_rows_fit(k, 16, written) && kv_rows_fit(v, 16, written),
               "%s: cache rows must be contiguous, 16-byte aligned, with pitches that are multiples of 16%s", name, written ? " and not shared" : "");
    B200_CHECK(ks.aligned(4) && vs.aligned(4) && kv_rows_fit(ks, 1, written) && kv_rows_fit(vs, 1, written), "%s: scales of neighbouring slots must be neighbours", name);
    return diopiSuccess;
}

}  // namespace b200

using namespace b200;

extern "C" {

diopiError_t diopiB200RopeQuantAppendKV(diopiContextHandle_t ctx, diopiTensorHandle_t q_out, diopiConstTensorHandle_t qkv, diopiConstTensorHandle_t cos,
                                        diopiConstTensorHandle_t sin, diopiConstTensorHandle_t positions, diopiTensorHandle_t k_cache,
                                        diopiTensorHandle_t k_scale, diopiTensorHandle_t v_cache, diopiTensorHandle_t v_scale, bool interleaved) {
    const char* name = "diopiB200RopeQuantAppendKV";
    B200_VIEW(vx, qkv);
    B200_VIEW(vp, positions);
    B200_VIEW(vk, k_cache);
    B200_VIEW(vks, k_scale);
    B200_VIEW(vv, v_cache);
    B200_VIEW(vvs, v_scale);
    TensorView vq, vc, vsn;
    if (q_out && !make_view(q_out, &vq, "q_out")) return diopiErrorOccurred;
    B200_CHECK((cos == nullptr) == (sin == nullptr), "%s: cos and sin go together", name);
    if (cos && (!make_view(cos, &vc, "cos") || !make_view(sin, &vsn, "sin"))) return diopiErrorOccurred;
    if (diopiError_t e = kv_cache_check(name, vk, vks, vv, vvs, true); e != diopiSuccess) return e;
    B200_CHECK(vx.ndim == 2 || vx.ndim == 3, "%s: qkv must be [batch, (Hq + 2 Hkv) D] or [batch, tokens, (Hq + 2 Hkv) D]", name);
    const bool tokens = vx.ndim == 3;
    const int64_t B = vx.shape[0], S = tokens ? vx.shape[1] : 1, width = vx.shape[vx.ndim - 1];
    const int64_t Hkv = vk.shape[1], L = vk.shape[2], D = vk.shape[3];
    B200_CHECK(D == 64 || D == 128, "%s: head dim 64 or 128, got %lld", name, (long long)D);
    int64_t Hq = 0;
    if (q_out) {
        B200_CHECK(vq.ndim == vx.ndim + 1 && vq.shape[0] == B && (!tokens || vq.shape[1] == S) && vq.shape[vq.ndim - 1] == D,
                   "%s: q_out must be [batch, Hq, D], with the tokens in between if qkv has them", name);
        Hq = vq.shape[vq.ndim - 2];
        B200_CHECK(vq.dtype == vx.dtype && vq.device == diopi_device && vq.aligned(16) && kv_rows_fit(vq, 8, true),
                   "%s: q_out must have qkv's dtype, contiguous 16-byte aligned rows and pitches that are multiples of 8", name);
    }
    B200_CHECK(vk.shape[0] == B && width == (Hq + 2 * Hkv) * D, "%s: qkv has %lld columns and %lld sequences, the heads and the caches need %lld and %lld", name,
               (long long)width, (long long)B, (long long)((Hq + 2 * Hkv) * D), (long long)vk.shape[0]);
    B200_CHECK(model_type(vx.dtype) && vx.device == diopi_device && vx.aligned(16) && kv_rows_fit(vx, 8, false),
               "%s: qkv must be bfloat16 or float16 with contiguous 16-byte aligned rows and pitches that are multiples of 8", name);
    B200_CHECK(vp.dtype == diopi_dtype_int64 && vp.ndim == 1 && vp.shape[0] == B && vp.is_contiguous() && vp.device == diopi_device,
               "%s: positions must be a dense int64 tensor [batch] on the device", name);
    int64_t rot = 0, table_rows = 0;
    if (cos) {
        B200_CHECK(vc.ndim == 2 && vsn.ndim == 2 && vc.shape[0] == vsn.shape[0] && vc.shape[1] == vsn.shape[1] && vc.dtype == diopi_dtype_float32 &&
                       vsn.dtype == diopi_dtype_float32 && vc.is_contiguous() && vsn.is_contiguous() && vc.aligned(16) && vsn.aligned(16) &&
                       vc.device == diopi_device && vsn.device == diopi_device,
                   "%s: cos / sin must be dense 16-byte aligned float32 tables [positions, rotated / 2] on the device", name);
        table_rows = vc.shape[0];
        rot = 2 * vc.shape[1];
        B200_CHECK(rot <= D && rot % 8 == 0, "%s: the rotated part (%lld) must be a multiple of 8 and at most the head dim", name, (long long)rot);
    }
    if (vx.numel == 0 || L == 0) return diopiSuccess;
    AppendParams p = {};
    p.qkv = vx.data; p.x_sb = vx.stride[0]; p.x_ss = tokens ? vx.stride[1] : 0;
    if (q_out) {
        p.q_out = vq.data; p.q_sb = vq.stride[0]; p.q_ss = tokens ? vq.stride[1] : 0; p.q_sh = vq.stride[vq.ndim - 2];
    }
    p.k_cache = static_cast<int8_t*>(vk.data); p.v_cache = static_cast<int8_t*>(vv.data);
    p.k_scale = static_cast<float*>(vks.data); p.v_scale = static_cast<float*>(vvs.data);
    p.k_sb = vk.stride[0]; p.k_sh = vk.stride[1]; p.k_sl = vk.stride[2];
    p.v_sb = vv.stride[0]; p.v_sh = vv.stride[1]; p.v_sl = vv.stride[2];
    p.ks_sb = vks.stride[0]; p.ks_sh = vks.stride[1]; p.vs_sb = vvs.stride[0]; p.vs_sh = vvs.stride[1];
    if (cos) {
        p.cos_t = static_cast<const float*>(vc.data); p.sin_t = static_cast<const float*>(vsn.data);
    }
    p.positions = static_cast<const int64_t*>(vp.data);
    p.S = S; p.L = L; p.table_rows = table_rows; p.rot = static_cast<int>(rot);
    B200_CHECK(Hq + 2 * Hkv < (1 << 24), "%s: too many heads", name);
    p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv);
    p.items = B * S * (Hq + 2 * Hkv);
    const int64_t per_cta = 256 / (D / 8), ctas = (p.items + per_cta - 1) / per_cta;
    B200_CHECK(ctas < 0x7fffffffLL, "%s: too many elements", name);
    cudaStream_t stream = stream_of(ctx);
    const unsigned grid = static_cast<unsigned>(ctas);
#define LAUNCH_APPEND(T, DIM)                                                                             \
    do {                                                                                                  \
        if (interleaved) rope_quant_append_kernel<T, DIM, true><<<grid, 256, 0, stream>>>(p);             \
        else rope_quant_append_kernel<T, DIM, false><<<grid, 256, 0, stream>>>(p);                        \
    } while (0)
    if (vx.dtype == diopi_dtype_bfloat16) {
        if (D == 128) LAUNCH_APPEND(bf16, 128); else LAUNCH_APPEND(bf16, 64);
    } else {
        if (D == 128) LAUNCH_APPEND(fp16, 128); else LAUNCH_APPEND(fp16, 64);
    }
#undef LAUNCH_APPEND
    B200_LAUNCH_CHECK(name);
    return diopiSuccess;
}

diopiError_t diopiB200DequantKV(diopiContextHandle_t ctx, diopiTensorHandle_t k_out, diopiTensorHandle_t v_out, diopiConstTensorHandle_t k_cache,
                                diopiConstTensorHandle_t k_scale, diopiConstTensorHandle_t v_cache, diopiConstTensorHandle_t v_scale,
                                diopiConstTensorHandle_t positions) {
    const char* name = "diopiB200DequantKV";
    B200_VIEW(vko, k_out);
    B200_VIEW(vvo, v_out);
    B200_VIEW(vk, k_cache);
    B200_VIEW(vks, k_scale);
    B200_VIEW(vv, v_cache);
    B200_VIEW(vvs, v_scale);
    TensorView vp;
    if (positions && !make_view(positions, &vp, "positions")) return diopiErrorOccurred;
    if (diopiError_t e = kv_cache_check(name, vk, vks, vv, vvs, false); e != diopiSuccess) return e;
    const int64_t B = vk.shape[0], Hkv = vk.shape[1], L = vk.shape[2], D = vk.shape[3];
    B200_CHECK(D == 64 || D == 128, "%s: head dim 64 or 128, got %lld", name, (long long)D);
    B200_CHECK(vko.ndim == 4 && vvo.ndim == 4 && vko.shape[0] == B && vko.shape[2] == Hkv && vko.shape[3] == D, "%s: outputs must be [batch, tokens, kv heads, dim]", name);
    for (int d = 0; d < 4; ++d) B200_CHECK(vko.shape[d] == vvo.shape[d], "%s: k_out and v_out must have the same shape", name);
    const int64_t S = vko.shape[1];
    B200_CHECK(model_type(vko.dtype) && vvo.dtype == vko.dtype && vko.device == diopi_device && vvo.device == diopi_device && vko.aligned(16) && vvo.aligned(16) &&
                   kv_rows_fit(vko, 8, true) && kv_rows_fit(vvo, 8, true),
               "%s: outputs must be bfloat16 or float16 of one dtype with contiguous 16-byte aligned rows and pitches that are multiples of 8", name);
    if (positions) {
        B200_CHECK(vp.dtype == diopi_dtype_int64 && vp.ndim == 1 && vp.shape[0] == B && vp.is_contiguous() && vp.device == diopi_device,
                   "%s: positions must be a dense int64 tensor [batch] on the device", name);
    } else {
        B200_CHECK(S <= L, "%s: %lld slots asked of a cache of %lld", name, (long long)S, (long long)L);
    }
    if (vko.numel == 0 || L == 0) return diopiSuccess;
    DequantParams p = {};
    const TensorView* caches[2] = {&vk, &vv};
    const TensorView* scales[2] = {&vks, &vvs};
    const TensorView* outs[2] = {&vko, &vvo};
    for (int i = 0; i < 2; ++i) {
        p.cache[i] = static_cast<const int8_t*>(caches[i]->data); p.scale[i] = static_cast<const float*>(scales[i]->data); p.out[i] = outs[i]->data;
        p.c_sb[i] = caches[i]->stride[0]; p.c_sh[i] = caches[i]->stride[1]; p.c_sl[i] = caches[i]->stride[2];
        p.s_sb[i] = scales[i]->stride[0]; p.s_sh[i] = scales[i]->stride[1];
        p.o_sb[i] = outs[i]->stride[0]; p.o_ss[i] = outs[i]->stride[1]; p.o_sh[i] = outs[i]->stride[2];
    }
    p.positions = positions ? static_cast<const int64_t*>(vp.data) : nullptr;
    p.S = S; p.L = L; p.items = B * S * Hkv;
    B200_CHECK(Hkv < (1 << 24), "%s: too many heads", name);
    p.Hkv = static_cast<int>(Hkv);
    const int64_t per_cta = 256 / (D / 8), ctas = (p.items + per_cta - 1) / per_cta;
    B200_CHECK(ctas < 0x7fffffffLL, "%s: too many elements", name);
    cudaStream_t stream = stream_of(ctx);
    const dim3 grid(static_cast<unsigned>(ctas), 2);
    if (vko.dtype == diopi_dtype_bfloat16) {
        if (D == 128) dequant_kernel<bf16, 128><<<grid, 256, 0, stream>>>(p); else dequant_kernel<bf16, 64><<<grid, 256, 0, stream>>>(p);
    } else {
        if (D == 128) dequant_kernel<fp16, 128><<<grid, 256, 0, stream>>>(p); else dequant_kernel<fp16, 64><<<grid, 256, 0, stream>>>(p);
    }
    B200_LAUNCH_CHECK(name);
    return diopiSuccess;
}

}  // extern "C"
