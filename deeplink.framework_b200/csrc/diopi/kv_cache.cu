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

constexpr int kPasses = 3;         // rows a thread of the writer has in flight
// From so many rows on the writer's threads take 16 values instead of 8: less work around a row (1.57 M rows of 128: 152 us against
// 179; 98 k: 13.0 against 13.7), but a longer chain (6144 rows: 3.3 us against 3.0; 49 k: 7.9 against 7.8).
constexpr int64_t kManyRows = 65536;
constexpr int kTokens = 2;         // tokens a CTA of the read-back takes

struct AppendParams {
    const void* qkv;
    int64_t x_sb, x_ss;            // element pitches between sequences and tokens
    void* q_out;
    int64_t q_sb, q_ss, q_sh;
    int8_t* cache[2];              // k, v
    float* scale[2];
    int64_t c_sb[2], c_sh[2], c_sl[2];   // cache pitches (bytes = elements)
    int64_t s_sb[2], s_sh[2];            // scale pitches; slots are neighbours
    const float* cos_t;
    const float* sin_t;            // [table_rows, rot / 2]
    const int64_t* positions;
    int64_t L, table_rows;
    int S, Hq, Hkv, rot;
    int per_cta;                   // passes a CTA takes, at most kPasses
};

// Largest of three magnitudes; a NaN among them is the result.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_abs(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
__device__ __forceinline__ float max_abs8(float2 a, float2 b, float2 c, float2 d) {
    return max_abs(max_abs3(max_abs3(a.x, a.y, b.x), b.y, c.x), max_abs3(c.y, d.x, d.y));
}

// The codes of 8 values, four to a word. amax: the row's largest magnitude, NaN if it holds one.
__device__ __forceinline__ uint2 quantise(const float2 (&y)[4], float amax, float scale) {
    uint32_t code[8];
    // The fast division gives 0 for a divisor above 2^126.
    if (amax > 1e-30f && amax < 0x1p126f) {
        // y * (127 / max|y|) + 1.5 * 2^23, rounded once to nearest even: the low byte of the sum is the code. Where the product is
        // within 2^-12 of a tie (it is within 127 * 2^-20 of the quotient) the quotient decides: a row's values are few bits long,
        // so half of the largest one, code 63.5, is no rare value.
        const float r = __fdividef(127.f, amax);
        const float2 rr = make_float2(r, r), magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-1.f, -1.f);
        float2 d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 s = fma2(y[i], rr, magic);
            code[2 * i] = __float_as_uint(s.x);
            code[2 * i + 1] = __float_as_uint(s.y);
            d[i] = fma2(y[i], rr, fma2(s, minus, magic));   // the product minus its code
        }
        if (max_abs8(d[0], d[1], d[2], d[3]) > 0.5f - 0x1p-12f) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float di = (i & 1) ? d[i >> 1].y : d[i >> 1].x;
                if (fabsf(di) > 0.5f - 0x1p-12f) {
                    // The border h = k + 1/2 next to it, and y - h scale, exact (the difference is small and the product 32 bits
                    // long): the fp32 quotient is h itself up to half a unit in its last place, and then goes to the even side.
                    const float v = (i & 1) ? y[i >> 1].y : y[i >> 1].x;
                    const float k = __uint_as_float(code[i]) - 12582912.f, h = k + copysignf(0.5f, di), rest = fmaf(-h, scale, v);
                    const float half_unit = __uint_as_float((__float_as_uint(h) & 0x7f800000u) - (24u << 23));
                    const float to = fabsf(rest) <= half_unit * scale ? rintf(h) : (rest > 0.f ? ceilf(h) : floorf(h));
                    code[i] = __float_as_uint(to + 12582912.f);
                }
            }
        }
    } else {
        // rows so small or so large that 127 / max|y| leaves its range, rows of zeros (also those whose scale underflows to zero), rows that
        // are not finite
        const bool zero = !(amax < INFINITY) || scale == 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = (i & 1) ? y[i >> 1].y : y[i >> 1].x;
            code[i] = zero ? 0u : static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x / scale, -127.f), 127.f)));
        }
    }
    return make_uint2(__byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(code[4], code[5], 0x0040), __byte_perm(code[6], code[7], 0x0040), 0x5410));
}

// H consecutive 2-byte values of a row, H = 4 or 8.
template <int H>
struct Half {
    uint32_t w[H / 2];
    template <typename T>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (H == 8) {
            const uint4 v = ld16_stream_raw(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
            w[0] = v.x; w[1] = v.y;
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (H == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    }
};

// A thread takes 2 H values of a row in two groups, one in each half of the part they belong to (the rotated part, the part behind it;
// a value row is one part): in the half-split layout these are partners, and in every layout the threads of a row touch
// neighbouring memory with each access. The rows of a token come
// in passes of as many rows as the CTA has groups of D / 2H threads, first those of q, then those of k and v; a CTA takes up to
// kPasses of them and has their loads in flight together. Whether a pass is q or not is the same for the whole CTA, and a thread's
// angles serve all its rows. Moves 2 D bytes in per row, 2 D (q) or D + 4 out; 16384 tokens of 32 + 2 x 32 heads of 128 take 152 us,
// 4.4 TB/s. Not at the memory's rate: 5 warps a scheduler (76 registers) keep the issue slots 66 % busy and the ALU 53 %, the
// rest are waits for fixed latencies and for loads. kPasses = 3: such a token's three passes in one CTA.
template <typename T, int D, bool INTERLEAVED, int H>
__global__ void __launch_bounds__(256, 3) rope_quant_append_kernel(const AppendParams p) {
    constexpr int LANES = D / (2 * H), ROWS = 256 / LANES;
    const int c = threadIdx.x % LANES, r = threadIdx.x / LANES;
    grid_launch_dependents();   // the attention that follows may set itself up meanwhile
    const int b = blockIdx.x / static_cast<unsigned>(p.S), s = static_cast<int>(blockIdx.x - static_cast<unsigned>(b) * p.S);
    const int64_t start = p.positions[b];
    const int q_passes = (p.Hq + ROWS - 1) / ROWS, first = blockIdx.y * p.per_cta;
    const bool turns = c < p.rot / (2 * H);
    const int mine_lo = turns ? H * c : p.rot / 2 + H * c, mine_hi = mine_lo + (turns ? p.rot / 2 : (D - p.rot) / 2);
    const T* src = static_cast<const T*>(p.qkv) + b * p.x_sb + s * p.x_ss;
    Half<H> wa[kPasses], wb[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int pass = first + u;
        const int h = pass < q_passes ? pass * ROWS + r : p.Hq + (pass - q_passes) * ROWS + r;
        wa[u] = wb[u] = Half<H>{};
        if (u < p.per_cta && h < (pass < q_passes ? p.Hq : p.Hq + 2 * p.Hkv)) {
            const bool is_v = h >= p.Hq + p.Hkv;
            wa[u].load(src + h * D + (is_v ? H * c : mine_lo));
            wb[u].load(src + h * D + (is_v ? D / 2 + H * c : mine_hi));
        }
    }
    if (start < 0 || start >= p.L) return;
    const int64_t slot = start + s;
    if (slot >= p.L || (p.rot != 0 && slot >= p.table_rows)) return;
    // half-split: the angles of the pairs (lo i, hi i); interleaved: those of the lo group's pairs, then of the hi group's
    float2 cs[H / 2], sn[H / 2];
    if constexpr (INTERLEAVED && H == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t at = slot * (p.rot / 2) + 2 * c + i * (p.rot / 4);
            cs[i] = turns ? *reinterpret_cast<const float2*>(p.cos_t + at) : make_float2(0.f, 0.f);
            sn[i] = turns ? *reinterpret_cast<const float2*>(p.sin_t + at) : make_float2(0.f, 0.f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < H / 4; ++i) {
            const int64_t at = slot * (p.rot / 2) + (INTERLEAVED ? H / 2 * c + i * (p.rot / 4) : H * c + 4 * i);
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
            if (turns) {
                x = *reinterpret_cast<const float4*>(p.cos_t + at);
                y = *reinterpret_cast<const float4*>(p.sin_t + at);
            }
            cs[2 * i] = make_float2(x.x, x.y); cs[2 * i + 1] = make_float2(x.z, x.w);
            sn[2 * i] = make_float2(y.x, y.y); sn[2 * i + 1] = make_float2(y.z, y.w);
        }
    }
    T* const q_dst = static_cast<T*>(p.q_out) + b * p.q_sb + s * p.q_ss;
    int8_t* const k_dst = p.cache[0] + b * p.c_sb[0] + slot * p.c_sl[0];
    int8_t* const v_dst = p.cache[1] + b * p.c_sb[1] + slot * p.c_sl[1];
    float* const k_scale = p.scale[0] + b * p.s_sb[0] + slot;
    float* const v_scale = p.scale[1] + b * p.s_sb[1] + slot;
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int pass = first + u;
        if (u >= p.per_cta || (pass >= q_passes && (pass - q_passes) * ROWS >= 2 * p.Hkv)) return;
        const bool is_q = pass < q_passes;
        const int h = (is_q ? pass : pass - q_passes) * ROWS + r;
        const bool is_v = !is_q && h >= p.Hkv;
        float2 y[H];   // the first group's pairs of neighbours, then the second's
#pragma unroll
        for (int i = 0; i < H / 2; ++i) {
            y[i] = Pair<T>::widen(wa[u].w[i]);
            y[H / 2 + i] = Pair<T>::widen(wb[u].w[i]);
        }
        if (turns && !is_v) {
#pragma unroll
            for (int i = 0; i < H / 2; ++i) {
                if (INTERLEAVED) {
                    const float2 a = y[2 * i], bb = y[2 * i + 1];
                    y[2 * i] = make_float2(fmaf(a.y, -sn[i].x, a.x * cs[i].x), fmaf(a.x, sn[i].x, a.y * cs[i].x));
                    y[2 * i + 1] = make_float2(fmaf(bb.y, -sn[i].y, bb.x * cs[i].y), fmaf(bb.x, sn[i].y, bb.y * cs[i].y));
                } else {
                    const float2 a = y[i], bb = y[H / 2 + i];
                    y[i] = fma2(bb, make_float2(-sn[i].x, -sn[i].y), mul2(a, cs[i]));
                    y[H / 2 + i] = fma2(a, sn[i], mul2(bb, cs[i]));
                }
            }
        }
        if (is_q) {
            if (h < p.Hq) {
                Half<H> lo, hi;
#pragma unroll
                for (int i = 0; i < H / 2; ++i) {
                    lo.w[i] = Pair<T>::narrow(y[i]);
                    hi.w[i] = Pair<T>::narrow(y[H / 2 + i]);
                }
                T* dst = q_dst + h * p.q_sh;
                lo.store(dst + mine_lo);
                hi.store(dst + mine_hi);
            }
        } else {
            float amax = max_abs8(y[0], y[1], y[2], y[3]);
            if constexpr (H == 8) amax = max_abs(amax, max_abs8(y[4], y[5], y[6], y[7]));
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) amax = max_abs(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            if (h < 2 * p.Hkv) {
                const float scale = amax < INFINITY ? amax / 127.f : __uint_as_float(0x7fc00000u);
                const int hk = is_v ? h - p.Hkv : h;
                int8_t* dst = (is_v ? v_dst : k_dst) + hk * (is_v ? p.c_sh[1] : p.c_sh[0]);
                int8_t *lo = dst + (is_v ? H * c : mine_lo), *hi = dst + (is_v ? D / 2 + H * c : mine_hi);
                if constexpr (H == 8) {
                    *reinterpret_cast<uint2*>(lo) = quantise({y[0], y[1], y[2], y[3]}, amax, scale);
                    *reinterpret_cast<uint2*>(hi) = quantise({y[4], y[5], y[6], y[7]}, amax, scale);
                } else {
                    const uint2 w = quantise({y[0], y[1], y[2], y[3]}, amax, scale);
                    *reinterpret_cast<uint32_t*>(lo) = w.x;
                    *reinterpret_cast<uint32_t*>(hi) = w.y;
                }
                if (c == 0) *((is_v ? v_scale : k_scale) + hk * (is_v ? p.s_sh[1] : p.s_sh[0])) = scale;
            }
        }
    }
}

struct DequantParams {
    const int8_t* cache[2];
    const float* scale[2];
    void* out[2];
    int64_t c_sb[2], c_sh[2], c_sl[2], s_sb[2], s_sh[2], o_sb[2], o_ss[2], o_sh[2];
    const int64_t* positions;      // optional
    int64_t L;
    int S, chunks, Hkv;            // chunks of kTokens tokens per sequence
};

// D / 16 threads take a row, 8 values of each half: a CTA takes 256 / (D / 16) heads of kTokens tokens, of k and of v, with all loads
// in flight. A code becomes fp32 as the low byte of 2^23 + 128 + code, exactly, and then one product is rounded.
// Bound by memory: D + 4 bytes in, 2 D out; 16384 tokens of 2 x 32 heads of 128 take 64 us, 6.3 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(256) dequant_kernel(const DequantParams p) {
    constexpr int LANES = D / 16, ROWS = 256 / LANES;
    const int c = threadIdx.x % LANES, h = blockIdx.y * ROWS + threadIdx.x / LANES;
    const int b = blockIdx.x / static_cast<unsigned>(p.chunks), s0 = static_cast<int>(blockIdx.x - static_cast<unsigned>(b) * p.chunks) * kTokens;
    const int64_t start = p.positions != nullptr ? p.positions[b] : 0;
    if (h >= p.Hkv || start < 0 || start >= p.L || start + s0 >= p.L) return;
    const int64_t slot = start + s0;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(min(kTokens, p.S - s0)), p.L - slot));
    uint2 v[2][kTokens][2];
    float f[2][kTokens];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int8_t* src = p.cache[w] + b * p.c_sb[w] + h * p.c_sh[w] + slot * p.c_sl[w] + 8 * c;
        const float* scales = p.scale[w] + b * p.s_sb[w] + h * p.s_sh[w] + slot;
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            if (t < tokens) {
                v[w][t][0] = __ldcs(reinterpret_cast<const uint2*>(src + t * p.c_sl[w]));
                v[w][t][1] = __ldcs(reinterpret_cast<const uint2*>(src + t * p.c_sl[w] + D / 2));
                f[w][t] = scales[t];
            }
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        T* out = static_cast<T*>(p.out[w]) + b * p.o_sb[w] + s0 * p.o_ss[w] + h * p.o_sh[w] + 8 * c;
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            if (t < tokens) {
                uint32_t o[8];
                const float2 ff = make_float2(f[w][t], f[w][t]), bias = make_float2(-8388736.f, -8388736.f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = ((i & 1) ? v[w][t][i >> 1].y : v[w][t][i >> 1].x) ^ 0x80808080u;
                    const float2 lo = make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7441)));
                    const float2 hi = make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7443)));
                    o[2 * i] = Pair<T>::narrow(mul2(add2(lo, bias), ff));
                    o[2 * i + 1] = Pair<T>::narrow(mul2(add2(hi, bias), ff));
                }
                T* dst = out + t * p.o_ss[w];
                *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(o[4], o[5], o[6], o[7]);
            }
        }
    }
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

diopiError_t one_device(const char* name, std::initializer_list<diopiConstTensorHandle_t> tensors) {
    int current = -1;
    if (cudaGetDevice(&current) != cudaSuccess) {   // no device at all: the launch will say so
        (void)cudaGetLastError();
        current = -1;
    }
    for (diopiConstTensorHandle_t t : tensors) {
        if (t == nullptr) continue;
        diopiDeviceIndex_t index = 0;
        B200_CHECK(diopiGetTensorDeviceIndex(t, &index) == diopiSuccess, "%s: host callback failed while reading a tensor's device", name);
        if (current < 0) current = index;
        B200_CHECK(index == current, "%s: all tensors must live on one device, the current one (found devices %d and %d)", name, current, static_cast<int>(index));
    }
    return diopiSuccess;
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
        B200_CHECK(rot <= D && rot % 16 == 0, "%s: the rotated part (%lld) must be a multiple of 16 and at most the head dim", name, (long long)rot);
    }
    if (diopiError_t e = one_device(name, {q_out, qkv, cos, sin, positions, k_cache, k_scale, v_cache, v_scale}); e != diopiSuccess) return e;
    if (vx.numel == 0 || L == 0) return diopiSuccess;
    B200_CHECK(vk.numel == 0 || (vk.data != vv.data && vks.data != vvs.data), "%s: k and v must have caches and scales of their own", name);
    B200_CHECK(B * S < 0x7fffffffLL && Hq + 2 * Hkv < 65536, "%s: too many tokens or heads", name);
    AppendParams p = {};
    p.qkv = vx.data; p.x_sb = vx.stride[0]; p.x_ss = tokens ? vx.stride[1] : 0;
    if (q_out) {
        p.q_out = vq.data; p.q_sb = vq.stride[0]; p.q_ss = tokens ? vq.stride[1] : 0; p.q_sh = vq.stride[vq.ndim - 2];
    }
    const TensorView* caches[2] = {&vk, &vv};
    const TensorView* scales[2] = {&vks, &vvs};
    for (int i = 0; i < 2; ++i) {
        p.cache[i] = static_cast<int8_t*>(caches[i]->data); p.scale[i] = static_cast<float*>(scales[i]->data);
        p.c_sb[i] = caches[i]->stride[0]; p.c_sh[i] = caches[i]->stride[1]; p.c_sl[i] = caches[i]->stride[2];
        p.s_sb[i] = scales[i]->stride[0]; p.s_sh[i] = scales[i]->stride[1];
    }
    if (cos) {
        p.cos_t = static_cast<const float*>(vc.data); p.sin_t = static_cast<const float*>(vsn.data);
    }
    p.positions = static_cast<const int64_t*>(vp.data);
    p.L = L; p.table_rows = table_rows; p.S = static_cast<int>(S); p.rot = static_cast<int>(rot);
    p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv);
    const bool many = B * S * (Hq + 2 * Hkv) >= kManyRows;
    const int64_t rows = 256 / (D / (many ? 16 : 8)), passes = (Hq + rows - 1) / rows + (2 * Hkv + rows - 1) / rows;
    // as many passes as a CTA can have in flight, fewer while there are not two CTAs for every SM
    int64_t per = kPasses;
    while (per > 1 && B * S * ((passes + per - 1) / per) < 2 * sm_count()) --per;
    p.per_cta = static_cast<int>(per);
    cudaStream_t stream = stream_of(ctx);
    const dim3 grid(static_cast<unsigned>(B * S), static_cast<unsigned>((passes + p.per_cta - 1) / p.per_cta));
#define LAUNCH_APPEND_H(T, DIM, H)                                                                        \
    do {                                                                                                  \
        if (interleaved) rope_quant_append_kernel<T, DIM, true, H><<<grid, 256, 0, stream>>>(p);          \
        else rope_quant_append_kernel<T, DIM, false, H><<<grid, 256, 0, stream>>>(p);                     \
    } while (0)
#define LAUNCH_APPEND(T, DIM)                  \
    do {                                       \
        if (many) LAUNCH_APPEND_H(T, DIM, 8);  \
        else LAUNCH_APPEND_H(T, DIM, 4);       \
    } while (0)
    if (vx.dtype == diopi_dtype_bfloat16) {
        if (D == 128) LAUNCH_APPEND(bf16, 128); else LAUNCH_APPEND(bf16, 64);
    } else {
        if (D == 128) LAUNCH_APPEND(fp16, 128); else LAUNCH_APPEND(fp16, 64);
    }
#undef LAUNCH_APPEND
#undef LAUNCH_APPEND_H
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
    if (diopiError_t e = one_device(name, {k_out, v_out, k_cache, k_scale, v_cache, v_scale, positions}); e != diopiSuccess) return e;
    if (vko.numel == 0 || L == 0) return diopiSuccess;
    B200_CHECK(vko.data != vvo.data, "%s: k_out and v_out must be two tensors", name);
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
    B200_CHECK(B * S < 0x7fffffffLL && Hkv < 65536, "%s: too many tokens or heads", name);
    p.L = L; p.S = static_cast<int>(S); p.Hkv = static_cast<int>(Hkv);
    p.chunks = static_cast<int>((S + kTokens - 1) / kTokens);
    const int64_t rows = 256 / (D / 16);
    cudaStream_t stream = stream_of(ctx);
    const dim3 grid(static_cast<unsigned>(B * p.chunks), static_cast<unsigned>((Hkv + rows - 1) / rows));
    if (vko.dtype == diopi_dtype_bfloat16) {
        if (D == 128) dequant_kernel<bf16, 128><<<grid, 256, 0, stream>>>(p); else dequant_kernel<bf16, 64><<<grid, 256, 0, stream>>>(p);
    } else {
        if (D == 128) dequant_kernel<fp16, 128><<<grid, 256, 0, stream>>>(p); else dequant_kernel<fp16, 64><<<grid, 256, 0, stream>>>(p);
    }
    B200_LAUNCH_CHECK(name);
    return diopiSuccess;
}

}  // extern "C"
