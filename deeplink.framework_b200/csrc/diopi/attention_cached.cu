// Attention of one new token per sequence over caches of ragged lengths, with or without a prompt that the batch shares.
//
//   diopiB200CachedAttention        softmax(scale * q K_b^T) V_b, K_b / V_b the first lengths[b] rows of sequence b's cache, which is
//                                   int8 codes with one scale per row (kv_cache.cu) or holds the model's type
//   diopiB200SharedPrefixAttention  the same over the rows of a prompt [P, Hkv, D], stored once, and then the sequence's own rows
//
// Bound by reading the cache: 2 D (+ 8 bytes of scales) bytes per int8 row pair against 4 D group flops.
//
// Work is cut evenly, whatever the lengths. A segment is one sequence x key head x group of up to 8 NT query heads; its keys count in
// units of 64. The units of all segments, in order, are dealt to the CTAs in equal consecutive ranges, so a long sequence is spread
// over many CTAs and a CTA may finish several short ones. The lengths are device data: every CTA sums them itself. A segment that one
// CTA holds whole is finished there; the pieces of the others go to a workspace (at most two per CTA: its first and its last
// segment) and a second kernel joins them in a fixed order - no atomics, the same bits every time.
//
// A warp takes 16 keys of a unit. The products run on mma.sync.m16n8k16 with the KEYS as the 16 rows and the query heads as the 8
// columns: S^T = K Q^T, O^T = V^T P^T. At a few flops per byte the tensor cores idle either way; what this shape saves is the
// feeding: the rows go from global memory straight into operand registers, no shared memory, because the order of the contracted
// index is free. For S^T a lane takes 16-byte chunks of its two key rows and the queries are laid out the same way; for O^T a lane
// takes 16 neighbouring columns of its four key rows and pairs of keys are zipped with byte permutes. int8 codes become fp16 exactly
// (a byte under the exponent of 1024, minus 1152), 1.25 instructions a value against 2 for a conversion to fp32 and its product.
#include <cmath>
#include <type_traits>

#include "attention_cached.h"
#include "device_utils.cuh"
#include "diopi/functions_b200.h"
#include "kv_cache.h"

namespace b200 {
namespace {

constexpr int kUnit = 64;            // keys per unit: 16 for each of a CTA's four warps
constexpr int kMinUnits = 2;         // fewer units than this per CTA are not worth a piece of their own
constexpr int64_t kWholeKeys = 256;  // caches of at most this capacity: whole segments, one launch
constexpr float kGrow = 8.f;         // the running maximum follows only when a score outgrows it by this (log2): P stays below 2^8

struct CachedAttnParams {
    const void* q;
    void* out;
    float* lse;                    // optional [B, Hq]
    int64_t q_sb, q_sh, o_sb, o_sh, lse_sb, lse_sh;
    const void* k;
    const void* v;
    const float* ks;               // NULL: caches in the model's type
    const float* vs;
    int64_t k_sb, k_sh, k_sl, v_sb, v_sh, v_sl, ks_sb, ks_sh, vs_sb, vs_sh;   // elements
    const int64_t* lengths;
    int64_t L;
    int B, Hq, Hkv, group;
    int tiles;                     // groups of 8 NT query heads per key head
    int whole;                     // 1: a CTA takes whole segments, nothing is joined
    int own;                       // 0: no own keys at all (capacity 0)
    int max_ctas;
    float scale_log2;
    // workspace
    int64_t* before;               // [B + 1]: units of the sequences before b (per key head and tile); [B]: of all
    float* part_o;                 // [2 max_ctas (+ B Hkv tiles with a prefix)][8 NT][D]
    float2* part_ml;               // the same slots' running maximum (log2) and sum
    PrefixParts prefix;            // splits = 0: no prefix
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int64_t units_of(const CachedAttnParams& p, int64_t b, int64_t* len) {
    const int64_t n = min(max(p.lengths[b], int64_t(0)), p.L);
    *len = n;
    return n == 0 ? 1 : (n + kUnit - 1) / kUnit;   // an empty sequence is visited too: someone has to write its zeros
}
// CTAs that get work, and the CTA that holds unit u of `total` dealt to `ctas`.
__device__ __forceinline__ int64_t ctas_of(const CachedAttnParams& p, int64_t total) {
    return min(static_cast<int64_t>(p.max_ctas), p.whole ? total : (total + kMinUnits - 1) / kMinUnits);
}
__device__ __forceinline__ int64_t holder(int64_t u, int64_t total, int64_t ctas) { return ((u + 1) * ctas - 1) / total; }

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, bf16>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
// Transposes an 8 x 8 matrix of 2-byte elements held as lane (row lane / 4, columns 2 (lane % 4), + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// Two biased codes (code + 128, bytes 0 and 1 or 2 and 3 of u) as fp16: 1024 + u, minus 1152.
template <int SEL>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t u) {
    const uint32_t h = __byte_perm(u, 0x64646464u, SEL);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint4 ldg16_once(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ uint2 ldg8_once(const void* p) {
    uint2 r;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
}

template <typename T, bool QUANT, int D, int NT>
__global__ void __launch_bounds__(128) cached_attention_kernel(const CachedAttnParams p) {
    using M = typename std::conditional<QUANT, fp16, T>::type;    // operand type of the products
    constexpr int ROW = D * (QUANT ? 1 : 2);                      // bytes of a cache row
    constexpr int KC = ROW / 64;                                  // 16-byte chunks of a key row per lane
    constexpr int VW = ROW / 32;                                  // 4-byte words of a value row per lane
    constexpr int KS = D / 16;                                    // contraction steps of S^T = tiles of 16 columns of O
    constexpr int NQ = 8 * NT;
    __shared__ float sh_o[4][NQ][D + 4];
    __shared__ float sh_m[4][NQ], sh_l[4][NQ], sh_ref[4];
    __shared__ int64_t sh_sum[4], sh_pos[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- this CTA's range of units ----
    const int64_t W = static_cast<int64_t>(p.Hkv) * p.tiles;
    const int64_t per = (p.B + 127) / 128;
    const int64_t b_lo = min(static_cast<int64_t>(p.B), threadIdx.x * per), b_hi = min(static_cast<int64_t>(p.B), b_lo + per);
    int64_t mine = 0, n = 0;
    for (int64_t i = b_lo; i < b_hi; ++i) mine += units_of(p, i, &n);
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) sh_sum[warp] = incl;
    __syncthreads();
    int64_t excl = incl - mine, all = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < warp) excl += sh_sum[w];
        all += sh_sum[w];
    }
    if (blockIdx.x == 0 && p.before != nullptr) {
        int64_t x = excl;
        for (int64_t i = b_lo; i < b_hi; ++i) {
            p.before[i] = x;
            x += units_of(p, i, &n);
        }
        if (threadIdx.x == 0) p.before[p.B] = all;
    }
    const int64_t total = all * W;
    const int64_t ctas = ctas_of(p, total);
    if (blockIdx.x >= ctas) return;
    int64_t u = total * blockIdx.x / ctas;
    const int64_t u_end = total * (blockIdx.x + 1) / ctas;
    if (u >= u_end) return;
    if (u >= excl * W && u < (excl + mine) * W) {
        int64_t x = excl;
        for (int64_t i = b_lo; i < b_hi; ++i) {
            const int64_t nb = units_of(p, i, &n);
            if (u < (x + nb) * W) {
                sh_pos[0] = i;
                sh_pos[1] = x;
                break;
            }
            x += nb;
        }
    }
    __syncthreads();
    int64_t b = sh_pos[0];
    int64_t nb = units_of(p, b, &n);
    int64_t hw, kb;
    {
        const int64_t r = u - sh_pos[1] * W;
        hw = r / nb;
        kb = r - hw * nb;
    }
    if (p.whole && kb != 0) {   // whole segments: those that start in the range
        u += nb - kb;
        kb = 0;
        ++hw;
    }

    while (u < u_end) {
        if (hw == W) {
            hw = 0;
            ++b;
            nb = units_of(p, b, &n);
        }
        const int hk = static_cast<int>(hw / p.tiles), tile = static_cast<int>(hw - static_cast<int64_t>(hk) * p.tiles);
        const int row0 = hk * p.group + tile * NQ;             // first query head of the segment
        const int rows = min(NQ, p.group - tile * NQ);
        const int64_t kb_first = kb;
        const int64_t kb_end = p.whole ? nb : min(nb, kb + (u_end - u));
        u += p.whole ? nb : kb_end - kb;

        // ---- queries as the second operand of S^T: column g, the contracted index in the order of the key rows ----
        uint32_t qf[NT][KS][2];
        float sl[NT][2];                                       // softmax scale of columns 2t and 2t + 1, in log2
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const bool have = nt * 8 + g < rows;
            const T* src = static_cast<const T*>(p.q) + b * p.q_sb + static_cast<int64_t>(row0 + nt * 8 + g) * p.q_sh;
            float back = 1.f;
            if constexpr (QUANT) {
                uint4 w[KC][2];
#pragma unroll
                for (int c = 0; c < KC; ++c) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) w[c][i] = have ? *reinterpret_cast<const uint4*>(src + c * 64 + t * 16 + i * 8) : make_uint4(0, 0, 0, 0);
                }
                float up = 1.f;
                if constexpr (std::is_same<T, bf16>::value) {
                    // bf16 reaches beyond fp16: the row is multiplied by the power of two that takes its largest value to
                    // [2^14, 2^15). Exact, except for values below 2^-28 of that largest one.
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float2 x = Pair<T>::widen(word(w[c][i], j));
                                top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                            }
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 126);
                    up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
                    back = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
                }
#pragma unroll
                for (int c = 0; c < KC; ++c) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 ww = w[c][j >> 1];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t x = word(ww, (j & 1) * 2 + i);
                            qf[nt][c * 4 + j][i] = std::is_same<T, bf16>::value ? Pair<fp16>::narrow(mul2(Pair<T>::widen(x), make_float2(up, up))) : x;
                        }
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const uint4 w = have ? *reinterpret_cast<const uint4*>(src + c * 32 + t * 8) : make_uint4(0, 0, 0, 0);
                    qf[nt][c * 2][0] = w.x; qf[nt][c * 2][1] = w.y;
                    qf[nt][c * 2 + 1][0] = w.z; qf[nt][c * 2 + 1][1] = w.w;
                }
            }
            sl[nt][0] = p.scale_log2 * __shfl_sync(0xffffffffu, back, t * 8);
            sl[nt][1] = p.scale_log2 * __shfl_sync(0xffffffffu, back, t * 8 + 4);
        }

        float m[NT][2], l[NT][2], acc[NT][KS][4];
        float vref = 0.f, ivref = 0.f;   // QUANT: P is held relative to the largest value scale so far (rounded up to a power of two)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }

        const char* kbase = static_cast<const char*>(p.k) + (b * p.k_sb + hk * p.k_sh) * (QUANT ? 1 : 2) + t * 16;
        const char* vbase = static_cast<const char*>(p.v) + (b * p.v_sb + hk * p.v_sh) * (QUANT ? 1 : 2) + g * (VW * 4 > 16 ? 16 : VW * 4);
        const float* ksb = QUANT ? p.ks + b * p.ks_sb + hk * p.ks_sh : nullptr;
        const float* vsb = QUANT ? p.vs + b * p.vs_sb + hk * p.vs_sh : nullptr;
        const int64_t k_row = p.k_sl * (QUANT ? 1 : 2), v_row = p.v_sl * (QUANT ? 1 : 2);
        // The last row a lane may read: rows behind the sequence are replaced by its last one and their scores by -inf
        const int64_t last = n - 1;
        uint4 kw[2][KC];
        uint32_t vw[4][VW];
        float ksc[2], vsc[2];
        auto load_k = [&](int64_t k0) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int64_t row = min(k0 + g + 8 * r, last);
#pragma unroll
                for (int c = 0; c < KC; ++c) kw[r][c] = ldg16_once(kbase + row * k_row + c * 64);
                if (QUANT) {
                    ksc[r] = ksb[row];
                    vsc[r] = vsb[row];
                }
            }
        };
        auto load_v = [&](int64_t k0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t row = min(k0 + 2 * t + (r & 1) + 8 * (r >> 1), last);
                const char* src = vbase + row * v_row;
                if constexpr (VW == 2) {
                    const uint2 x = ldg8_once(src);
                    vw[r][0] = x.x; vw[r][1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const uint4 x = ldg16_once(src + c * 128);
                        vw[r][4 * c] = x.x; vw[r][4 * c + 1] = x.y; vw[r][4 * c + 2] = x.z; vw[r][4 * c + 3] = x.w;
                    }
                }
            }
        };
        int64_t k0 = kb * kUnit + warp * 16;
        const int64_t k_stop = min(kb_end * kUnit, n);
        if (k0 < k_stop) {
            load_k(k0);
            load_v(k0);
        }
        for (; k0 < k_stop; k0 += kUnit) {
            const bool more = k0 + kUnit < k_stop;
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t a[4];
                if constexpr (QUANT) {
                    const uint32_t w0 = word(kw[0][i >> 2], i & 3) ^ 0x80808080u, w1 = word(kw[1][i >> 2], i & 3) ^ 0x80808080u;
                    a[0] = codes_to_half2<0x4140>(w0); a[1] = codes_to_half2<0x4140>(w1);
                    a[2] = codes_to_half2<0x4342>(w0); a[3] = codes_to_half2<0x4342>(w1);
                } else {
                    a[0] = word(kw[0][i >> 1], (i & 1) * 2); a[1] = word(kw[1][i >> 1], (i & 1) * 2);
                    a[2] = word(kw[0][i >> 1], (i & 1) * 2 + 1); a[3] = word(kw[1][i >> 1], (i & 1) * 2 + 1);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<M>(s[nt], a, qf[nt][i][0], qf[nt][i][1]);
            }
            const float ks0 = QUANT ? ksc[0] : 1.f, ks1 = QUANT ? ksc[1] : 1.f;
            float vs0 = 1.f, vs1 = 1.f;
            if (QUANT) {
                vs0 = vsc[0];
                vs1 = vsc[1];
            }
            if (more) load_k(k0 + kUnit);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                s[nt][0] *= ks0 * sl[nt][0]; s[nt][1] *= ks0 * sl[nt][1];
                s[nt][2] *= ks1 * sl[nt][0]; s[nt][3] *= ks1 * sl[nt][1];
            }
            if (k0 + 16 > n) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (k0 + g >= n) s[nt][0] = s[nt][1] = -INFINITY;
                    if (k0 + g + 8 >= n) s[nt][2] = s[nt][3] = -INFINITY;
                }
            }
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) grow |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + kGrow || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + kGrow;
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x = fmaxf(s[nt][c], s[nt][2 + c]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        x = fmaxf(x, m[nt][c]);
                        const float f = m[nt][c] == -INFINITY ? 0.f : exp2_approx(m[nt][c] - x);
                        m[nt][c] = x;
                        l[nt][c] *= f;
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            acc[nt][i][c] *= f;
                            acc[nt][i][2 + c] *= f;
                        }
                    }
                }
            }
            if (QUANT) {
                const uint32_t vm = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(vs0), fabsf(vs1))));
                if (vm > __float_as_uint(vref) && vm < 0x7f000000u) {
                    const float up = __uint_as_float((vm & 0x7f800000u) + 0x00800000u);
                    ivref = 1.f / up;
                    const float f = vref * ivref;
                    vref = up;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            acc[nt][i][0] *= f; acc[nt][i][1] *= f;
                            acc[nt][i][2] *= f; acc[nt][i][3] *= f;
                        }
                    }
                }
                vs0 *= ivref;
                vs1 *= ivref;
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
                const float e0 = exp2_approx(s[nt][0] - m0), e1 = exp2_approx(s[nt][1] - m1);
                const float e2 = exp2_approx(s[nt][2] - m0), e3 = exp2_approx(s[nt][3] - m1);
                l[nt][0] += e0 + e2;
                l[nt][1] += e1 + e3;
                pb[nt][0] = transpose8x8(Pair<M>::narrow(make_float2(e0 * vs0, e1 * vs0)));
                pb[nt][1] = transpose8x8(Pair<M>::narrow(make_float2(e2 * vs1, e3 * vs1)));
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t a[4];
                if constexpr (QUANT) {
                    constexpr int kLo = 0x5140, kHi = 0x7362;
                    const uint32_t w0 = __byte_perm(vw[0][i >> 1] ^ 0x80808080u, vw[1][i >> 1] ^ 0x80808080u, (i & 1) ? kHi : kLo);
                    const uint32_t w1 = __byte_perm(vw[2][i >> 1] ^ 0x80808080u, vw[3][i >> 1] ^ 0x80808080u, (i & 1) ? kHi : kLo);
                    a[0] = codes_to_half2<0x4140>(w0); a[1] = codes_to_half2<0x4342>(w0);
                    a[2] = codes_to_half2<0x4140>(w1); a[3] = codes_to_half2<0x4342>(w1);
                } else {
                    a[0] = __byte_perm(vw[0][i], vw[1][i], 0x5410); a[1] = __byte_perm(vw[0][i], vw[1][i], 0x7632);
                    a[2] = __byte_perm(vw[2][i], vw[3][i], 0x5410); a[3] = __byte_perm(vw[2][i], vw[3][i], 0x7632);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<M>(acc[nt][i], a, pb[nt][0], pb[nt][1]);
            }
            if (more) load_v(k0 + kUnit);
        }

        // ---- join the four warps ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[nt][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int q = nt * 8 + 2 * t + c;
                if (g == 0) {
                    sh_m[warp][q] = m[nt][c];
                    sh_l[warp][q] = x;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    // columns 2i and 2i + 1 of the lane's value chunk(s)
                    const int e = VW > 4 ? ((2 * i) >> 3) * 64 + g * 8 + ((2 * i) & 7) : g * KS * 2 + 2 * i;
                    *reinterpret_cast<float2*>(&sh_o[warp][q][e]) = make_float2(acc[nt][i][c], acc[nt][i][2 + c]);
                }
            }
        }
        if (lane == 0) sh_ref[warp] = QUANT ? vref : 1.f;
        __syncthreads();
        const bool complete = p.whole || (kb_first == 0 && kb_end == nb);
        for (int item = threadIdx.x; item < rows * (D / 4); item += 128) {
            const int q = item / (D / 4), c = (item - q * (D / 4)) * 4;
            float mm = fmaxf(fmaxf(sh_m[0][q], sh_m[1][q]), fmaxf(sh_m[2][q], sh_m[3][q]));
            const float base = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = exp2_approx(sh_m[w][q] - base), fo = f * sh_ref[w];
                ll += sh_l[w][q] * f;
                const float4 x = *reinterpret_cast<const float4*>(&sh_o[w][q][c]);
                o.x += x.x * fo; o.y += x.y * fo; o.z += x.z * fo; o.w += x.w * fo;
            }
            if (complete && p.prefix.splits == 0) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                T* dst = static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(row0 + q) * p.o_sh + c;
                *reinterpret_cast<uint2*>(dst) = make_uint2(Pair<T>::narrow(make_float2(o.x * inv, o.y * inv)), Pair<T>::narrow(make_float2(o.z * inv, o.w * inv)));
                if (c == 0 && p.lse != nullptr)
                    p.lse[b * p.lse_sb + static_cast<int64_t>(row0 + q) * p.lse_sh] = ll == 0.f ? -INFINITY : (base + log2f(ll)) * 0.6931471805599453f;
            } else {
                const int64_t slot = complete ? (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + b * W + hw : 2 * static_cast<int64_t>(blockIdx.x) + (kb_first == 0 ? 1 : 0);
                *reinterpret_cast<float4*>(p.part_o + (slot * NQ + q) * D + c) = o;
                if (c == 0) p.part_ml[slot * NQ + q] = make_float2(mm, ll);
            }
        }
        __syncthreads();
        kb = kb_end;
        if (kb == nb) {
            kb = 0;
            ++hw;
        }
    }
}

// Joins the pieces of one (sequence, query head): those of the prefix, if there is one, and those of the own keys.
template <typename T, int D>
__global__ void __launch_bounds__(128) cached_attention_join_kernel(const CachedAttnParams p, int nq) {
    __shared__ float red[4];
    __shared__ float sh_l[4];
    __shared__ float sh_o[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t b = blockIdx.x / p.Hq;
    const int h = static_cast<int>(blockIdx.x - b * p.Hq), hk = h / p.group, in_group = h - hk * p.group;
    const int tile = in_group / nq, q = in_group - tile * nq;
    const int64_t W = static_cast<int64_t>(p.Hkv) * p.tiles, hw = static_cast<int64_t>(hk) * p.tiles + tile;
    grid_launch_dependents();
    grid_dependency_wait();
    int64_t c0 = 0, pieces = 0;      // own pieces: of CTAs c0, c0 + 1, ...
    bool complete = false;
    if (p.own) {
        const int64_t units = p.before[b + 1] - p.before[b], total = p.before[p.B] * W;
        const int64_t first = p.before[b] * W + hw * units;
        const int64_t ctas = ctas_of(p, total);
        c0 = holder(first, total, ctas);
        pieces = holder(first + units - 1, total, ctas) - c0 + 1;
        complete = pieces == 1 || p.whole;
        if (complete) pieces = 1;
        if (complete && p.prefix.splits == 0) return;
    }
    const int64_t shared_row = p.prefix.splits == 0 ? 0 : hk * p.prefix.rows + b * p.group + in_group;
    const int64_t shared_step = p.prefix.splits == 0 ? 0 : static_cast<int64_t>(p.Hkv) * p.prefix.rows;
    const int64_t count = p.prefix.splits + pieces;
    auto at = [&](int64_t i, const float2** ml, const float** o) {
        if (i < p.prefix.splits) {
            const int64_t r = i * shared_step + shared_row;
            *ml = p.prefix.ml + r;
            *o = p.prefix.o + r * D;
            return;
        }
        i -= p.prefix.splits;
        const int64_t slot = complete ? (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + b * W + hw : 2 * (c0 + i) + (i == 0 ? 1 : 0);
        *ml = p.part_ml + slot * nq + q;
        *o = p.part_o + (slot * nq + q) * D;
    };
    const float2* ml;
    const float* src;
    float mm = -INFINITY;
    for (int64_t i = threadIdx.x; i < count; i += 128) {
        at(i, &ml, &src);
        mm = fmaxf(mm, ml->x);
    }
    mm = warp_max(mm);
    if (lane == 0) red[warp] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = mm == -INFINITY ? 0.f : mm;
    constexpr int N = D / 32;
    float o[N], l = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int64_t i = warp; i < count; i += 4) {
        at(i, &ml, &src);
        const float2 x = *ml;
        const float f = exp2_approx(x.x - base);
        l += x.y * f;
        if constexpr (N == 4) {
            const float4 y = *reinterpret_cast<const float4*>(src + lane * 4);
            o[0] += y.x * f; o[1] += y.y * f; o[2] += y.z * f; o[3] += y.w * f;
        } else {
            const float2 y = *reinterpret_cast<const float2*>(src + lane * 2);
            o[0] += y.x * f; o[1] += y.y * f;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) sh_o[warp][lane * N + i] = o[i];
    if (lane == 0) sh_l[warp] = l;
    __syncthreads();
    const float ll = (sh_l[0] + sh_l[1]) + (sh_l[2] + sh_l[3]);
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    for (int c = threadIdx.x * 2; c < D; c += 256) {
        const float x = ((sh_o[0][c] + sh_o[1][c]) + (sh_o[2][c] + sh_o[3][c])) * inv, y = ((sh_o[0][c + 1] + sh_o[1][c + 1]) + (sh_o[2][c + 1] + sh_o[3][c + 1])) * inv;
        *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(h) * p.o_sh + c) = Pair<T>::narrow(make_float2(x, y));
    }
    if (threadIdx.x == 0 && p.lse != nullptr) p.lse[b * p.lse_sb + static_cast<int64_t>(h) * p.lse_sh] = ll == 0.f ? -INFINITY : (base + log2f(ll)) * 0.6931471805599453f;
}

template <typename T, bool QUANT, int D>
cudaError_t launch_own(const CachedAttnParams& p, int nt, cudaStream_t stream) {
    return nt == 1 ? launch_dependent(cached_attention_kernel<T, QUANT, D, 1>, static_cast<unsigned>(p.max_ctas), 128, 0, stream, p)
                   : launch_dependent(cached_attention_kernel<T, QUANT, D, 2>, static_cast<unsigned>(p.max_ctas), 128, 0, stream, p);
}
template <typename T, int D>
cudaError_t launch_attention(const CachedAttnParams& p, int nt, cudaStream_t stream) {
    if (p.own) {
        const cudaError_t e = p.ks != nullptr ? launch_own<T, true, D>(p, nt, stream) : launch_own<T, false, D>(p, nt, stream);
        if (e != cudaSuccess) return e;
    }
    if (p.whole && p.own && p.prefix.splits == 0) return cudaSuccess;
    return launch_dependent(cached_attention_join_kernel<T, D>, static_cast<unsigned>(static_cast<int64_t>(p.B) * p.Hq), 128, 0, stream, p, 8 * nt);
}

// CTAs of a variant that an SM holds at once.
template <typename T, bool QUANT, int D, int NT>
int resident_of() {
    static const int n = [] {
        int v = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&v, cached_attention_kernel<T, QUANT, D, NT>, 128, 0) != cudaSuccess || v < 1) v = 1;
        return v;
    }();
    return n;
}
template <typename T>
int resident_ctas(int64_t D, bool quant, int nt) {
    if (D == 128) return quant ? (nt == 1 ? resident_of<T, true, 128, 1>() : resident_of<T, true, 128, 2>())
                               : (nt == 1 ? resident_of<T, false, 128, 1>() : resident_of<T, false, 128, 2>());
    return quant ? (nt == 1 ? resident_of<T, true, 64, 1>() : resident_of<T, true, 64, 2>())
                 : (nt == 1 ? resident_of<T, false, 64, 1>() : resident_of<T, false, 64, 2>());
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
        for (const TensorView* x : {&vpk, &vpv}) {
            const int64_t lo = x->stride[0] < x->stride[1] ? x->stride[0] : x->stride[1], hi = x->stride[0] < x->stride[1] ? x->stride[1] : x->stride[0];
            B200_CHECK(P <= 1 || Hkv == 1 || hi % lo == 0, "%s: one of the prefix's pitches must be a multiple of the other", name);
            B200_CHECK(hi < (1ll << 38), "%s: the prefix's pitches are too large", name);
        }
    }
    B200_CHECK(P < (1ll << 30) && L < (1ll << 30), "%s: sequence too long", name);
    B200_CHECK(B < (1 << 24) && Hq < 65536 && B * Hq < 0x7fffffffLL, "%s: too many sequences or heads", name);
    if (vq.numel == 0) return diopiSuccess;
    const int64_t group = Hq / Hkv;
    const int nt = group <= 8 ? 1 : 2;
    const int64_t tiles = (group + 8 * nt - 1) / (8 * nt), segments = B * Hkv * tiles, most_units = segments * ((L + kUnit - 1) / kUnit);
    B200_CHECK(most_units < (1ll << 40), "%s: too many keys", name);
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
    p.B = static_cast<int>(B); p.Hq = static_cast<int>(Hq); p.Hkv = static_cast<int>(Hkv); p.group = static_cast<int>(group);
    p.tiles = static_cast<int>(tiles);
    p.own = L > 0 ? 1 : 0;
    p.whole = L <= kWholeKeys ? 1 : 0;
    p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
    const bool wide = vq.dtype == diopi_dtype_bfloat16;
    const int64_t resident = static_cast<int64_t>(sm_count()) * (wide ? resident_ctas<bf16>(D, k_scale != nullptr, nt) : resident_ctas<fp16>(D, k_scale != nullptr, nt));
    const int64_t wanted = p.whole ? segments : (most_units + kMinUnits - 1) / kMinUnits;
    p.max_ctas = static_cast<int>(wanted < resident ? (wanted < 1 ? 1 : wanted) : resident);
    cudaStream_t stream = stream_of(ctx);
    if (P > 0) {
        const diopiError_t e = prefix_attention(name, ctx, vq, vpk, vpv, p.scale_log2, &p.prefix, stream);
        if (e != diopiSuccess) return e;
    }
    const bool join = !p.whole || p.prefix.splits > 0;
    if (p.own && join) {
        const int64_t slots = (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + (P > 0 ? segments : 0), rows = slots * 8 * nt;
        const int64_t head = ((B + 1) * 8 + 255) / 256 * 256;
        diopiTensorHandle_t ws = nullptr;
        void* ptr = nullptr;
        B200_CHECK(diopiRequireBuffer(ctx, &ws, head + rows * (D * 4 + 8), diopi_device) == diopiSuccess && ws != nullptr, "%s: workspace allocation failed", name);
        B200_CHECK(diopiGetTensorData(ws, &ptr) == diopiSuccess && ptr != nullptr, "%s: workspace has no data pointer", name);
        p.before = static_cast<int64_t*>(ptr);
        p.part_o = reinterpret_cast<float*>(static_cast<char*>(ptr) + head);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * D);
    }
    cudaError_t e;
    if (wide) e = D == 128 ? launch_attention<bf16, 128>(p, nt, stream) : launch_attention<bf16, 64>(p, nt, stream);
    else e = D == 128 ? launch_attention<fp16, 128>(p, nt, stream) : launch_attention<fp16, 64>(p, nt, stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        B200_FAIL("%s: kernel launch failed: %s", name, cudaGetErrorString(e));
    }
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
