// Attention of one new token per sequence over caches of ragged lengths, with or without a prompt that the batch shares.
//
//   diopiB200CachedAttention        softmax(scale * q K_b^T) V_b, K_b / V_b the first lengths[b] rows of sequence b's cache, which is
//                                   int8 codes with one scale per row (kv_cache.cu) or holds the model's type
//   diopiB200SharedPrefixAttention  the same over the rows of a prompt [P, Hkv, D], stored once, and then the sequence's own rows
//
// Bound by reading the cache: 2 (D + 4) bytes a key and key head (int8) against 4 D group flops. 64 sequences x 32 heads x 4096 keys x
// 128: 2.22 GB in 364 us, 6.1 TB/s, in a single launch at 1.78 GHz; the card's power limit takes a steady loop to 1.65 GHz and 410 - 425 us.
//
// Work is cut evenly, whatever the lengths. A segment is one sequence x key head x group of up to 8 NT query heads; its keys count in
// units of 64. The units of all segments, in order, are dealt to the CTAs in equal consecutive ranges, so a long sequence is spread
// over many CTAs and a CTA may finish several short ones. The lengths are device data: every CTA sums them itself. A segment that one
// CTA holds whole is finished there; the pieces of the others go to a workspace (at most two per CTA: its first and its last
// segment) and a second kernel joins them in a fixed order - no atomics, the same bits every time.
//
// A warp takes 16 keys of a unit. Asynchronous copies bring its rows into a ring of its own in shared memory, two or three tiles ahead
// and across the ends of segments: some 100 KB in flight on an SM, where register loads held a third (427 -> 354 us). The products run on
// mma.sync.m16n8k16 with the KEYS as the 16 rows and the query heads as the 8 columns: S^T = K Q^T, O^T = V^T P^T. At a few flops per
// byte a larger instruction would not be filled; what this shape saves is the feeding, because the order of the contracted index is
// free. For S^T a lane takes 16-byte chunks of its two key rows and the queries are laid out the same way; for O^T a lane takes 16
// neighbouring columns of its four key rows and pairs of keys are zipped with byte permutes. int8 codes become fp16 exactly (a byte
// under the exponent of 1024, minus 1152), 1.25 to 1.5 instructions a value.
//
// A tile costs a warp about 430 instructions in one chain - scores, maximum, exponentials, transposition, values - that three warps a
// scheduler do not hide: issue slots 60 % busy, the busiest pipe 52 %, waits for fixed latencies the largest stall. 8 % fewer instructions
// took 411 us against 413; the copies without the products take 347 at any clock.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "attention_cached.h"
#include "device_utils.cuh"
#include "diopi/functions_b200.h"
#include "gemm.h"
#include "kv_cache.h"

namespace b200 {
namespace {

constexpr int kUnit = 64;            // keys per unit: 16 for each of a CTA's four warps
// What a segment's start and end cost, in units (loading its queries, joining four warps, storing). Ragged batch of 44 sequences, 1 to
// 16384 keys, int8: 164 / 166 / 137 / 133 / 137 us with 0 / 1 / 2 / 3 / 5; 64 sequences of 1 to 1024 own keys
// behind a prompt: 137 / 108 / 94 / 96 / 100.
constexpr int kStart = 2;
constexpr int kMinPlaces = kStart + 1;   // fewer places than this per CTA are not worth a piece of their own
// Caches of at most this capacity: whole segments, one launch (64 x 32 heads of 400 keys: 52 us against 59 with pieces and their join;
// at 1024 slots one sequence of 8 heads takes 12.9 us whole and 8.6 in pieces).
constexpr int64_t kWholeKeys = 512;
// From so many (sequence, query head) rows on the join has a warp for each, below that a CTA of sixteen (whole calls: 4096 rows of one
// piece 36 us against 54, 2048 rows of five 93 against 103, 2048 of two 44 either way; 1024 rows of four pieces 44 us against 38, 512
// of one 99 against 95, 64 of 55 pieces 67 against 40).
constexpr int64_t kWarpRows = 2048;
constexpr float kLowest = -3e38f;    // a running maximum before the first score: finite, so that no difference with it is NaN
constexpr float kGrow = 8.f;         // the running maximum follows only when a score outgrows it by this (log2)

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
    const void* pv;                // the shared prompt's values, P rows
    int64_t pv_sp, pv_sh, P;
    int B, Hq, Hkv, group;
    int tiles;                     // groups of 8 NT query heads per key head
    int whole;                     // 1: a CTA takes whole segments, nothing is joined
    int own;                       // 0: no own keys at all (capacity 0)
    int max_ctas;
    float scale_log2;
    // workspace
    int* before;                   // [B + 1]: places of the sequences before b (per key head and tile); [B]: of all
    float* part_o;                 // [2 max_ctas (+ B Hkv tiles with a prefix)][8 NT][D]
    float2* part_ml;               // the same slots' running maximum (log2) and sum
    PrefixParts prefix;            // splits = 0: no prefix
};

// Over int8 rows the second operand of O^T is P = e vs gain, e = 2^(s - m) <= 1, vs the row's scale: fp16, whose range is small beside
// that of e vs. So every query head has a gain of its own, a power of two that has taken the largest e vs so far to [2^6, 2^7) and
// follows when P outgrows kTop: a key without weight, whatever its scale, and a key of large weight and small scale leave the
// others their bits. Below 2^-31 of the largest e vs a product has lost all of them. O is divided by the gain at the end.
constexpr float kTop = 32768.f;
__device__ __forceinline__ float gain_of(float largest) {     // finite, not negative
    const int e = max(static_cast<int>(__float_as_uint(largest) >> 23) - 127, -120);
    return __uint_as_float(static_cast<uint32_t>(127 + 6 - e) << 23);
}
__device__ __forceinline__ float inverse(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }   // of a power of two
// What 2^6 stands for under a gain, after the running maximum has taken the products down by f.
__device__ __forceinline__ float held(float gain, float f) { return f * (64.f * inverse(gain)); }
// From one gain to the next, with the running maximum's factor.
__device__ __forceinline__ float step(float from, float to, float f) { return f * to * inverse(from); }
__device__ __forceinline__ float finite_or_zero(float x) { return x < INFINITY ? x : 0.f; }

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Units of sequence b and its length. An empty sequence counts one: someone has to write its zeros.
__device__ __forceinline__ int units_of(const CachedAttnParams& p, int b, int* len) {
    const int n = static_cast<int>(min(max(p.lengths[b], int64_t(0)), p.L));
    *len = n;
    return max(1, (n + kUnit - 1) / kUnit);
}
// The dealing works on places: a segment takes kStart places, for what its start and end cost, and then one for each of its units.
// Of `total` places dealt to `ctas` CTAs, CTA c has [total c / ctas, total (c + 1) / ctas).
__device__ __forceinline__ int ctas_of(const CachedAttnParams& p, int total) { return min(p.max_ctas, (total + kMinPlaces - 1) / kMinPlaces); }
__device__ __forceinline__ int place_of(int total, int c, int ctas) { return static_cast<int>(static_cast<int64_t>(total) * c / ctas); }

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, bf16>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
// The same with a zero addend.
template <typename T>
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, bf16>::value) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// Shared memory of a variant: every warp's ring of key tiles (with the scales of the key and value rows) and value tiles, then the
// two slots of the join.
template <bool QUANT, int D, int NT>
struct Ring {
    static constexpr int kRow = D * (QUANT ? 1 : 2);                       // bytes of a cache row
    static constexpr int kKeys = 16 * kRow + (QUANT ? 128 : 0);
    static constexpr int kStage = kKeys + 16 * kRow;
    static constexpr int kStages = QUANT || D == 64 ? 3 : 2;
    static constexpr int kJoinFloats = NT * (D / 4 + 4) + 4;               // per lane: O, maximum and sum, reference
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kTotal = 4 * kWarp + 2 * kJoinFloats * 128;
    static constexpr int kCtas = std::min(3, 232448 / (kTotal + 1024 + 64));   // an SM holds
};

// Where a chunk of 16 bytes of a row lies, so that neither the copies nor the operand reads (eight lanes at a time: two key rows x
// four chunks; four value rows x two chunks) meet in a bank.
template <int CH>
__device__ __forceinline__ int k_chunk(int row, int chunk) { return CH >= 8 ? chunk ^ ((row & 1) << 2) : chunk; }
template <int CH>
__device__ __forceinline__ int v_chunk(int row, int chunk) { return CH >= 8 ? chunk ^ (row & 6) : chunk ^ ((row >> 1) & 3); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Barriers of two of the CTA's warps: one waits, the other one only reports.
enum { kGiven1 = 1, kGiven2, kGiven3, kTaken2, kTaken3 };
__device__ __forceinline__ void barrier_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void barrier_arrive(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }

// A place in the sequence of units: unit kb of the nb units of segment (b, hw), whose sequence has n keys.
struct Cursor {
    int b, hw, kb, nb, n, left;    // left: units of the CTA from here on
    __device__ __forceinline__ void enter(const CachedAttnParams& p, int sequence) {
        b = sequence;
        nb = units_of(p, b, &n);
    }
    // To the start of the next segment, if the CTA has units there.
    __device__ __forceinline__ void next(const CachedAttnParams& p, int W) {
        kb = 0;
        if (++hw == W) {
            hw = 0;
            if (left > 0) enter(p, b + 1);
        }
    }
};

// The infinities of out's row (b, h), where some of it is not finite although its softmax is. Probabilities are positive, so a column with
// an infinity among its values is that infinity, or NaN beside one of the other sign or a NaN; but a probability in two terms, one
// that rounds to zero and the copies that fill a short tile make it inf - inf or 0 * inf. So the values alone decide, taken down far enough
// that finite ones stay finite. One warp, two rows at a time (four: half the time, but registers that cost the join 1 us of 95 behind a
// shared prompt), 240 ns a row; it stops where NaN is all that can come out.
template <typename T, int D>
__device__ __noinline__ void settle_infinities(const CachedAttnParams& p, int b, int h) {
    constexpr int N = D / 32, AT_ONCE = 2;
    const int lane = threadIdx.x & 31, at = lane * N, hk = h / p.group;
    T* const dst = static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(h) * p.o_sh + at;
    const int64_t n = p.own ? min(max(p.lengths[b], int64_t(0)), p.L) : 0;
    const float* const scales = p.ks != nullptr ? p.vs + b * p.vs_sb + hk * p.vs_sh : nullptr;
    __syncwarp();                     // other lanes wrote some of the row
    if (scales != nullptr) {          // codes are finite: nothing to do beside a scale that is NaN, nor without one that is infinite
        bool nan = false, inf = false;
        for (int64_t i = lane; i < n; i += 32) {
            nan |= isnan(scales[i]);
            inf |= isinf(scales[i]);
        }
        if (__any_sync(0xffffffffu, nan) || (p.P == 0 && !__any_sync(0xffffffffu, inf))) return;
    }
    float o[N];
    bool open[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        o[i] = 0.f;
        open[i] = !(fabsf(to_f32(dst[i])) < INFINITY);
    }
    auto add = [&](const auto* v, int64_t pitch, const float* vs, int64_t count) {
        for (int64_t j = 0; j < count; j += AT_ONCE) {
            bool more = false;
            typename std::remove_const<typename std::remove_pointer<decltype(v)>::type>::type x[AT_ONCE][N];
            float f[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const int64_t r = min(j + u, count - 1);
                memcpy(x[u], __builtin_assume_aligned(v + r * pitch, sizeof(x[u])), sizeof(x[u]));
                f[u] = vs != nullptr ? vs[r] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
#pragma unroll
                for (int i = 0; i < N; ++i) o[i] = fmaf(to_f32(x[u][i]) * f[u], 0x1p-64f, o[i]);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) more |= open[i] && !isnan(o[i]);
            if (!__any_sync(0xffffffffu, more)) return;
        }
    };
    if (p.P > 0) add(static_cast<const T*>(p.pv) + hk * p.pv_sh + at, p.pv_sp, nullptr, p.P);
    const int64_t v0 = b * p.v_sb + hk * p.v_sh + at;
    if (scales != nullptr) add(static_cast<const int8_t*>(p.v) + v0, p.v_sl, scales, n);
    else add(static_cast<const T*>(p.v) + v0, p.v_sl, nullptr, n);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (open[i] && !(fabsf(o[i]) < INFINITY)) dst[i] = from_f32<T>(o[i]);
    }
}

template <typename T, bool QUANT, int D, int NT>
__global__ void __launch_bounds__(128, Ring<QUANT, D, NT>::kCtas) cached_attention_kernel(const __grid_constant__ CachedAttnParams p) {
    using M = typename std::conditional<QUANT, fp16, T>::type;    // operand type of the products
    using R = Ring<QUANT, D, NT>;
    constexpr int ROW = R::kRow;
    constexpr int CH = ROW / 16;                                  // 16-byte chunks of a row
    constexpr int KC = ROW / 64;                                  // chunks of a key row per lane
    constexpr int VW = ROW / 32;                                  // 4-byte words of a value row per lane
    constexpr int KS = D / 16;                                    // contraction steps of S^T = tiles of 16 columns of O
    constexpr int NQ = 8 * NT;
    constexpr int ES = QUANT ? 1 : 2;
    // m is the running maximum less this, so e <= 2^(kGrow + LIFT). fp16 keeps probabilities down to 2^-31 of the largest one that way;
    // the products with bf16 values, which may come near fp32's largest, and their sums stay in range.
    constexpr float LIFT = QUANT ? -kGrow : (std::is_same<T, fp16>::value ? 7.f : -24.f);
    // One term of P is as coarse as the result where both have the same type; there P takes two terms, P rounded and what the rounding
    // left, in two products: the tensor cores have the time. Over int8 rows P is fp16, eight times as fine as a bf16 result: one term.
    constexpr int TERMS = QUANT && std::is_same<T, bf16>::value ? 1 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int sh_sum[4], sh_pos[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- this CTA's range of units ----
    const int W = p.Hkv * p.tiles;
    Cursor at;
    {
        const int per = (p.B + 127) / 128;
        const int b_lo = min(p.B, static_cast<int>(threadIdx.x) * per), b_hi = min(p.B, b_lo + per);
        int mine = 0, n = 0;
#pragma unroll 4
        for (int i = b_lo; i < b_hi; ++i) mine += kStart + units_of(p, i, &n);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) sh_sum[warp] = incl;
        __syncthreads();
        int excl = incl - mine, all = 0;
        for (int w = 0; w < 4; ++w) {
            if (w < warp) excl += sh_sum[w];
            all += sh_sum[w];
        }
        if (blockIdx.x == 0 && p.before != nullptr) {
            int x = excl;
#pragma unroll 4
            for (int i = b_lo; i < b_hi; ++i) {
                p.before[i] = x;
                x += kStart + units_of(p, i, &n);
            }
            if (threadIdx.x == 0) p.before[p.B] = all;
        }
        const int total = all * W, ctas = ctas_of(p, total);
        if (blockIdx.x >= ctas) return;
        const int x0 = place_of(total, blockIdx.x, ctas), x1 = place_of(total, blockIdx.x + 1, ctas);
        // the sequences that hold x0 and x1 (x1 = total: behind the last one)
        if (threadIdx.x == 0) {
            sh_pos[2] = p.B;
            sh_pos[3] = all;
        }
        __syncthreads();
        const int lo = excl * W, hi = (excl + mine) * W;
        if ((x0 >= lo && x0 < hi) || (x1 >= lo && x1 < hi)) {
            int x = excl;
            for (int i = b_lo; i < b_hi; ++i) {
                const int w = kStart + units_of(p, i, &n);
                if (x0 >= x * W && x0 < (x + w) * W) {
                    sh_pos[0] = i;
                    sh_pos[1] = x;
                }
                if (x1 >= x * W && x1 < (x + w) * W) {
                    sh_pos[2] = i;
                    sh_pos[3] = x;
                }
                x += w;
            }
        }
        __syncthreads();
        // units in front of a place: the places in front of its segment without the segments' own, and what the segment adds
        at.enter(p, sh_pos[0]);
        const int r0 = x0 - sh_pos[1] * W;
        at.hw = r0 / (kStart + at.nb);
        at.kb = max(0, r0 - at.hw * (kStart + at.nb) - kStart);
        const int front0 = (sh_pos[1] - kStart * at.b) * W + at.hw * at.nb + at.kb;
        int front1 = (all - kStart * p.B) * W, over = 0, nb1 = 0;
        if (sh_pos[2] < p.B) {
            nb1 = units_of(p, sh_pos[2], &n);
            const int r1 = x1 - sh_pos[3] * W, hw1 = r1 / (kStart + nb1);
            over = max(0, r1 - hw1 * (kStart + nb1) - kStart);
            front1 = (sh_pos[3] - kStart * sh_pos[2]) * W + hw1 * nb1 + over;
        }
        at.left = front1 - front0;
        if (p.whole) {   // whole segments, those whose first unit is in the range
            const int skip = at.kb == 0 ? 0 : at.nb - at.kb;
            at.left += (over == 0 ? 0 : nb1 - over) - skip;
            if (skip != 0) at.next(p, W);
        }
        if (at.left <= 0) return;
    }

    // ---- the copies, up to `kStages` tiles ahead of the products, across the ends of segments ----
    // Keys and values go in copy groups of their own, so that a tile's key rows are replaced as soon as its scores are there.
    uint8_t* ring = smem + warp * R::kWarp;
    constexpr int RPC = 512 / ROW, NC = 16 / RPC;     // rows a copy instruction of the warp covers; copies of a tile
    const int my_row = lane / CH, my_chunk = lane % CH;
    const uint32_t k_dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + my_row * ROW + k_chunk<CH>(my_row, my_chunk) * 16;
    const uint32_t v_dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + R::kKeys + my_row * ROW;
    const int64_t k_pitch = p.k_sl * ES, v_pitch = p.v_sl * ES;
    Cursor ahead = at;
    int ahead_run = 0;                                // units of the current segment still to be copied
    int ahead_k0 = 0;                                 // first key of the warp's next tile
    const uint8_t *k_src = nullptr, *v_src = nullptr; // that key's row, this lane's part of it
    const float* s_src = nullptr;
    uint32_t put = 0;                                 // byte offset of the stage to fill
    auto copy_keys = [&]() {
        if (ahead_run == 0 && ahead.left > 0) {       // the next segment
            ahead_run = min(ahead.nb - ahead.kb, ahead.left);
            ahead_k0 = ahead.kb * kUnit + warp * 16;
            const int hk = ahead.hw / p.tiles;
            k_src = static_cast<const uint8_t*>(p.k) + (ahead.b * p.k_sb + hk * p.k_sh) * ES + (ahead_k0 + my_row) * k_pitch + my_chunk * 16;
            v_src = static_cast<const uint8_t*>(p.v) + (ahead.b * p.v_sb + hk * p.v_sh) * ES + (ahead_k0 + my_row) * v_pitch + my_chunk * 16;
            if (QUANT) s_src = (lane < 16 ? p.ks + ahead.b * p.ks_sb + hk * p.ks_sh : p.vs + ahead.b * p.vs_sb + hk * p.vs_sh) + ahead_k0;
        }
        if (ahead_run > 0 && ahead_k0 < ahead.n) {
            const int last = ahead.n - 1 - ahead_k0;  // rows behind the sequence are replaced by its last one (their scores become -inf)
            if (last >= 15) {
                const uint8_t* src = k_src;
#pragma unroll
                for (int i = 0; i < NC; ++i, src += RPC * k_pitch) copy16(k_dst + put + i * 512, src);
            } else {
#pragma unroll
                for (int i = 0; i < NC; ++i) copy16(k_dst + put + i * 512, k_src + (min(my_row + i * RPC, last) - my_row) * k_pitch);
            }
            if (QUANT) copy4(k_dst + put - my_row * ROW - k_chunk<CH>(my_row, my_chunk) * 16 + 16 * ROW + lane * 4, s_src + min(lane & 15, last));
        }
        copies_commit();
    };
    auto copy_values = [&]() {
        if (ahead_run > 0) {
            if (ahead_k0 < ahead.n) {
                const int last = ahead.n - 1 - ahead_k0;
                if (last >= 15) {
                    const uint8_t* src = v_src;
#pragma unroll
                    for (int i = 0; i < NC; ++i, src += RPC * v_pitch) copy16(v_dst + put + i * 512 + v_chunk<CH>(my_row + i * RPC, my_chunk) * 16, src);
                } else {
#pragma unroll
                    for (int i = 0; i < NC; ++i)
                        copy16(v_dst + put + i * 512 + v_chunk<CH>(my_row + i * RPC, my_chunk) * 16, v_src + (min(my_row + i * RPC, last) - my_row) * v_pitch);
                }
            }
            ahead_k0 += kUnit;
            k_src += kUnit * k_pitch;
            v_src += kUnit * v_pitch;
            if (QUANT) s_src += kUnit;
            --ahead.left;
            if (--ahead_run == 0) ahead.next(p, W);
        }
        copies_commit();
        put += R::kStage;
        if (put == R::kWarp) put = 0;
    };
#pragma unroll
    for (int i = 0; i < R::kStages; ++i) {
        copy_keys();
        copy_values();
    }

    float* join = reinterpret_cast<float*>(smem + 4 * R::kWarp);
    // A segment's query rows, as they come: this lane's 16-byte chunks of row g (of each group of eight). Loaded before the previous
    // segment is finished.
    constexpr int QW = D / 32;
    uint4 qw[NT][QW];
    auto load_queries = [&]() {
        const int hk = at.hw / p.tiles, tile = at.hw - hk * p.tiles;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int q = tile * NQ + nt * 8 + g;
            const T* src = static_cast<const T*>(p.q) + at.b * p.q_sb + static_cast<int64_t>(hk * p.group + q) * p.q_sh;
#pragma unroll
            for (int i = 0; i < QW; ++i) {
                const int e = QUANT ? (i >> 1) * 64 + t * 16 + (i & 1) * 8 : i * 32 + t * 8;
                qw[nt][i] = q < p.group ? *reinterpret_cast<const uint4*>(src + e) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    load_queries();
    uint32_t get = 0;
    bool first = true;
    while (at.left > 0) {
        const int b = at.b, hw = at.hw, n = at.n;
        const int hk = hw / p.tiles, tile = hw - hk * p.tiles;
        const int row0 = hk * p.group + tile * NQ;             // first query head of the segment
        const int rows = min(NQ, p.group - tile * NQ);
        const int run = min(at.nb - at.kb, at.left);
        const bool complete = at.kb == 0 && run == at.nb, from_start = at.kb == 0;
        int k0 = at.kb * kUnit + warp * 16;
        at.left -= run;
        at.next(p, W);

        // ---- queries as the second operand of S^T: column g, the contracted index in the order of the key rows ----
        uint32_t qf[NT][KS][2];
        float sl[NT][2];                                       // softmax scale of columns 2t and 2t + 1, in log2
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float back = 1.f;
            if constexpr (QUANT) {
                float up = 1.f;
                if constexpr (std::is_same<T, bf16>::value) {
                    // bf16 reaches beyond fp16: the row is multiplied by the power of two that takes its largest value to
                    // [2^14, 2^15). Exact, except for values below 2^-28 of that largest one.
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < QW; ++i) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 x = Pair<T>::widen(word(qw[nt][i], j));
                            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                        }
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100), 126);
                    up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23);
                    back = __uint_as_float(static_cast<uint32_t>(127 - 14 + e) << 23);
                }
#pragma unroll
                for (int j = 0; j < KS; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t x = word(qw[nt][j >> 1], (j & 1) * 2 + i);
                        qf[nt][j][i] = std::is_same<T, bf16>::value ? Pair<fp16>::narrow(mul2(Pair<T>::widen(x), make_float2(up, up))) : x;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) qf[nt][j][i] = word(qw[nt][j >> 1], (j & 1) * 2 + i);
                }
            }
            sl[nt][0] = p.scale_log2 * __shfl_sync(0xffffffffu, back, t * 8);
            sl[nt][1] = p.scale_log2 * __shfl_sync(0xffffffffu, back, t * 8 + 4);
        }

        float m[NT][2], l[NT][2], acc[NT][KS][4];
        float gain[NT][2];               // QUANT
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = kLowest;
            gain[nt][0] = gain[nt][1] = 1.f;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }

#pragma unroll 1
        for (int u = 0; u < run; ++u, k0 += kUnit) {
            copies_wait<2 * R::kStages - 1>();
            __syncwarp();
            uint32_t pb[TERMS][NT][2];
            const uint8_t* stage = ring + get;
            if (k0 < n) {
                float s[NT][4], s2[NT][4];
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    const uint4 kw0 = *reinterpret_cast<const uint4*>(stage + g * ROW + k_chunk<CH>(g, t + 4 * c) * 16);
                    const uint4 kw1 = *reinterpret_cast<const uint4*>(stage + (g + 8) * ROW + k_chunk<CH>(g + 8, t + 4 * c) * 16);
                    constexpr int PER = QUANT ? 4 : 2;
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const int i = c * PER + j;
                        uint32_t a[4];
                        if constexpr (QUANT) {
                            const uint32_t w0 = word(kw0, j) ^ 0x80808080u, w1 = word(kw1, j) ^ 0x80808080u;
                            a[0] = codes_to_half2<0x4140>(w0); a[1] = codes_to_half2<0x4140>(w1);
                            a[2] = codes_to_half2<0x4342>(w0); a[3] = codes_to_half2<0x4342>(w1);
                        } else {
                            a[0] = word(kw0, 2 * j); a[1] = word(kw1, 2 * j);
                            a[2] = word(kw0, 2 * j + 1); a[3] = word(kw1, 2 * j + 1);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {   // two chains: half the latency
                            if (i < 2) mma16816_first<M>(i == 0 ? s[nt] : s2[nt], a, qf[nt][i][0], qf[nt][i][1]);
                            else mma16816<M>((i & 1) ? s2[nt] : s[nt], a, qf[nt][i][0], qf[nt][i][1]);
                        }
                    }
                }
                float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;
                if (QUANT) {
                    const float* sc = reinterpret_cast<const float*>(stage + 16 * ROW);
                    ks0 = sc[g]; ks1 = sc[g + 8];
                    vs0 = sc[16 + g]; vs1 = sc[24 + g];
                }
                __syncwarp();       // every lane has read the key rows: the next ones go there
                copy_keys();
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][0] = (s[nt][0] + s2[nt][0]) * (ks0 * sl[nt][0]); s[nt][1] = (s[nt][1] + s2[nt][1]) * (ks0 * sl[nt][1]);
                    s[nt][2] = (s[nt][2] + s2[nt][2]) * (ks1 * sl[nt][0]); s[nt][3] = (s[nt][3] + s2[nt][3]) * (ks1 * sl[nt][1]);
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
                for (int nt = 0; nt < NT; ++nt) grow |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + (kGrow + LIFT) || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + (kGrow + LIFT);
                grow = __any_sync(0xffffffffu, grow);
                float f[NT][2];     // what the growth of the maxima takes older probabilities down by
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) f[nt][0] = f[nt][1] = 1.f;
                if (grow) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float x = fmaxf(s[nt][c], s[nt][2 + c]);
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            x = fmaxf(x - LIFT, m[nt][c]);
                            f[nt][c] = exp2_approx(m[nt][c] - x);
                            m[nt][c] = x;
                            l[nt][c] *= f[nt][c];
                            if constexpr (!QUANT) {
#pragma unroll
                                for (int i = 0; i < KS; ++i) {
                                    acc[nt][i][c] *= f[nt][c];
                                    acc[nt][i][2 + c] *= f[nt][c];
                                }
                            }
                        }
                    }
                }
                float e[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        e[nt][c] = exp2_approx(s[nt][c] - m[nt][c]);
                        e[nt][2 + c] = exp2_approx(s[nt][2 + c] - m[nt][c]);
                        l[nt][c] += e[nt][c] + e[nt][2 + c];
                    }
                }
                if constexpr (QUANT) {
                    bool over = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            e[nt][c] *= vs0;
                            e[nt][2 + c] *= vs1;
                            over |= fmaxf(fabsf(e[nt][c]), fabsf(e[nt][2 + c])) * gain[nt][c] > kTop;
                        }
                    }
                    if (__any_sync(0xffffffffu, over) || grow) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float x = fmaxf(finite_or_zero(fabsf(e[nt][c])), finite_or_zero(fabsf(e[nt][2 + c])));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                                const float to = gain_of(fmaxf(x, held(gain[nt][c], f[nt][c]))), k = step(gain[nt][c], to, f[nt][c]);
                                gain[nt][c] = to;
#pragma unroll
                                for (int i = 0; i < KS; ++i) {
                                    acc[nt][i][c] *= k;
                                    acc[nt][i][2 + c] *= k;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            e[nt][c] *= gain[nt][c];
                            e[nt][2 + c] *= gain[nt][c];
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float2 lo = make_float2(e[nt][0], e[nt][1]), hi = make_float2(e[nt][2], e[nt][3]);   // keys g, g + 8
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        const uint32_t a = Pair<M>::narrow(lo), c = Pair<M>::narrow(hi);
                        pb[k][nt][0] = transpose8x8(a);
                        pb[k][nt][1] = transpose8x8(c);
                        if (k + 1 < TERMS) {
                            const float2 ra = Pair<M>::widen(a), rc = Pair<M>::widen(c);
                            lo = make_float2(lo.x - ra.x, lo.y - ra.y);
                            hi = make_float2(hi.x - rc.x, hi.y - rc.y);
                        }
                    }
                }
            } else {
                copy_keys();
            }
            copies_wait<2 * R::kStages - 1>();
            __syncwarp();
            if (k0 < n) {
                const uint8_t* vt = stage + R::kKeys;
                uint32_t vw[4][VW];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 2 * t + (r & 1) + 8 * (r >> 1);
                    if constexpr (VW == 2) {
                        const uint2 x = *reinterpret_cast<const uint2*>(vt + row * ROW + v_chunk<CH>(row, g >> 1) * 16 + (g & 1) * 8);
                        vw[r][0] = x.x; vw[r][1] = x.y;
                    } else {
#pragma unroll
                        for (int c = 0; c < VW / 4; ++c) {
                            const uint4 x = *reinterpret_cast<const uint4*>(vt + row * ROW + v_chunk<CH>(row, g + 8 * c) * 16);
                            vw[r][4 * c] = x.x; vw[r][4 * c + 1] = x.y; vw[r][4 * c + 2] = x.z; vw[r][4 * c + 3] = x.w;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t a[4];
                    if constexpr (QUANT) {
                        const uint32_t w0 = __byte_perm(vw[0][i >> 1], vw[1][i >> 1], (i & 1) ? 0x7362 : 0x5140) ^ 0x80808080u;
                        const uint32_t w1 = __byte_perm(vw[2][i >> 1], vw[3][i >> 1], (i & 1) ? 0x7362 : 0x5140) ^ 0x80808080u;
                        a[0] = codes_to_half2<0x4140>(w0); a[1] = codes_to_half2<0x4342>(w0);
                        a[2] = codes_to_half2<0x4140>(w1); a[3] = codes_to_half2<0x4342>(w1);
                    } else {
                        a[0] = __byte_perm(vw[0][i], vw[1][i], 0x5410); a[1] = __byte_perm(vw[0][i], vw[1][i], 0x7632);
                        a[2] = __byte_perm(vw[2][i], vw[3][i], 0x5410); a[3] = __byte_perm(vw[2][i], vw[3][i], 0x7632);
                    }
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816<M>(acc[nt][i], a, pb[k][nt][0], pb[k][nt][1]);
                    }
                }
            }
            get += R::kStage;
            if (get == R::kWarp) get = 0;
            __syncwarp();           // and the value rows
            copy_values();
        }

        if (at.left > 0) load_queries();
        // ---- join the four warps: 2 and 3 into 0 and 1, then 1 into 0. A lane's values meet the same lane's ----
        auto put_slot = [&](float* slot) {
            float4* d = reinterpret_cast<float4*>(slot) + lane;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < KS; ++i) d[(nt * (KS + 1) + i) * 32] = make_float4(acc[nt][i][0], acc[nt][i][1], acc[nt][i][2], acc[nt][i][3]);
                d[(nt * (KS + 1) + KS) * 32] = make_float4(m[nt][0], m[nt][1], l[nt][0], l[nt][1]);
            }
            if constexpr (QUANT) d[NT * (KS + 1) * 32] = make_float4(gain[0][0], gain[0][1], gain[NT - 1][0], gain[NT - 1][1]);
        };
        auto add_slot = [&](const float* slot) {
            const float4* d = reinterpret_cast<const float4*>(slot) + lane;
            const float4 gains = QUANT ? d[NT * (KS + 1) * 32] : make_float4(1.f, 1.f, 1.f, 1.f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float4 x = d[(nt * (KS + 1) + KS) * 32];
                const float m0 = fmaxf(m[nt][0], x.x), m1 = fmaxf(m[nt][1], x.y);
                float fa0 = exp2_approx(m[nt][0] - m0), fa1 = exp2_approx(m[nt][1] - m1), fb0 = exp2_approx(x.x - m0), fb1 = exp2_approx(x.y - m1);
                l[nt][0] = l[nt][0] * fa0 + x.z * fb0;
                l[nt][1] = l[nt][1] * fa1 + x.w * fb1;
                m[nt][0] = m0;
                m[nt][1] = m1;
                if constexpr (QUANT) {
                    const float g0 = nt == 0 ? gains.x : gains.z, g1 = nt == 0 ? gains.y : gains.w;
                    const float to0 = gain_of(fmaxf(held(gain[nt][0], fa0), held(g0, fb0))), to1 = gain_of(fmaxf(held(gain[nt][1], fa1), held(g1, fb1)));
                    fa0 = step(gain[nt][0], to0, fa0); fb0 = step(g0, to0, fb0);
                    fa1 = step(gain[nt][1], to1, fa1); fb1 = step(g1, to1, fb1);
                    gain[nt][0] = to0;
                    gain[nt][1] = to1;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const float4 o = d[(nt * (KS + 1) + i) * 32];
                    acc[nt][i][0] = acc[nt][i][0] * fa0 + o.x * fb0;
                    acc[nt][i][1] = acc[nt][i][1] * fa1 + o.y * fb1;
                    acc[nt][i][2] = acc[nt][i][2] * fa0 + o.z * fb0;
                    acc[nt][i][3] = acc[nt][i][3] * fa1 + o.w * fb1;
                }
            }
        };
        // Pairwise barriers: who only gives goes on to the next segment. kTaken: warp 0 has read what warp 2 (3) gave the last time.
        float* const slot0 = join;
        float* const slot1 = join + R::kJoinFloats * 32;
        if (warp >= 2) {
            if (!first) barrier_sync(warp == 2 ? kTaken2 : kTaken3);
            put_slot(warp == 2 ? slot0 : slot1);
            barrier_arrive(warp == 2 ? kGiven2 : kGiven3);
        } else if (warp == 1) {
            barrier_sync(kGiven3);
            add_slot(slot1);
            __syncwarp();
            put_slot(slot1);
            barrier_arrive(kGiven1);
        } else {
            barrier_sync(kGiven2);
            add_slot(slot0);
            if (at.left > 0) barrier_arrive(kTaken2);
            barrier_sync(kGiven1);
            add_slot(slot1);
            if (at.left > 0) barrier_arrive(kTaken3);
            const bool last_word = complete && p.prefix.splits == 0;
            uint32_t settle = 0;      // query heads whose row is not finite
            const int64_t slot = complete ? (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + static_cast<int64_t>(b) * W + hw : 2 * static_cast<int64_t>(blockIdx.x) + (from_start ? 1 : 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float ll = l[nt][c];
                    ll += __shfl_xor_sync(0xffffffffu, ll, 4);
                    ll += __shfl_xor_sync(0xffffffffu, ll, 8);
                    ll += __shfl_xor_sync(0xffffffffu, ll, 16);
                    const int q = nt * 8 + 2 * t + c;
                    if (q >= rows) continue;
                    const float back = QUANT ? inverse(gain[nt][c]) : 1.f;
                    constexpr float DOWN = QUANT ? 16.f : 0.f, BY = QUANT ? 0x1p-16f : 1.f;   // a piece of int8 rows takes the values' sums down, too
                    // a lane holds runs of 8 (int8 rows of 128: 16) neighbouring columns
                    if (last_word) {
                        const float f = ll == 0.f ? 0.f : back / ll;
                        T* dst = static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(row0 + q) * p.o_sh;
                        float sum = 0.f;      // finite if all values are
#pragma unroll
                        for (int i = 0; i < KS; i += 4) {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float2 x = make_float2(acc[nt][i + j][c] * f, acc[nt][i + j][2 + c] * f);
                                w[j] = Pair<T>::narrow(x);
                                sum = fmaf(x.x, 0x1p-8f, fmaf(x.y, 0x1p-8f, sum));
                            }
                            *reinterpret_cast<uint4*>(dst + (VW > 4 ? (i >> 2) * 64 + g * 8 : g * KS * 2 + 2 * i)) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        if (!(fabsf(sum) < INFINITY) && ll > 0.f) settle |= 1u << (2 * nt + c);
                        if (g == 0 && p.lse != nullptr)
                            p.lse[b * p.lse_sb + static_cast<int64_t>(row0 + q) * p.lse_sh] = ll == 0.f ? -INFINITY : (m[nt][c] + log2f(ll)) * 0.6931471805599453f;
                    } else {
                        float* dst = p.part_o + (slot * NQ + q) * D;
#pragma unroll
                        for (int i = 0; i < KS; i += 2) {
                            *reinterpret_cast<float4*>(dst + (VW > 4 ? (i >> 2) * 64 + g * 8 + (2 * i & 7) : g * KS * 2 + 2 * i)) =
                                make_float4(acc[nt][i][c] * (back * BY), acc[nt][i][2 + c] * (back * BY), acc[nt][i + 1][c] * (back * BY), acc[nt][i + 1][2 + c] * (back * BY));
                        }
                        if (g == 0) p.part_ml[slot * NQ + q] = make_float2(m[nt][c] + DOWN, ll * BY);
                    }
                }
            }
            if (last_word && __any_sync(0xffffffffu, settle != 0)) {
                for (int q = 0; q < rows; ++q) {
                    const uint32_t lanes = __ballot_sync(0xffffffffu, (settle >> (q / 8 * 2 + (q & 1))) & 1);
                    if (lanes & (0x11111111u << ((q & 7) >> 1))) settle_infinities<T, D>(p, b, row0 + q);
                }
            }
        }
        first = false;
    }
    copies_wait<0>();
}

// Joins the pieces of one (sequence, query head): those of the prefix, if there is one, and those of the own keys. WARPS warps take a
// row: a CTA's sixteen where rows are few and have many pieces, one where rows are many. A warp keeps a running maximum over its
// pieces, so that maxima and outputs are fetched together.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : 32 * WARPS) cached_attention_join_kernel(const __grid_constant__ CachedAttnParams p, int nq) {
    constexpr int N = D / 32;
    __shared__ float sh_m[WARPS], sh_l[WARPS];
    __shared__ float sh_o[WARPS][D];
    const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
    const int64_t bh = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    if (bh >= static_cast<int64_t>(p.B) * p.Hq) return;   // with one warp per row only: whole warps
    const int b = static_cast<int>(static_cast<uint32_t>(bh) / static_cast<uint32_t>(p.Hq));
    const int h = static_cast<int>(bh) - b * p.Hq, hk = h / p.group, in_group = h - hk * p.group;
    const int tile = in_group / nq, q = in_group - tile * nq;
    const int W = p.Hkv * p.tiles, hw = hk * p.tiles + tile;
    int c0 = 0, pieces = 0;          // own pieces: of CTAs c0, c0 + 1, ...
    bool complete = false;
    if (p.own) {
        const int before = p.before[b], places = p.before[b + 1] - before, total = p.before[p.B] * W;
        const int first = before * W + hw * places, ctas = ctas_of(p, total);
        c0 = place_holder(first + kStart, total, ctas);
        pieces = place_holder(first + places - 1, total, ctas) - c0 + 1;
        complete = pieces == 1 || p.whole;
        if (complete) pieces = 1;
        if (complete && p.prefix.splits == 0) return;
    }
    const int64_t shared_row = static_cast<int64_t>(hk) * p.prefix.rows + static_cast<int64_t>(b) * p.group + in_group, shared_step = static_cast<int64_t>(p.Hkv) * p.prefix.rows;
    int shared = 0;                  // the prefix's pieces
    if (p.prefix.splits > 0) {
        const int at = (hk * p.prefix.row_blocks + static_cast<int>((static_cast<int64_t>(b) * p.group + in_group) / kPrefixRows)) * p.prefix.blocks;
        shared = place_holder(at + p.prefix.blocks - 1, p.prefix.total, p.prefix.ctas) - place_holder(at, p.prefix.total, p.prefix.ctas) + 1;
    }
    const int count = shared + pieces;
    float m = kLowest, l = 0.f, o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int i = warp; i < count; i += WARPS) {
        const float2* ml;
        const float* src;
        if (i < shared) {
            const int64_t r = i * shared_step + shared_row;
            ml = p.prefix.ml + r;
            src = p.prefix.o + r * D;
        } else {
            const int j = i - shared;
            const int64_t slot = complete ? (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + static_cast<int64_t>(b) * W + hw : 2 * static_cast<int64_t>(c0 + j) + (j == 0 ? 1 : 0);
            ml = p.part_ml + slot * nq + q;
            src = p.part_o + (slot * nq + q) * D;
        }
        const float2 x = *ml;
        float y[N];
        if constexpr (N == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src + lane * 4);
            y[0] = v.x; y[1] = v.y; y[2] = v.z; y[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2*>(src + lane * 2);
            y[0] = v.x; y[1] = v.y;
        }
        const float top = fmaxf(m, x.x), fa = exp2_approx(m - top), fb = exp2_approx(x.x - top);
        m = top;
        l = l * fa + x.y * fb;
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] = o[k] * fa + y[k] * fb;
    }
    if constexpr (WARPS > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) sh_o[warp][lane * N + i] = o[i];
        if (lane == 0) {
            sh_m[warp] = m;
            sh_l[warp] = l;
        }
        __syncthreads();
        if (warp != 0) return;
        m = warp_max(lane < WARPS ? sh_m[lane] : kLowest);
        l = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2_approx(sh_m[w] - m);
            l += sh_l[w] * f;
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] += sh_o[w][lane * N + i] * f;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(h) * p.o_sh) + lane * (N / 2);
    float sum = 0.f;                 // finite if all values are
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 x = make_float2(o[i] * inv, o[i + 1] * inv);
        dst[i / 2] = Pair<T>::narrow(x);
        sum = fmaf(x.x, 0x1p-8f, fmaf(x.y, 0x1p-8f, sum));
    }
    if (__any_sync(0xffffffffu, !(fabsf(sum) < INFINITY)) && l > 0.f) settle_infinities<T, D>(p, b, h);
    if (lane == 0 && p.lse != nullptr) p.lse[b * p.lse_sb + static_cast<int64_t>(h) * p.lse_sh] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

template <typename T, bool QUANT, int D, int NT>
cudaError_t launch_own(const CachedAttnParams& p, cudaStream_t stream) {
    const auto kernel = cached_attention_kernel<T, QUANT, D, NT>;
    constexpr int smem = Ring<QUANT, D, NT>::kTotal;
    if (cudaError_t e = tc_ensure_smem_attr(reinterpret_cast<const void*>(kernel), smem); e != cudaSuccess) return e;
    return launch_dependent(kernel, static_cast<unsigned>(p.max_ctas), 128, smem, stream, p);
}
template <typename T, int D>
cudaError_t launch_attention(const CachedAttnParams& p, int nt, cudaStream_t stream) {
    if (p.own) {
        cudaError_t e;
        if (p.ks != nullptr) e = nt == 1 ? launch_own<T, true, D, 1>(p, stream) : launch_own<T, true, D, 2>(p, stream);
        else e = nt == 1 ? launch_own<T, false, D, 1>(p, stream) : launch_own<T, false, D, 2>(p, stream);
        if (e != cudaSuccess) return e;
    }
    if (p.whole && p.own && p.prefix.splits == 0) return cudaSuccess;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hq;
    if (rows >= kWarpRows) return launch_dependent(cached_attention_join_kernel<T, D, 1>, static_cast<unsigned>((rows + 3) / 4), 128, 0, stream, p, 8 * nt);
    return launch_dependent(cached_attention_join_kernel<T, D, 16>, static_cast<unsigned>(rows), 512, 0, stream, p, 8 * nt);
}

// CTAs of a variant that an SM holds at once.
int resident_ctas(int64_t D, bool quant, int nt) {
    if (D == 128) return quant ? (nt == 1 ? Ring<true, 128, 1>::kCtas : Ring<true, 128, 2>::kCtas) : (nt == 1 ? Ring<false, 128, 1>::kCtas : Ring<false, 128, 2>::kCtas);
    return quant ? (nt == 1 ? Ring<true, 64, 1>::kCtas : Ring<true, 64, 2>::kCtas) : (nt == 1 ? Ring<false, 64, 1>::kCtas : Ring<false, 64, 2>::kCtas);
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
    const double scale_log2 = scale * 1.4426950408889634;
    B200_CHECK(std::isfinite(scale) && scale > 0.0, "%s: scale must be positive, got %g", name, scale);
    B200_CHECK(scale_log2 >= FLT_MIN && scale_log2 <= FLT_MAX, "%s: scale leaves float32's range, got %g", name, scale);
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
    if (diopiError_t e = one_device(name, {out, softmax_lse, q, prefix_k, prefix_v, k_cache, k_scale, v_cache, v_scale, lengths}); e != diopiSuccess) return e;
    B200_CHECK(P < (1ll << 30) && L < (1ll << 30), "%s: sequence too long", name);
    B200_CHECK(B < (1 << 24) && Hq < 65536 && B * Hq < 0x7fffffffLL, "%s: too many sequences or heads", name);
    if (vq.numel == 0) return diopiSuccess;
    const int64_t group = Hq / Hkv;
    const int nt = group <= 8 ? 1 : 2;
    const int64_t tiles = (group + 8 * nt - 1) / (8 * nt), segments = B * Hkv * tiles, most_places = segments * ((L + kUnit - 1) / kUnit + 1 + kStart);
    B200_CHECK(segments < (1ll << 31) && most_places < (1ll << 31), "%s: too many keys", name);
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
    p.scale_log2 = static_cast<float>(scale_log2);
    const bool wide = vq.dtype == diopi_dtype_bfloat16;
    const int64_t resident = static_cast<int64_t>(sm_count()) * resident_ctas(D, k_scale != nullptr, nt);
    const int64_t wanted = p.whole ? segments : (most_places + kMinPlaces - 1) / kMinPlaces;
    p.max_ctas = static_cast<int>(wanted < resident ? (wanted < 1 ? 1 : wanted) : resident);
    cudaStream_t stream = stream_of(ctx);
    if (P > 0) {
        p.pv = vpv.data; p.pv_sp = vpv.stride[0]; p.pv_sh = vpv.stride[1]; p.P = P;
        const diopiError_t e = prefix_attention(name, ctx, vq, vpk, vpv, p.scale_log2, &p.prefix, stream);
        if (e != diopiSuccess) return e;
    }
    const bool join = !p.whole || p.prefix.splits > 0;
    if (p.own && join) {
        const int64_t slots = (p.whole ? 0 : 2 * static_cast<int64_t>(p.max_ctas)) + (P > 0 ? segments : 0), rows = slots * 8 * nt;
        const int64_t head = ((B + 1) * 4 + 255) / 256 * 256;
        diopiTensorHandle_t ws = nullptr;
        void* ptr = nullptr;
        B200_CHECK(diopiRequireBuffer(ctx, &ws, head + rows * (D * 4 + 8), diopi_device) == diopiSuccess && ws != nullptr, "%s: workspace allocation failed", name);
        B200_CHECK(diopiGetTensorData(ws, &ptr) == diopiSuccess && ptr != nullptr, "%s: workspace has no data pointer", name);
        p.before = static_cast<int*>(ptr);
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
