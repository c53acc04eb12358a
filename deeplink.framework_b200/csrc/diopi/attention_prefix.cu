// Attention of the whole batch's query rows over the rows of a prompt that the sequences share: the pieces that
// attention_cached.cu joins with those of the sequences' own keys.
//
// The query rows of all sequences that share a key head - sequence * group + head in group - are the rows of one matrix, so the
// prompt is read once per 256 of them instead of once per sequence, and the products S = Q K^T, O = P V have 128-row tiles for the
// tensor cores: 4 D flops per row and key against 4 D bytes per key, bound by the tensor cores (by the exponentials beside
// them) from some 200 rows on and by reading the prompt below that.
//
// The blocks of 128 keys of all (key head, 256 query rows) pairs, in order, are dealt to at most one CTA per SM in equal consecutive
// ranges; what a CTA has of one pair is a segment, and every segment leaves its unnormalised fp32 output, running maximum and sum.
// 384 threads, the structure of the prefill kernel (attention.cu):
//   warp 0       TMA producer: K and V blocks of 128 keys through a 3-slot ring, the keys one block ahead of the values
//   warp 1, 3    MMA issuers (one thread each) for row tile 0 and 1: scores and O in TMEM
//   warp 2       TMEM allocation
//   warps 4..7   softmax of tile 0, warps 8..11 of tile 1, one thread per row; the two warps of a scheduler take turns at the
//                exponentials. Before that the same warps copy the tile's query rows into swizzled shared memory: rows of
//                neighbouring sequences are `group` heads apart in general, which no tensor map describes for every group.
// The ring and the barriers run on from one segment to the next. Every wait is bounded (gemm_sm100.cuh); a time-out ends the kernel
// and raises the status word. 256 sequences x 64 heads behind 32768 tokens,
// 8 key heads of 128: 288 us, 955 TFLOP/s at 1.59 GHz. Shared memory is the tightest: both products read both operands there.
#include <cuda.h>

#include <cmath>
#include <type_traits>

#include "attention_cached.h"
#include "device_utils.cuh"
#include "gemm.h"
#include "gemm_sm100.cuh"

namespace b200 {
namespace {

using namespace sm100;

constexpr int kTile = 128;             // query rows per tile (one TMEM lane each)
constexpr int kBlock = 128;            // keys per block
constexpr int kRing = 3;
constexpr int kHalf = 128 * 128;       // 128 rows of 128 bytes (64 two-byte columns), 128-byte swizzle
constexpr int kPBytes = 2 * kHalf;     // P tile: 128 x 128 two-byte
constexpr float kRescale = 8.f;        // log2 units: the running maximum follows when a score outgrows it by this

template <int D>
struct Smem {
    static constexpr int kTileBytes = D / 64 * kHalf;    // Q, K or V tile
    static constexpr int kBars = 2 * kTileBytes + 2 * kPBytes + kRing * kTileBytes;
    static constexpr int kTotal = kBars + 1024 /*alignment*/ + 256 /*barriers*/;
};
static_assert(Smem<128>::kTotal <= 232448, "shared memory budget");

struct PrefixParams {
    const void* q;
    int64_t q_sb, q_sh;
    int rows, group, Hkv, P;
    int row_blocks, blocks;            // blocks of keys
    int total, ctas;                   // blocks of all pairs, CTAs they are dealt to
    int k_hfirst, v_hfirst;            // order of the tensor maps' head and row dimensions
    float scale_log2;
    uint32_t idesc_s, idesc_pv;
    float* o;
    float2* ml;
    uint32_t* status;
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Position of block j's keys / values in the load order K0, K1, V0, K2, V1, ..., K(n-1), V(n-2), V(n-1).
__device__ __forceinline__ int load_of_k(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int load_of_v(int j, int n) { return min(2 * j + 2, 2 * n - 1); }

template <typename T, int D>
__global__ void __launch_bounds__(384, 1) prefix_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams p) {
    using S = Smem<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* smem_q = smem;
    uint8_t* smem_p = smem + 2 * S::kTileBytes;
    uint8_t* smem_kv = smem_p + 2 * kPBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* q_full = bars;                   // [2] softmax -> MMA: the tile's queries are in shared memory
    uint64_t* kv_full = q_full + 2;            // [kRing] producer -> MMA
    uint64_t* kv_empty = kv_full + kRing;      // [kRing] MMA -> producer
    uint64_t* s_full = kv_empty + kRing;       // [2] MMA -> softmax: scores of the block are in TMEM
    uint64_t* s_free = s_full + 2;             // [2] softmax -> MMA: the scores are in registers
    uint64_t* p_full = s_free + 2;             // [2] softmax -> MMA: P is in shared memory
    uint64_t* pv_done = p_full + 2;            // [2] MMA -> softmax: O holds the block, P may be overwritten
    uint64_t* turn = pv_done + 2;              // [4 quarters][2] softmax warp -> its partner of the other tile: exponentials done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 8);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int x0 = static_cast<int>(static_cast<int64_t>(p.total) * blockIdx.x / p.ctas), x1 = static_cast<int>(static_cast<int64_t>(p.total) * (blockIdx.x + 1) / p.ctas);
    // The CTA's segment that starts at place x: key head, first query row, first block, blocks; n1: those of tile 1, which has no rows in
    // the last row block of some batches.
    struct Segment {
        int hk, q0, blk0, n, n1, piece;
    };
    auto segment = [&](int x) {
        Segment g;
        const int pair = x / p.blocks;
        g.hk = pair / p.row_blocks;
        g.q0 = (pair - g.hk * p.row_blocks) * 2 * kTile;
        g.blk0 = x - pair * p.blocks;
        g.n = min(p.blocks - g.blk0, x1 - x);
        g.n1 = g.q0 + kTile < p.rows ? g.n : 0;
        g.piece = static_cast<int>(blockIdx.x) - place_holder(pair * p.blocks, p.total, p.ctas);
        return g;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kRing; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 2);   // one arrival per tile
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 4);
            mbar_init(&s_full[t], 1);
            mbar_init(&s_free[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&pv_done[t], 1);
        }
        for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
        *abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
        prefetch_tensormap(&map_k);
        prefetch_tensormap(&map_v);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_launch_dependents();
    grid_dependency_wait();   // from here on global memory is read

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int base = 0;   // loads of the segments before
            for (int x = x0; x < x1 && ok;) {
                const Segment g = segment(x);
                for (int r = 0; r < 2 * g.n; ++r) {
                    const int slot = (base + r) % kRing;
                    ok = mbar_wait(&kv_empty[slot], (static_cast<uint32_t>((base + r) / kRing) & 1u) ^ 1u, abort_flag);
                    if (!ok) break;
                    mbar_arrive_expect_tx(&kv_full[slot], S::kTileBytes);
                    const bool is_v = r == 2 * g.n - 1 || (r != 0 && (r & 1) == 0);
                    const int blk = is_v ? (r == 2 * g.n - 1 ? g.n - 1 : (r - 2) / 2) : (r + 1) / 2;
                    const int row = (g.blk0 + blk) * kBlock;   // rows behind the prompt are filled with zeros by the copy engine
                    const int hfirst = is_v ? p.v_hfirst : p.k_hfirst;
                    for (int c = 0; c < D / 64; ++c) {
                        tma_load_4d(smem_kv + slot * S::kTileBytes + c * kHalf, is_v ? &map_v : &map_k, &kv_full[slot], c * 64, hfirst ? g.hk : row, hfirst ? row : g.hk, 0);
                    }
                }
                base += 2 * g.n;
                x += g.n;
            }
        }
    } else if (warp == 1 || warp == 3) {
        if (lane == 0) {
            const int t = warp == 1 ? 0 : 1;
            bool ok = true;
            int base = 0, done = 0, queries = 0;   // loads, blocks of this tile and tiles of queries of the segments before
            for (int x = x0; x < x1 && ok;) {
                const Segment g = segment(x);
                const int n_t = t == 0 ? g.n : g.n1;
                auto scores = [&](int j) -> bool {
                    const int r = base + load_of_k(j), slot = r % kRing;
                    if (done + j > 0 && !mbar_wait(&s_free[t], static_cast<uint32_t>(done + j - 1) & 1u, abort_flag)) return false;
                    if (!mbar_wait(&kv_full[slot], static_cast<uint32_t>(r / kRing) & 1u, abort_flag)) return false;
                    tc_fence_after();
                    const uint32_t qa = smem_u32(smem_q + t * S::kTileBytes), ka = smem_u32(smem_kv + slot * S::kTileBytes);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t off = (k >> 2) * kHalf + (k & 3) * 32;
                        umma_f16_ss(tmem_base + t * 128, make_smem_desc_sw128(qa + off, 16, 1024), make_smem_desc_sw128(ka + off, 16, 1024), p.idesc_s, k != 0 ? 1u : 0u);
                    }
                    umma_commit(&s_full[t]);
                    umma_commit(&kv_empty[slot]);
                    return true;
                };
                // A tile without rows hands the blocks straight back: it has to see every phase of the ring's barriers, since a wait names a
                // phase by its parity only and would take one two phases back for the one it means.
                for (int r = base; n_t == 0 && ok && r < base + 2 * g.n; ++r) {
                    ok = mbar_wait(&kv_full[r % kRing], static_cast<uint32_t>(r / kRing) & 1u, abort_flag);
                    if (ok) mbar_arrive(&kv_empty[r % kRing]);
                }
                if (n_t > 0) ok = mbar_wait(&q_full[t], static_cast<uint32_t>(queries) & 1u, abort_flag) && scores(0);
                for (int j = 0; j < n_t && ok; ++j) {
                    if (j + 1 < n_t && !(ok = scores(j + 1))) break;
                    const int r = base + load_of_v(j, g.n), slot = r % kRing;
                    ok = mbar_wait(&p_full[t], static_cast<uint32_t>(done + j) & 1u, abort_flag) &&
                         mbar_wait(&kv_full[slot], static_cast<uint32_t>(r / kRing) & 1u, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t pa = smem_u32(smem_p + t * kPBytes), va = smem_u32(smem_kv + slot * S::kTileBytes);
#pragma unroll
                    for (int k = 0; k < kBlock / 16; ++k) {
                        // V is N-contiguous: 16 keys are 16 rows of 128 bytes; with two column halves they lie kHalf apart
                        umma_f16_ss(tmem_base + 256 + t * 128, make_smem_desc_sw128(pa + (k >> 2) * kHalf + (k & 3) * 32, 16, 1024),
                                    make_smem_desc_sw128(va + k * 2048, kHalf, 1024), p.idesc_pv, (j > 0 || k != 0) ? 1u : 0u);
                    }
                    umma_commit(&pv_done[t]);
                    umma_commit(&kv_empty[slot]);
                }
                base += 2 * g.n;
                done += n_t;
                queries += n_t > 0 ? 1 : 0;
                x += g.n;
            }
        }
    } else if (warp >= 4) {
        const int t = (warp - 4) >> 2, quarter = warp & 3, r_in_tile = quarter * 32 + lane;
        uint8_t* pbuf = smem_p + t * kPBytes;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_tmem = lane_base + t * 128, o_tmem = lane_base + 256 + t * 128;
        bool ok = true;
        // m_used is the running maximum less this, so P stays below 2^(kRescale + LIFT): fp16 keeps probabilities down to 2^-31 of the
        // largest one that way, and sums of bf16 values, which may come near fp32's largest, stay in range.
        constexpr float LIFT = std::is_same<T, fp16>::value ? 7.f : -24.f;
        int done = 0, turns = 0;   // blocks of this tile, and blocks that both tiles have, of the segments before
        for (int x = x0; x < x1 && ok;) {
            const Segment g = segment(x);
            const int n_t = t == 0 ? g.n : g.n1;
            const bool both = g.n1 > 0;
            const int row = g.q0 + t * kTile + r_in_tile;
            if (n_t > 0) {
                // The tile's query rows, 16 bytes a thread; chunk c of a row sits at c ^ (row & 7) of its 128-byte line. The products over the
                // previous segment's queries are over: this warp has seen their last scores.
                for (int i = r_in_tile; i < kTile * (D / 8); i += 128) {
                    const int r = i / (D / 8), c = i - r * (D / 8), qr = g.q0 + t * kTile + r;
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (qr < p.rows) {
                        const int b = qr / p.group, h = qr - b * p.group;
                        w = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_sb + static_cast<int64_t>(g.hk * p.group + h) * p.q_sh + c * 8);
                    }
                    *reinterpret_cast<uint4*>(smem_q + t * S::kTileBytes + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) * 16)) = w;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[t]);
            }
            float m_used = -INFINITY, l_sum = 0.f;
            for (int j = 0; j < n_t; ++j) {
                if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], static_cast<uint32_t>(done + j) & 1u, abort_flag))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_tmem + c * 32, s[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_free[t]);
                const int left = p.P - (g.blk0 + j) * kBlock;   // keys of this block
                if (left < kBlock) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (c * 32 + i >= left) s[c][i] = __float_as_uint(-INFINITY);
                        }
                    }
                }
                float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) mxs[i & 3] = fmaxf(mxs[i & 3], __uint_as_float(s[c][i]));
                }
                const float mx = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3])) * p.scale_log2;
                bool rescale = false;
                float factor = 1.f;
                if (j == 0) {
                    m_used = mx - LIFT;
                } else {
                    rescale = __any_sync(0xffffffffu, mx > m_used + (kRescale + LIFT));
                    if (rescale) {
                        const float m_new = fmaxf(m_used, mx - LIFT);
                        factor = (m_used == -INFINITY) ? 0.f : exp2_approx(m_used - m_new);
                        m_used = m_new;
                        l_sum *= factor;
                    }
                }
                const float base = (m_used == -INFINITY) ? 0.f : m_used;
                // tile 0 block j, tile 1 block j, tile 0 block j + 1, ...: turns at the exponentials, as far as both tiles exist
                bool go = true;
                if (both && t == 0 && turns + j > 0) go = mbar_wait(&turn[quarter * 2], static_cast<uint32_t>(turns + j - 1) & 1u, abort_flag);
                if (both && t == 1) go = mbar_wait(&turn[quarter * 2 + 1], static_cast<uint32_t>(turns + j) & 1u, abort_flag);
                if (!__all_sync(0xffffffffu, go)) {
                    ok = false;
                    break;
                }
                float parts[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float e[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            e[u] = exp2_approx(fmaf(__uint_as_float(s[c][i + u]), p.scale_log2, -base));
                            parts[u & 3] += e[u];
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) s[c][i / 2 + u] = Pair<T>::narrow(make_float2(e[2 * u], e[2 * u + 1]));
                    }
                }
                __syncwarp();
                if (both && lane == 0) mbar_arrive(&turn[quarter * 2 + (t == 0 ? 1 : 0)]);
                if (j > 0) {   // P of the previous block has been consumed and O is at rest
                    if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[t], static_cast<uint32_t>(done + j - 1) & 1u, abort_flag))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                }
                if (rescale) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld_32x32(o_tmem + c * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                        tmem_st_32x32(o_tmem + c * 32, o);
                    }
                    tmem_st_wait();
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        const int col = c * 32 + i, chunk = (col & 63) >> 3;
                        *reinterpret_cast<uint4*>(pbuf + (col >> 6) * kHalf + r_in_tile * 128 + ((chunk ^ (r_in_tile & 7)) * 16)) =
                            make_uint4(s[c][i / 2], s[c][i / 2 + 1], s[c][i / 2 + 2], s[c][i / 2 + 3]);
                    }
                }
                l_sum += (parts[0] + parts[1]) + (parts[2] + parts[3]);
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (ok && n_t > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], static_cast<uint32_t>(done + n_t - 1) & 1u, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const int64_t at = (static_cast<int64_t>(g.piece) * p.Hkv + g.hk) * p.rows + row;
                if (row < p.rows) p.ml[at] = make_float2(m_used, l_sum);
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld_32x32(o_tmem + c * 32, o);
                    tmem_ld_wait();
                    if (row < p.rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(p.o + at * D + c * 32 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                tc_fence_before();   // O is read before the next segment's first product overwrites it
            }
            done += n_t;
            turns += both ? g.n : 0;
            x += g.n;
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_flag != 0) {
        // A wait timed out. Copies and products still in flight get time to land before shared and tensor memory are released.
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
        if (threadIdx.x == 0) atomicExch(p.status, 2u);
    }
    __syncthreads();
    if (warp == 2) tmem_dealloc(tmem_base, 512);
}

template <typename T, int D>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const PrefixParams& p, unsigned grid, cudaStream_t stream) {
    const auto kernel = prefix_attention_kernel<T, D>;
    if (cudaError_t e = tc_ensure_smem_attr(reinterpret_cast<const void*>(kernel), Smem<D>::kTotal); e != cudaSuccess) return e;
    return launch_dependent(kernel, grid, 384, Smem<D>::kTotal, stream, mk, mv, p);
}

// [P, Hkv, D] as a tensor map of 64-column x 128-row boxes. The driver wants every pitch to be a multiple of the one before it,
// so the head and row dimensions are ordered by pitch.
bool map_of(const TensorView& t, CUtensorMap* map, int* hfirst) {
    const int64_t P = t.shape[0], H = t.shape[1], D = t.shape[2];
    const int64_t pr = P == 1 ? (H == 1 ? D : t.stride[1] * H) : t.stride[0], ph = H == 1 ? (P == 1 ? D : t.stride[0] * P) : t.stride[1];
    const bool hf = ph <= pr;
    *hfirst = hf ? 1 : 0;
    const int64_t dims[4] = {D, hf ? H : P, hf ? P : H, 1}, pitches[3] = {hf ? ph : pr, hf ? pr : ph, hf ? pr * P : ph * H};
    return tc_encode_map4(reinterpret_cast<::CUtensorMap_st*>(map), t.dtype, t.data, dims, pitches, hf ? 1 : kBlock, hf ? kBlock : 1);
}

// CTAs the blocks are dealt to: a multiple of the pairs (each pair in as many equal ranges), or all SMs (ranges that cross from one pair
// to the next) where no multiple comes near. All SMs pay only for a large gap, because the power limit lowers the clock with
// every SM that multiplies. Whole calls of head dim 128 in us: 300 sequences x 64 heads (80 pairs) behind 8192 tokens 135 on 148
// SMs, 167 on 80; 256 behind 32768 (64 pairs) 290 on 148 as on 128; 128 behind 16384 (32 pairs) 112 and 100; 64 x 32 heads (8 pairs)
// behind 8192 53 and 42. The constants are those of head dim 128, in microseconds: 2 for a block of a CTA (two 128 x 128 x D products for
// each of two tiles, or 64 KiB at a 148th of the memory rate), 4 for a segment's start and end, 5 TB/s for the fp32 pieces, written and
// read back. At head dim 64, where a block takes less, the same four batches took 113 and 158, 257 and 279 (the choice, 8 % behind
// the best), 88 either way, 40 and 35; in three more batches of either head dim the choice was the best of all that were tried.
int plan(int64_t pairs, int64_t blocks, int64_t piece_bytes, int sms) {
    const int64_t total = pairs * blocks;
    auto cost = [&](int64_t ctas) {
        const double pieces = static_cast<double>(ctas) / pairs + (ctas % pairs == 0 ? 0.0 : 1.0);
        const double segments = ctas % pairs == 0 ? 1.0 : static_cast<double>(pairs) / ctas + 1.0;
        return 2.0 * ((total + ctas - 1) / ctas) + 4.0 * segments + pieces * piece_bytes * 2 / 5e6;
    };
    const int64_t all = total < sms ? total : sms;
    int64_t best = 0;
    for (int64_t ctas = pairs; ctas <= all; ctas += pairs) {
        if (best == 0 || cost(ctas) < cost(best)) best = ctas;
    }
    if (best == 0 || 1.25 * cost(all) < cost(best)) best = all;
    return static_cast<int>(best);
}

}  // namespace

diopiError_t prefix_attention(const char* name, diopiContextHandle_t ctx, const TensorView& q, const TensorView& k, const TensorView& v, float scale_log2,
                              PrefixParts* parts, cudaStream_t stream) {
    const int64_t B = q.shape[0], Hq = q.shape[1], D = q.shape[2], P = k.shape[0], Hkv = k.shape[1], group = Hq / Hkv, rows = B * group;
    PrefixParams p = {};
    p.q = q.data; p.q_sb = q.stride[0]; p.q_sh = q.stride[1];
    p.rows = static_cast<int>(rows); p.group = static_cast<int>(group); p.Hkv = static_cast<int>(Hkv); p.P = static_cast<int>(P);
    p.row_blocks = static_cast<int>((rows + 2 * kTile - 1) / (2 * kTile));
    p.scale_log2 = scale_log2;
    const int64_t blocks = (P + kBlock - 1) / kBlock, pairs = Hkv * p.row_blocks;
    B200_CHECK(pairs * blocks < 0x7fffffffLL, "%s: too many query rows", name);
    p.blocks = static_cast<int>(blocks);
    p.total = static_cast<int>(pairs * blocks);
    p.ctas = plan(pairs, blocks, rows * Hkv * (D * 4 + 8), sm_count());
    const int64_t splits = (blocks - 1) * p.ctas / p.total + 2;   // pieces a pair has at most
    const int fmt = q.dtype == diopi_dtype_bfloat16 ? 1 : 0;
    p.idesc_s = make_idesc_f16(fmt, false, kTile, kBlock);
    p.idesc_pv = make_idesc_f16(fmt, true, kTile, static_cast<int>(D));
    p.status = tc_status_word();
    B200_CHECK(p.status != nullptr, "%s: cannot allocate the status word", name);
    CUtensorMap mk, mv;
    B200_CHECK(map_of(k, &mk, &p.k_hfirst) && map_of(v, &mv, &p.v_hfirst), "%s: cuTensorMapEncodeTiled rejected the prefix", name);
    diopiTensorHandle_t ws = nullptr;
    void* ptr = nullptr;
    B200_CHECK(diopiRequireBuffer(ctx, &ws, splits * Hkv * rows * (D * 4 + 8), diopi_device) == diopiSuccess && ws != nullptr, "%s: workspace allocation failed", name);
    B200_CHECK(diopiGetTensorData(ws, &ptr) == diopiSuccess && ptr != nullptr, "%s: workspace has no data pointer", name);
    p.o = static_cast<float*>(ptr);
    p.ml = reinterpret_cast<float2*>(p.o + splits * Hkv * rows * D);
    const unsigned grid = static_cast<unsigned>(p.ctas);
    cudaError_t e;
    if (fmt == 1) e = D == 128 ? launch<bf16, 128>(mk, mv, p, grid, stream) : launch<bf16, 64>(mk, mv, p, grid, stream);
    else e = D == 128 ? launch<fp16, 128>(mk, mv, p, grid, stream) : launch<fp16, 64>(mk, mv, p, grid, stream);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        B200_FAIL("%s: kernel launch failed: %s", name, cudaGetErrorString(e));
    }
    parts->o = p.o; parts->ml = p.ml; parts->rows = rows;
    parts->splits = static_cast<int>(splits); parts->blocks = p.blocks; parts->total = p.total; parts->ctas = p.ctas; parts->row_blocks = p.row_blocks;
    return diopiSuccess;
}

}  // namespace b200
