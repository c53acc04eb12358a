// What the attention over ragged caches (attention_cached.cu) and the attention over a shared prompt (attention_prefix.cu) hand over.
#pragma once

#include <cuda_runtime.h>

#include "common.h"

namespace b200 {

// Softmax pieces over the rows of a shared prompt. The blocks of all (key head h, row block) pairs are dealt to `ctas` CTAs in equal
// ranges; piece i of a pair is what the i-th CTA with blocks of it has. For query row r = sequence * group + head in group:
// o[((i * Hkv + h) * rows + r) * D ..], unnormalised, relative to the maximum ml.x (log2); ml.y is the sum of the exponentials.
constexpr int kPrefixRows = 256;       // query rows of a row block
struct PrefixParts {
    const float* o = nullptr;
    const float2* ml = nullptr;
    int64_t rows = 0;
    int splits = 0;                    // pieces a pair has at most; 0: no prefix
    int blocks = 0, total = 0, ctas = 0, row_blocks = 0;
};

// The CTA of place `place` among `total` places dealt to `ctas` CTAs; CTA c has [total c / ctas, total (c + 1) / ctas).
__host__ __device__ __forceinline__ int place_holder(int place, int total, int ctas) { return static_cast<int>(((static_cast<int64_t>(place) + 1) * ctas - 1) / total); }

// A launch that may set itself up while the kernel before it in the stream ends; the kernel waits (grid_dependency_wait) before it
// touches global memory.
template <typename... Params, typename... Args>
cudaError_t launch_dependent(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// q [B, Hq, D], k / v [P, Hkv, D], P > 0, checked by the caller. The pieces lie in workspace of `ctx`.
diopiError_t prefix_attention(const char* name, diopiContextHandle_t ctx, const TensorView& q, const TensorView& k, const TensorView& v, float scale_log2,
                              PrefixParts* parts, cudaStream_t stream);

}  // namespace b200
