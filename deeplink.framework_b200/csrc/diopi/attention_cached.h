// What the attention over ragged caches (attention_cached.cu) and the attention over a shared prompt (attention_prefix.cu) hand over.
#pragma once

#include <cuda_runtime.h>

#include "common.h"

namespace b200 {

// Softmax pieces over the rows of a shared prompt, cut into `splits` ranges of keys: for range s, key head h and query row
// r = sequence * group + head in group: o[((s * Hkv + h) * rows + r) * D ..], unnormalised, relative to the maximum ml.x (log2);
// ml.y is the sum of the exponentials.
struct PrefixParts {
    const float* o = nullptr;
    const float2* ml = nullptr;
    int64_t rows = 0;
    int splits = 0;
};

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
