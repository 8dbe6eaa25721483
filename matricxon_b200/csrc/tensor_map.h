// The driver's encoder of tensor maps, for every file that makes some (gemm_tcgen05.cu, attention_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

typedef CUresult (*MxEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                    const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                    CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Null where the driver has none. The first call of any thread looks it up, once, while others wait. The encoder wants a
// context on the thread that calls it, which a thread that has made no runtime call yet does not have (it answers 201,
// "invalid context"): each thread's first call here gives it that of its device.
inline MxEncodeTiledFn mx_encode_tiled() {
    static const MxEncodeTiledFn encode = [] {
        void* found = nullptr;
        cudaDriverEntryPointQueryResult query;
        const bool there = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &found, cudaEnableDefault, &query) == cudaSuccess &&
                           query == cudaDriverEntryPointSuccess;
        return there ? reinterpret_cast<MxEncodeTiledFn>(found) : nullptr;
    }();
    static thread_local bool has_context = false;
    if (!has_context) {
        int device = 0;
        has_context = cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess;
    }
    return encode;
}
