// What the translation units share on the host: status codes of launches, and what atlas_b200.cu knows of the device.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "atlas_b200.h"

namespace atlas {

static inline int cuda_status(cudaError_t e) { return e == cudaSuccess ? ATLAS_B200_OK : ATLAS_B200_ERR_CUDA_BASE - int(e); }
static inline int launch_status() { return cuda_status(cudaGetLastError()); }
// A launch of a kernel that begins with pdl_wait(): it may start while its predecessor in the stream finishes.
template <typename... P, typename... A>
static int launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}
static inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// atlas_b200.cu
int device_sm_count();
bool device_is_sm100();           // and tensor maps can be encoded
bool encode_tensor_map(CUtensorMap* map, CUtensorMapDataType dt, uint32_t rank, const void* base, const uint64_t* dims, const uint64_t* strides,
                       const uint32_t* box, CUtensorMapSwizzle swz);
// cache_ops.cu: the status word of its kernels (they cannot share the other unit's)
int cache_device_status(uint32_t* out_word, int clear);

}  // namespace atlas
