// The paged caches' state on the device, and copies of whole pages.
#include "nh_kv_device.h"

namespace nh {

// ------------------------------------------------------------------ state
__global__ __launch_bounds__(512) void k_kv_patch(int* __restrict__ state, KvPatch p) {
    const int i = threadIdx.x;
    if (i < p.n) state[p.at[i]] = p.v[i];
}

hipError_t launch_kv_patch(int* state, const KvPatch& p, hipStream_t s) {
    static_assert(KvPatch::MAX <= 512 && sizeof(KvPatch) <= 4000, "one block, one argument segment");
    hipLaunchKernelGGL(k_kv_patch, dim3(1), dim3(512), 0, s, state, p);
    return hipGetLastError();
}

// ------------------------------------------------------------------ pages
// Whole pages, every layer and head: 16 bytes a thread (8 pages of 20 layers, 2.6
// MB in and out, 3.0 us: a launch's latency).
__global__ __launch_bounds__(256) void k_kv_pairs(uint8_t* data, size_t bytes, KvPairs p) {
    const size_t n = bytes / 16;
    const uint4* from = reinterpret_cast<const uint4*>(data) + (size_t)p.from[blockIdx.y] * n;
    uint4* to = reinterpret_cast<uint4*>(data) + (size_t)p.to[blockIdx.y] * n;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) to[i] = from[i];
}

hipError_t launch_kv_pairs(uint8_t* data, size_t page_bytes, const KvPairs& p, hipStream_t s) {
    static_assert(sizeof(KvPairs) <= 3900, "the argument segment");
    const size_t blocks = (page_bytes / 16 + 255) / 256;
    hipLaunchKernelGGL(k_kv_pairs, dim3((unsigned)(blocks < 1024 ? blocks : 1024), p.n), dim3(256), 0, s, data, page_bytes, p);
    return hipGetLastError();
}

}  // namespace nh
