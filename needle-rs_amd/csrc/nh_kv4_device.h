// Device helpers of the 4-bit cache's kernels.
#pragma once

#include "nh_device.h"
#include "nh_kv4.h"

namespace nh {

// Elements by type tag (Kv4Type), widened to f32.
template <int TYPE>
struct Kv4Elem;
template <>
struct Kv4Elem<KV4_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(const T* p) { return *p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = v; }
};
template <>
struct Kv4Elem<KV4_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = (_Float16)v; }
};
template <>
struct Kv4Elem<KV4_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = (__bf16)v; }
};

// Half of a scale dword: step (low half) or low (high half) as f32.
__device__ __forceinline__ float kv4_step(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)w); }
__device__ __forceinline__ float kv4_low(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }

// The batch entry that holds `row`: the count of entries that end at or
// before it (row0 ascends; an entry without rows is passed over).  One load
// for each 64 entries, the wavefront together; row is the same in every lane.
__device__ __forceinline__ int kv4_entry(const int* __restrict__ row0, int nb, int row, int lane) {
    int b = 0;
    for (int i = 0; i < nb; i += 64)
        b += __popcll(__ballot(i + lane < nb && row0[i + lane + 1] <= row));
    return b < nb ? b : nb - 1;
}

// Where position `pos` of sequence `seq` lies: its page id, or -1 outside the
// table (a state that no extend leaves).
__device__ __forceinline__ int kv4_page(const Kv4View& c, int seq, int pos) {
    if ((unsigned)(pos >> c.page_log2) >= (unsigned)c.table_ld) return -1;
    const int pg = c.table[(size_t)seq * c.table_ld + (pos >> c.page_log2)];
    return (unsigned)pg < (unsigned)c.pages ? pg : -1;
}

__device__ __forceinline__ uint8_t* kv4_block(const Kv4View& c, int page, int layer, int head) {
    return c.data + (((size_t)page * c.layers + layer) * c.heads + head) * c.block();
}

}  // namespace nh
