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

__device__ __forceinline__ float f16_value(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Where the step and the low of (slot, group) lie in a block, in bytes from
// its start: keys, values.
__device__ __forceinline__ uint32_t kv4_k_scale(const Kv4View& c, int slot, int g) { return c.ks_off() + 2 * (slot * c.groups() + g); }
__device__ __forceinline__ uint32_t kv4_k_low(const Kv4View& c, int slot, int g) { return c.kl_off() + 2 * (slot * c.groups() + g); }
__device__ __forceinline__ uint32_t kv4_v_scale(const Kv4View& c, int slot, int g) { return c.vs_off() + 2 * (slot * c.groups() + g); }
__device__ __forceinline__ uint32_t kv4_v_low(const Kv4View& c, int slot, int g) {
    return c.vl_off() + 2 * (((slot >> 2) * c.groups() + g) * 4 + (slot & 3));
}
__device__ __forceinline__ uint16_t& kv4_half(uint8_t* blk, uint32_t at) { return *reinterpret_cast<uint16_t*>(blk + at); }
__device__ __forceinline__ uint16_t kv4_half(const uint8_t* blk, uint32_t at) { return *reinterpret_cast<const uint16_t*>(blk + at); }

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
