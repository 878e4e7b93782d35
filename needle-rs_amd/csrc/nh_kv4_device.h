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

// Where things of position `slot` of a page lie in its block, in bytes from the
// block's start: the dword of key dims 8 t .. 8 t + 7, the half of value dims
// 64 b + 16 i + o, the group's steps and lows.
__device__ __forceinline__ uint32_t kv4_chunk_at(const Kv4View& c, int slot) { return (uint32_t)(slot >> 5) * c.chunk(); }
__device__ __forceinline__ uint32_t kv4_lane_dword(int lane, int u) { return (uint32_t)(u >> 2) * 1024 + lane * 16 + (u & 3) * 4; }
__device__ __forceinline__ uint32_t kv4_k_dword(const Kv4View& c, int slot, int t) {
    return kv4_chunk_at(c, slot) + kv4_lane_dword((t & 3) * 16 + (slot & 15), (slot >> 4 & 1) * (c.width / 32) + (t >> 2));
}
__device__ __forceinline__ uint32_t kv4_v_half(const Kv4View& c, int slot, int o, int b) {
    return kv4_chunk_at(c, slot) + 16 * c.width +
           kv4_lane_dword((slot >> 2 & 3) * 16 + o, (slot >> 4 & 1) * (c.width / 32) + (slot >> 1 & 1) * (c.width / 64) + b) +
           2 * (slot & 1);
}
__device__ __forceinline__ uint32_t kv4_scale_at(const Kv4View& c, int slot, int array) {
    return kv4_chunk_at(c, slot) + 32 * c.width + array * 64 * c.groups();
}
__device__ __forceinline__ uint32_t kv4_k_scale(const Kv4View& c, int slot, int g) {
    return kv4_scale_at(c, slot, 0) + 2 * ((slot & 31) * c.groups() + g);
}
__device__ __forceinline__ uint32_t kv4_k_low(const Kv4View& c, int slot, int g) {
    return kv4_scale_at(c, slot, 1) + 2 * ((slot & 31) * c.groups() + g);
}
__device__ __forceinline__ uint32_t kv4_v_scale(const Kv4View& c, int slot, int g) {
    return kv4_scale_at(c, slot, 2) + 2 * ((slot & 31) * c.groups() + g);
}
__device__ __forceinline__ uint32_t kv4_v_low(const Kv4View& c, int slot, int g) {
    return kv4_scale_at(c, slot, 3) + 2 * (((slot >> 2 & 7) * c.groups() + g) * 4 + (slot & 3));
}
__device__ __forceinline__ uint32_t& kv4_word(uint8_t* blk, uint32_t at) { return *reinterpret_cast<uint32_t*>(blk + at); }
__device__ __forceinline__ uint32_t kv4_word(const uint8_t* blk, uint32_t at) { return *reinterpret_cast<const uint32_t*>(blk + at); }
__device__ __forceinline__ uint16_t& kv4_half(uint8_t* blk, uint32_t at) { return *reinterpret_cast<uint16_t*>(blk + at); }
__device__ __forceinline__ uint16_t kv4_half(const uint8_t* blk, uint32_t at) { return *reinterpret_cast<const uint16_t*>(blk + at); }

// The entry that holds `row`, of entries whose rows end at ends[i * stride]: the
// count of those that end at or before it (an entry without rows is passed
// over).  One load for each 64 entries, the wavefront together; row is the same
// in every lane.
__device__ __forceinline__ int kv4_entry(const int* __restrict__ ends, int stride, int n, int row, int lane) {
    int b = 0;
    for (int i = 0; i < n; i += 64) b += __popcll(__ballot(i + lane < n && ends[(i + lane) * stride] <= row));
    return b < n ? b : n - 1;
}
__device__ __forceinline__ Kv4Entry kv4_batch(const Kv4View& c, int b) {
    const int4 e = reinterpret_cast<const int4*>(c.batch)[b];
    return Kv4Entry{e.x, e.y, e.z, e.w};
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
