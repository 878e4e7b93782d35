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

// Where the things of position `slot` (0 .. 31) of a chunk lie, in bytes from
// the chunk's start: the dword of key dims 8 t .. 8 t + 7; the byte of value
// dims 2 x, 2 x + 1; a group's steps and lows.
template <int W, int G>
struct Kv4Lay {
    static constexpr int NG = W / G, NB = W / 64, NJ = W / 32;
    static constexpr uint32_t CHUNK = 32 * (W + 8 * NG);
    static __device__ __forceinline__ uint32_t lane_dword(int lane, int u) { return (uint32_t)(u >> 2) * 1024 + lane * 16 + (u & 3) * 4; }
    static __device__ __forceinline__ uint32_t k_dword(int slot, int t) {
        return lane_dword((t & 3) * 16 + (slot & 15), (slot >> 4) * NJ + (t >> 2));
    }
    static __device__ __forceinline__ uint32_t v_half(int slot, int o, int b) {
        return 16 * W + lane_dword((slot >> 2 & 3) * 16 + o, (slot >> 4) * NJ + (slot >> 1 & 1) * NB + b) + 2 * (slot & 1);
    }
    static __device__ __forceinline__ uint32_t v_byte(int slot, int x) { return v_half(slot, x & 15, x >> 5) + (x >> 4 & 1); }
    static __device__ __forceinline__ uint32_t k_step(int slot, int g) { return 32 * W + 2 * (slot * NG + g); }
    static __device__ __forceinline__ uint32_t k_low(int slot, int g) { return 32 * W + 64 * NG + 2 * (slot * NG + g); }
    static __device__ __forceinline__ uint32_t v_step(int slot, int g) {
        return 32 * W + 128 * NG + 2 * (((slot >> 2) * NG + g) * 4 + (slot & 3));
    }
    static __device__ __forceinline__ uint32_t v_low(int slot, int g) {
        return 32 * W + 192 * NG + 2 * (((slot >> 2) * NG + g) * 4 + (slot & 3));
    }
};
__device__ __forceinline__ uint32_t& kv4_word(uint8_t* p, uint32_t at) { return *reinterpret_cast<uint32_t*>(p + at); }
__device__ __forceinline__ uint32_t kv4_word(const uint8_t* p, uint32_t at) { return *reinterpret_cast<const uint32_t*>(p + at); }
__device__ __forceinline__ uint16_t& kv4_half(uint8_t* p, uint32_t at) { return *reinterpret_cast<uint16_t*>(p + at); }
__device__ __forceinline__ uint16_t kv4_half(const uint8_t* p, uint32_t at) { return *reinterpret_cast<const uint16_t*>(p + at); }

// The entry whose units (ascending, from first[i]) hold `unit`; the wavefront
// together, unit the same in every lane.
__device__ __forceinline__ int kv4_span(const int* __restrict__ first, int n, int unit, int lane) {
    int b = 0;
    for (int i = 0; i < n; i += 64) b += __popcll(__ballot(i + lane < n && first[i + lane + 1] <= unit));
    return b < n ? b : n - 1;
}
// The batch entry whose units(entry) hold `unit`, which becomes that entry's own;
// c.nb past the last.  The wavefront together.
template <class F>
__device__ __forceinline__ int kv4_find(const Kv4View& c, int& unit, int lane, F units) {
    int b = 0;
    for (int i = 0; i < c.nb; i += 64) {
        int sum = 0;
        if (i + lane < c.nb) {
            const int4 e = reinterpret_cast<const int4*>(c.batch)[i + lane];
            sum = units(Kv4Entry{e.x, e.y, e.z, e.w});
        }
#pragma unroll
        for (int h = 1; h < 64; h <<= 1) {
            const int x = __shfl_up(sum, h, 64);
            if (lane >= h) sum += x;
        }
        const int skip = __popcll(__ballot(sum <= unit && i + lane < c.nb));
        const int last = __shfl(sum, skip ? skip - 1 : 0, 64);
        b += skip;
        if (skip) unit -= last;
        if (skip < 64) break;
    }
    unit = __builtin_amdgcn_readfirstlane(unit);
    return __builtin_amdgcn_readfirstlane(b);
}
// The batch on the device is of the rows that this launch was made for: not so
// where a captured launch is replayed after an extend of other rows, or when
// the batch is over, whose grid and plan fit nothing that is there.
__device__ __forceinline__ bool kv4_current(const Kv4View& c) {
    const int2 s = *reinterpret_cast<const int2*>(c.batch - 4);
    return s.x == c.shape[0] && s.y == c.shape[1];
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
