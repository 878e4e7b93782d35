// Device helpers of the 4-bit cache's kernels.
#pragma once

#include "nh_kv4.h"
#include "nh_kv_device.h"

namespace nh {

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

__device__ __forceinline__ uint8_t* kv4_block(const Kv4View& c, int page, int layer, int head) {
    return c.data + (((size_t)page * c.layers + layer) * c.heads + head) * c.block();
}

}  // namespace nh
