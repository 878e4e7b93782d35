// What the paged caches' attention kernels share: lane exchanges, spans.
#pragma once

#include <type_traits>

#include "nh_kv_device.h"

namespace nh {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float KA_LOG2E = 1.44269504088896340736f;

// Maximum and sum over the four lane groups of a row's lane.
__device__ __forceinline__ float groups_max(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const float y = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const uint32_t z = __builtin_bit_cast(uint32_t, y);
    auto b = __builtin_amdgcn_permlane16_swap(z, z, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const float y = __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
    const uint32_t z = __builtin_bit_cast(uint32_t, y);
    auto b = __builtin_amdgcn_permlane16_swap(z, z, false, false);
    return __builtin_bit_cast(float, (uint32_t)b[0]) + __builtin_bit_cast(float, (uint32_t)b[1]);
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

struct KaPlan {
    int splits;      // key ranges of a sequence; more than one: partial results go to the workspace
    int tiles_each;  // row tiles of every sequence when they are equal, else 0
    int aligned;     // rows of q can be read 8 elements at a time
    int out_aligned; // rows of out can be written 4 elements at a time
};

// The chunks of CHUNK keys that a tile of rows at positions lo .. hi sees: [0, ns) and [w, n).
template <int CHUNK>
struct KaSpanOf {
    int ns, w, n;
    __device__ __forceinline__ KaSpanOf(int lo, int hi, int sink, int ring) {
        n = (hi + CHUNK) / CHUNK;  // (hi -1: none)
        ns = 0, w = 0;
        if (ring) {
            ns = min((int)(((int64_t)sink + CHUNK - 1) / CHUNK), n);
            w = max(ns, max(0, lo - ring + 1) / CHUNK);
        }
    }
    __device__ __forceinline__ int count() const { return ns + n - w; }
    __device__ __forceinline__ int at(int i) const { return i < ns ? i : i - ns + w; }
};

__device__ __forceinline__ float halves_max(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
}

}  // namespace nh
