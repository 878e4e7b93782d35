// Device helpers of the 8-bit cache's kernels.
#pragma once

#include "nh_kv8.h"
#include "nh_kv_attend.h"

namespace nh {

// A chunk of the cache: where its parts lie, in bytes from its start.
template <int WK, int WV>
struct Kv8Lay {
    static constexpr int NJ = WK / 64, NV = WV / 16;
    static constexpr uint32_t VALUES = 64 * WK, RECORD = 64 * (WK + WV), CHUNK = RECORD + sizeof(Kv8Record);
    // dims 64 j + 16 kg + 0 .. 15 of position 16 t + o
    static __device__ __forceinline__ uint32_t k_piece(int t, int j, int lane) { return (uint32_t)(t * NJ + j) * 1024 + lane * 16; }
    // dim 16 n + o, all positions of lane (o, kg); 4 positions of block t at + 4 t
    static __device__ __forceinline__ uint32_t v_piece(int n, int lane) { return VALUES + (uint32_t)n * 1024 + lane * 16; }
};

__device__ __forceinline__ uint8_t* kv8_block(const Kv8View& c, int page, int layer, int head) {
    return c.data + (((size_t)page * c.layers + layer) * c.heads + head) * c.block();
}

typedef KaSpanOf<KV8_CHUNK> Ka8Span;

// Whether rows at positions lo .. hi see any of the 16 from `block` on.
__device__ __forceinline__ bool ka8_sees(int block, int lo, int hi, int sink, int ring) {
    return (block <= hi) & ((block < sink) | (block + 15 > lo - ring));
}

// Four codes as f16: bytes 0, 1 and 2, 3.
__device__ __forceinline__ h2 codes2(uint32_t w, uint32_t which) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, which)) + (_Float16)-1152.0f;
}
__device__ __forceinline__ h8 codes8(uint32_t a, uint32_t b) {
    const h2 w = codes2(a, 0x04010400u), x = codes2(a, 0x04030402u), y = codes2(b, 0x04010400u), z = codes2(b, 0x04030402u);
    return h8{w[0], w[1], x[0], x[1], y[0], y[1], z[0], z[1]};
}
// The same, 128 more and 2^-24 times as large: a byte alone is an f16 subnormal,
// which the matrix instructions take exactly.
__device__ __forceinline__ uint32_t bytes2(uint32_t w, uint32_t which) { return __builtin_amdgcn_perm(w, w, which); }
__device__ __forceinline__ h8 bytes8(uint32_t a, uint32_t b) {
    const u32x4 w = {bytes2(a, 0x0c010c00u), bytes2(a, 0x0c030c02u), bytes2(b, 0x0c010c00u), bytes2(b, 0x0c030c02u)};
    return __builtin_bit_cast(h8, w);
}

}  // namespace nh
