// The 4-bit cache's rows and pages: storing and reading rows, copying pages,
// closing sequences up.  The layout and the format are in nh_kv4.h.
#include "nh_kv4_device.h"

namespace nh {

// ------------------------------------------------------------------ state
__global__ __launch_bounds__(512) void k_kv4_patch(int* __restrict__ state, Kv4Patch p) {
    const int i = threadIdx.x;
    if (i < p.n) state[p.at[i]] = p.v[i];
}

hipError_t launch_kv4_patch(int* state, const Kv4Patch& p, hipStream_t s) {
    static_assert(Kv4Patch::MAX <= 512 && sizeof(Kv4Patch) <= 4000, "one block, one argument segment");
    hipLaunchKernelGGL(k_kv4_patch, dim3(1), dim3(512), 0, s, state, p);
    return hipGetLastError();
}

// ------------------------------------------------------------------- rows
// Of one group: low, step and the reciprocal the codes are taken with.
struct Kv4Group {
    uint16_t sb, lb;  // step and low as stored
    float low, inv;   // inv 0: every code is 0
};
__device__ __forceinline__ Kv4Group kv4_group(float mn, float mx, bool bad) {
    const _Float16 low = (_Float16)mn;
    // The product is rounded to f32 and then to f16, as the format says; the
    // empty asm keeps the two apart (v_fma_mixlo_f16 would round once).
    float wide = (mx - mn) * bits_f32(0x3d888889u);  // f32(1/15)
    asm("" : "+v"(wide));
    const _Float16 step = (_Float16)wide;
    Kv4Group g;
    g.low = (float)low;
    g.inv = step > (_Float16)0.0f ? 1.0f / (float)step : 0.0f;
    g.sb = bad ? (uint16_t)0x7e00u : __builtin_bit_cast(uint16_t, step);
    g.lb = bad ? (uint16_t)0 : __builtin_bit_cast(uint16_t, low);
    if (bad) g.inv = 0.0f;
    return g;
}
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Group& g) {
    const float c = rintf((x - g.low) * g.inv);
    return (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f);
}

// One row of one head by 16 lanes, keys: dword t (dims 8 t ..) by lane t % 16;
// the group's range over 4 or 8 neighbouring lanes.
template <int TYPE, int W>
__device__ __forceinline__ void kv4_store_k(const Kv4View& c, const typename Kv4Elem<TYPE>::T* __restrict__ x, uint8_t* blk,
                                            int slot, int lane) {
    const int l = lane & 15, per = c.group / 8;
#pragma unroll
    for (int t0 = 0; t0 < W / 8; t0 += 16) {
        const int t = t0 + l;
        float v[8];
        float mn = __builtin_inff(), mx = -__builtin_inff();
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = t * 8 + e < c.dk;
            const float r = in ? Kv4Elem<TYPE>::get(x + t * 8 + e) : 0.0f;
            bad |= !(fabsf(r) < __builtin_inff());
            v[e] = fminf(fmaxf(r, -65504.0f), 65504.0f);
            if (in) mn = fminf(mn, v[e]), mx = fmaxf(mx, v[e]);
        }
        int nb = bad;
#pragma unroll
        for (int h = 1; h < 8; h <<= 1) {
            if (h * 8 >= c.group) break;
            mn = fminf(mn, lane_xor(mn, h, lane));
            mx = fmaxf(mx, lane_xor(mx, h, lane));
            nb |= __float_as_int(lane_xor(__int_as_float(nb), h, lane));
        }
        if (mn > mx) mn = mx = 0.0f;  // a group of padding
        const Kv4Group g = kv4_group(mn, mx, nb != 0);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (t * 8 + e < c.dk) w |= kv4_code(v[e], g) << (4 * ((e & 1) * 4 + (e >> 1)));
        if (t < W / 8) {
            kv4_word(blk, kv4_k_dword(c, slot, t)) = w;
            if (t % per == 0) {
                kv4_half(blk, kv4_k_scale(c, slot, t / per)) = g.sb;
                kv4_half(blk, kv4_k_low(c, slot, t / per)) = g.lb;
            }
        }
    }
}

// Values: lane o holds dims 16 i + o; the group's range over i and the 16 lanes.
template <int TYPE, int W>
__device__ __forceinline__ void kv4_store_v(const Kv4View& c, const typename Kv4Elem<TYPE>::T* __restrict__ x, uint8_t* blk,
                                            int slot, int lane) {
    constexpr int NB = W / 64;
    const int o = lane & 15;
    uint16_t half[NB] = {};
    float v[W / 16];
#pragma unroll
    for (int i = 0; i < W / 16; ++i) v[i] = 16 * i + o < c.dv ? Kv4Elem<TYPE>::get(x + 16 * i + o) : 0.0f;
    // `gi` dims of each lane to a group: 2 or 4
    auto group = [&](int i0, int gi) {
        float mn = __builtin_inff(), mx = -__builtin_inff();
        int bad = 0;
#pragma unroll
        for (int i = i0; i < i0 + gi; ++i) {
            bad |= !(fabsf(v[i]) < __builtin_inff());
            v[i] = fminf(fmaxf(v[i], -65504.0f), 65504.0f);
            if (16 * i + o < c.dv) mn = fminf(mn, v[i]), mx = fmaxf(mx, v[i]);
        }
#pragma unroll
        for (int h = 1; h < 16; h <<= 1) {
            mn = fminf(mn, lane_xor(mn, h, lane));
            mx = fmaxf(mx, lane_xor(mx, h, lane));
            bad |= __float_as_int(lane_xor(__int_as_float(bad), h, lane));
        }
        if (mn > mx) mn = mx = 0.0f;
        const Kv4Group g = kv4_group(mn, mx, bad != 0);
#pragma unroll
        for (int i = i0; i < i0 + gi; ++i)
            if (16 * i + o < c.dv) half[i / 4] |= (uint16_t)(kv4_code(v[i], g) << (4 * (i & 3)));
        if (o == 0) {
            kv4_half(blk, kv4_v_scale(c, slot, i0 / gi)) = g.sb;
            kv4_half(blk, kv4_v_low(c, slot, i0 / gi)) = g.lb;
        }
    };
    if (c.group == 32) {
#pragma unroll
        for (int g = 0; g < W / 32; ++g) group(2 * g, 2);
    } else {
#pragma unroll
        for (int g = 0; g < W / 64; ++g) group(4 * g, 4);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) kv4_half(blk, kv4_v_half(c, slot, o, b)) = half[b];
}

// A wavefront takes four heads' keys, or values, of one row.
template <int TYPE, int W>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4View c, int layer, const typename Kv4Elem<TYPE>::T* __restrict__ k,
                                                    const typename Kv4Elem<TYPE>::T* __restrict__ v, int64_t ldk,
                                                    int64_t ldv) {
    const int lane = threadIdx.x & 63;
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t quads = (c.heads + 3) / 4;
    const int row = (int)(w / (2 * quads));
    const uint32_t u = w % (2 * quads);
    if (row >= c.rows) return;
    const Kv4Entry e = kv4_batch(c, c.each ? row / c.each : kv4_entry(c.batch + 2, 4, c.nb, row, lane));
    const int pos = e.len - e.row1 + row;
    const int pg = pos < 0 ? -1 : kv4_page(c, e.seq, pos);
    const int head = (int)(u % quads) * 4 + (lane >> 4);
    if (pg < 0 || head >= c.heads) return;
    uint8_t* blk = kv4_block(c, pg, layer, head);
    const int slot = pos & (c.page() - 1);
    if (u < quads)
        kv4_store_k<TYPE, W>(c, k + row * ldk + (int64_t)head * c.dk, blk, slot, lane);
    else
        kv4_store_v<TYPE, W>(c, v + row * ldv + (int64_t)head * c.dv, blk, slot, lane);
}

template <int TYPE>
static hipError_t append_typed(const Kv4View& c, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv,
                               hipStream_t s) {
    typedef const typename Kv4Elem<TYPE>::T* P;
    const uint64_t blocks = ((uint64_t)c.rows * 2 * ((c.heads + 3) / 4) + 3) / 4;
    if (blocks > 0x3fffffffu) return hipErrorInvalidValue;
    auto kern = c.width == 64 ? k_kv4_append<TYPE, 64> : c.width == 128 ? k_kv4_append<TYPE, 128> : k_kv4_append<TYPE, 256>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, s, c, layer, (P)k, (P)v, ldk, ldv);
    return hipGetLastError();
}

hipError_t launch_kv4_append(const Kv4View& c, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int type,
                             hipStream_t s) {
    return type == KV4_F32   ? append_typed<KV4_F32>(c, layer, k, v, ldk, ldv, s)
           : type == KV4_F16 ? append_typed<KV4_F16>(c, layer, k, v, ldk, ldv, s)
                             : append_typed<KV4_BF16>(c, layer, k, v, ldk, ldv, s);
}

// The values held, a wavefront as in the store.  step * code is exact in f32,
// so the fma rounds once, as the product and the sum do.
template <int TYPE, int W>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4View c, int layer0, Kv4Spans p, int64_t rows, int64_t row_at,
                                                  typename Kv4Elem<TYPE>::T* __restrict__ k,
                                                  typename Kv4Elem<TYPE>::T* __restrict__ v) {
    const int lane = threadIdx.x & 63, o = lane & 15;
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t quads = (c.heads + 3) / 4;
    const int row = (int)(w / (2 * quads));
    const uint32_t u = w % (2 * quads);
    if (row >= p.row0[p.n]) return;
    const int b = kv4_entry(p.row0 + 1, 1, p.n, row, lane);
    const int pos = p.pos[b] + row - p.row0[b];
    const int pg = kv4_page(c, p.seq[b], pos);
    const int head = (int)(u % quads) * 4 + (lane >> 4);
    if (pg < 0 || head >= c.heads) return;
    const uint8_t* blk = kv4_block(c, pg, layer0 + (int)blockIdx.y, head);
    const int slot = pos & (c.page() - 1);
    const int64_t at = ((int64_t)blockIdx.y * rows + row_at + row) * c.heads + head;
    if (u < quads) {
#pragma unroll
        for (int t0 = 0; t0 < W / 8; t0 += 16) {
            const int t = t0 + o;
            if (t * 8 >= c.dk) continue;
            const uint32_t code = kv4_word(blk, kv4_k_dword(c, slot, t));
            const int g = t * 8 / c.group;
            const float step = f16_value(kv4_half(blk, kv4_k_scale(c, slot, g))), low = f16_value(kv4_half(blk, kv4_k_low(c, slot, g)));
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (t * 8 + e < c.dk)
                    Kv4Elem<TYPE>::put(k + at * c.dk + t * 8 + e,
                                       __builtin_fmaf(step, (float)((code >> (4 * ((e & 1) * 4 + (e >> 1)))) & 15u), low));
        }
    } else {
#pragma unroll
        for (int i = 0; i < W / 16; ++i) {
            const int d = 16 * i + o;
            if (d >= c.dv) continue;
            const int g = d / c.group;
            const uint32_t code = (uint32_t)kv4_half(blk, kv4_v_half(c, slot, o, i >> 2)) >> (4 * (i & 3)) & 15u;
            Kv4Elem<TYPE>::put(v + at * c.dv + d, __builtin_fmaf(f16_value(kv4_half(blk, kv4_v_scale(c, slot, g))), (float)code,
                                                                 f16_value(kv4_half(blk, kv4_v_low(c, slot, g)))));
        }
    }
}

template <int TYPE>
static hipError_t read_typed(const Kv4View& c, int layer, const Kv4Spans& p, int64_t rows, int64_t row, void* k, void* v,
                             hipStream_t s) {
    typedef typename Kv4Elem<TYPE>::T* P;
    const uint64_t blocks = ((uint64_t)p.row0[p.n] * 2 * ((c.heads + 3) / 4) + 3) / 4;
    if (blocks > 0x3fffffffu) return hipErrorInvalidValue;
    auto kern = c.width == 64 ? k_kv4_read<TYPE, 64> : c.width == 128 ? k_kv4_read<TYPE, 128> : k_kv4_read<TYPE, 256>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks, layer < 0 ? c.layers : 1), dim3(256), 0, s, c, layer < 0 ? 0 : layer, p,
                       rows, row, (P)k, (P)v);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4View& c, int layer, const Kv4Spans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s) {
    static_assert(sizeof(Kv4Spans) <= 3600, "the argument segment");
    return type == KV4_F32   ? read_typed<KV4_F32>(c, layer, p, rows, row, k, v, s)
           : type == KV4_F16 ? read_typed<KV4_F16>(c, layer, p, rows, row, k, v, s)
                             : read_typed<KV4_BF16>(c, layer, p, rows, row, k, v, s);
}

// ------------------------------------------------------------------ pages
// Whole pages, every layer and head: 16 bytes a thread.
__global__ __launch_bounds__(256) void k_kv4_pairs(Kv4View c, Kv4Pairs p) {
    const size_t n = c.page_bytes() / 16;
    const uint4* from = reinterpret_cast<const uint4*>(c.data) + (size_t)p.from[blockIdx.y] * n;
    uint4* to = reinterpret_cast<uint4*>(c.data) + (size_t)p.to[blockIdx.y] * n;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) to[i] = from[i];
}

hipError_t launch_kv4_pairs(const Kv4View& c, const Kv4Pairs& p, hipStream_t s) {
    static_assert(sizeof(Kv4Pairs) <= 3900, "the argument segment");
    const size_t blocks = (c.page_bytes() / 16 + 255) / 256;
    hipLaunchKernelGGL(k_kv4_pairs, dim3((unsigned)(blocks < 1024 ? blocks : 1024), p.n), dim3(256), 0, s, c, p);
    return hipGetLastError();
}

// One position of one (layer, head) by 16 lanes, four positions a wavefront.
// The fresh pages belong to this sequence alone and no position shares a byte
// with another, so the order of the moves does not matter.
__global__ __launch_bounds__(256) void k_kv4_runs(Kv4View c, const int* __restrict__ state, Kv4Runs r) {
    const int lane = threadIdx.x & 63, l = lane & 15;
    const int64_t i = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + (lane >> 4);
    if (i >= r.row0[r.n]) return;
    int lo = 0, hi = r.n - 1;  // the run that holds position i of the launch
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r.row0[mid] <= i) lo = mid;
        else hi = mid - 1;
    }
    const int off = (int)i - r.row0[lo];
    const int src = r.src[lo] + off, dst = r.dst[lo] + off;
    const int from = kv4_page(c, r.seq[lo], src), to = state[r.fresh[lo] + (dst >> c.page_log2)];
    if (from < 0) return;
    const int mask = c.page() - 1, s0 = src & mask, s1 = dst & mask, W = c.width, nb = W / 64, ng = c.groups();
    const uint8_t* a = kv4_block(c, from, (int)blockIdx.y, (int)blockIdx.z);
    uint8_t* z = kv4_block(c, to, (int)blockIdx.y, (int)blockIdx.z);
    for (int t = l; t < W / 8; t += 16) kv4_word(z, kv4_k_dword(c, s1, t)) = kv4_word(a, kv4_k_dword(c, s0, t));
    for (int b = 0; b < nb; ++b) kv4_half(z, kv4_v_half(c, s1, l, b)) = kv4_half(a, kv4_v_half(c, s0, l, b));
    if (l < ng) {
        kv4_half(z, kv4_k_scale(c, s1, l)) = kv4_half(a, kv4_k_scale(c, s0, l));
        kv4_half(z, kv4_k_low(c, s1, l)) = kv4_half(a, kv4_k_low(c, s0, l));
        kv4_half(z, kv4_v_scale(c, s1, l)) = kv4_half(a, kv4_v_scale(c, s0, l));
        kv4_half(z, kv4_v_low(c, s1, l)) = kv4_half(a, kv4_v_low(c, s0, l));
    }
}

hipError_t launch_kv4_runs(const Kv4View& c, const int* state, const Kv4Runs& r, hipStream_t s) {
    static_assert(sizeof(Kv4Runs) <= 3900, "the argument segment");
    const int64_t n = r.row0[r.n];
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(k_kv4_runs, dim3((unsigned)((n + 15) / 16), c.layers, c.heads), dim3(256), 0, s, c, state, r);
    return hipGetLastError();
}

}  // namespace nh
