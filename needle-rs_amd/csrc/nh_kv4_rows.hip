// The 4-bit cache's rows and pages: storing and reading rows, copying pages,
// closing sequences up.  The layout and the format are in nh_kv4.h.
#include "nh_kv4_device.h"

namespace nh {

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

// A workgroup's rows are those of one head in one chunk of 32 positions: their
// codes are put together in LDS as the chunk has them, and go out 16 bytes a
// thread if the rows fill the chunk, else piece by piece (the other positions'
// bytes are not touched).  16 lanes take a row, 8 dims each (twice at 256), its
// groups' ranges over 4 or 8 neighbouring lanes.
//
// Bound by memory, and by a launch's latency in a decoding step: 7,485 rows of 8
// heads of 128 in bf16 (40 MB in and out) take 16 us, 2.5 TB/s (33 us before the
// image: its bytes went out one by one); 8 rows of 2 heads 4.6 us.  What keeps it
// from the copy's 4.7 TB/s is the chain range, reciprocal, code in front of each
// store with two rows a lane in flight; both rows' loads issued first was slower
// (19 us: twice the code for rows that are mostly fetched once).
template <int TYPE, int W, int G, bool VALUES>
__device__ __forceinline__ void kv4_pack_row(const typename KvElem<TYPE>::T* __restrict__ x, int dim, bool vec, uint8_t* img,
                                             int slot, int lane, bool live) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(8)));
    typedef Kv4Lay<W, G> L;
#pragma unroll
    for (int t0 = 0; t0 < W / 8; t0 += 16) {
        const int t = t0 + (lane & 15), d = t * 8;
        float v[8];
        if (vec && live && d < dim) {  // (dim is a multiple of 8)
            const Vec y = *reinterpret_cast<const Vec*>(x + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)y[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = live && d + e < dim ? KvElem<TYPE>::get(x + d + e) : 0.0f;
        }
        float mn = __builtin_inff(), mx = -__builtin_inff();
        int bad = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bad |= !(fabsf(v[e]) < __builtin_inff());
            v[e] = fminf(fmaxf(v[e], -65504.0f), 65504.0f);
            if (d + e < dim) mn = fminf(mn, v[e]), mx = fmaxf(mx, v[e]);
        }
#pragma unroll
        for (int h = 1; h < G / 8; h <<= 1) {
            mn = fminf(mn, lane_xor(mn, h, lane));
            mx = fmaxf(mx, lane_xor(mx, h, lane));
            bad |= __float_as_int(lane_xor(__int_as_float(bad), h, lane));
        }
        if (mn > mx) mn = mx = 0.0f;  // a group of padding
        const Kv4Group g = kv4_group(mn, mx, bad != 0);
        uint32_t code[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) code[e] = d + e < dim ? kv4_code(v[e], g) : 0;
        if (!live || t >= W / 8) continue;
        if constexpr (VALUES) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) img[L::v_byte(slot, t * 4 + e / 2)] = (uint8_t)(code[e] | code[e + 1] << 4);
        } else {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) w |= code[e] << (4 * ((e & 1) * 4 + (e >> 1)));
            kv4_word(img, L::k_dword(slot, t)) = w;
        }
        if (t % (G / 8) == 0) {
            const int n = t / (G / 8);
            kv4_half(img, VALUES ? L::v_step(slot, n) : L::k_step(slot, n)) = g.sb;
            kv4_half(img, VALUES ? L::v_low(slot, n) : L::k_low(slot, n)) = g.lb;
        }
    }
}

// Positions lo .. hi of a chunk from `img` to `to` (two images of one layout), by
// the whole workgroup.
template <int W, int G, int THREADS>
__device__ __forceinline__ void kv4_put_chunk(const uint8_t* img, uint8_t* to, int lo, int hi, int tid) {
    typedef Kv4Lay<W, G> L;
    if (lo == 0 && hi == 31) {
        for (uint32_t i = tid; i < L::CHUNK / 16; i += THREADS)
            reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(img)[i];
        return;
    }
    // Key dwords, value halves, the four scales of a group: pieces of one position.
    constexpr int KD = W / 8, VH = W / 4, PIECES = KD + VH + 4 * L::NG;
    for (int i = tid; i < (hi - lo + 1) * PIECES; i += THREADS) {
        const int slot = lo + i / PIECES, p = i % PIECES;
        if (p < KD) {
            const uint32_t at = L::k_dword(slot, p);
            kv4_word(to, at) = kv4_word(img, at);
        } else {
            const int x = p - KD - VH, g = x >> 2;
            const uint32_t at = p < KD + VH    ? L::v_half(slot, (p - KD) & 15, (p - KD) >> 4)
                                : (x & 3) == 0 ? L::k_step(slot, g)
                                : (x & 3) == 1 ? L::k_low(slot, g)
                                : (x & 3) == 2 ? L::v_step(slot, g)
                                               : L::v_low(slot, g);
            kv4_half(to, at) = kv4_half(img, at);
        }
    }
}

struct Kv4Rows {  // the rows of an append, or of a read
    int64_t ldk, ldv;
    int veck, vecv;  // rows of k, of v can be taken 8 elements at a time
    int each;        // chunks of every sequence, when all have the same rows (the most), else 0
};

__host__ __device__ inline int kv4_most_chunks(int rows) { return rows ? (rows + 30) / 32 + 1 : 0; }

template <int TYPE, int W, int G>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4View c, int layer, const typename KvElem<TYPE>::T* __restrict__ k,
                                                    const typename KvElem<TYPE>::T* __restrict__ v, Kv4Rows a) {
    typedef Kv4Lay<W, G> L;
    __shared__ __align__(16) uint8_t img[L::CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.x % c.heads;
    int unit = blockIdx.x / c.heads, b;
    if (a.each) {
        b = unit / a.each;
        unit -= b * a.each;
    } else
        b = kv_find(c, unit, lane, [](const KvEntry& e) { return kv4_most_chunks(e.row1 - e.row0); });
    if (b >= c.nb) return;
    const KvEntry e = kv_batch(c, b);
    const int first = e.len - (e.row1 - e.row0);  // the position of row row0
    const int pos0 = ((first >> 5) + unit) << 5, lo = max(first - pos0, 0), hi = min(e.len - 1 - pos0, 31);
    if (!kv_current(c) || first < 0 || lo > hi || e.row1 > c.rows) return;
    const int pg = kv_page(c, e.seq, pos0);
    if (pg < 0) return;
#pragma unroll 1
    for (int s0 = lo; s0 <= hi; s0 += 16) {
        const int slot = s0 + (tid >> 4);
        const bool live = slot <= hi;
        const int64_t row = e.row0 + (live ? pos0 + slot - first : 0);
        kv4_pack_row<TYPE, W, G, false>(k + row * a.ldk + (int64_t)head * c.dk, c.dk, a.veck, img, slot, lane, live);
        kv4_pack_row<TYPE, W, G, true>(v + row * a.ldv + (int64_t)head * c.dv, c.dv, a.vecv, img, slot, lane, live);
    }
    __syncthreads();
    uint8_t* to = kv4_block(c, pg, layer, head) + (uint32_t)((pos0 & (c.page() - 1)) >> 5) * L::CHUNK;
    kv4_put_chunk<W, G, 256>(img, to, lo, hi, tid);
}

template <int TYPE>
static bool can_take8(const void* p, int64_t ld, int dim) {
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    return dim % 8 == 0 && (uintptr_t)p % 16 == 0 && ld * es % 16 == 0;
}

template <int TYPE, int G>
static hipError_t append_typed(const Kv4View& c, const int* row0, int layer, const void* k, const void* v, int64_t ldk,
                               int64_t ldv, hipStream_t s) {
    typedef const typename KvElem<TYPE>::T* P;
    Kv4Rows a{ldk, ldv, can_take8<TYPE>(k, ldk, c.dk), can_take8<TYPE>(v, ldv, c.dv), kv4_most_chunks(c.each)};
    int64_t units = (int64_t)a.each * c.nb;
    if (!a.each)
        for (int b = 0; b < c.nb; ++b) units += kv4_most_chunks(row0[b + 1] - row0[b]);
    if (units * c.heads > 0x7fffffff) return hipErrorInvalidValue;
    auto kern = c.width == 64    ? k_kv4_append<TYPE, 64, G>
                : c.width == 128 ? k_kv4_append<TYPE, 128, G>
                                 : k_kv4_append<TYPE, 256, G>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(units * c.heads)), dim3(256), 0, s, c, layer, (P)k, (P)v, a);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t append_typed(const Kv4View& c, const int* row0, int layer, const void* k, const void* v, int64_t ldk,
                               int64_t ldv, hipStream_t s) {
    return c.group == 32 ? append_typed<TYPE, 32>(c, row0, layer, k, v, ldk, ldv, s)
                         : append_typed<TYPE, 64>(c, row0, layer, k, v, ldk, ldv, s);
}

hipError_t launch_kv4_append(const Kv4View& c, const int* row0, int layer, const void* k, const void* v, int64_t ldk,
                             int64_t ldv, int type, hipStream_t s) {
    return type == KV_F32   ? append_typed<KV_F32>(c, row0, layer, k, v, ldk, ldv, s)
           : type == KV_F16 ? append_typed<KV_F16>(c, row0, layer, k, v, ldk, ldv, s)
                             : append_typed<KV_BF16>(c, row0, layer, k, v, ldk, ldv, s);
}

// Eight dims of a row of keys, or of values, out of a chunk's image.  step * code
// is exact in f32, so the fma rounds once, as the product and the sum do.
template <int TYPE, int W, int G, bool VALUES>
__device__ __forceinline__ void kv4_unpack8(const uint8_t* img, int slot, int t, typename KvElem<TYPE>::T* __restrict__ to,
                                            int dim, bool vec) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(8)));
    typedef Kv4Lay<W, G> L;
    const int g = t * 8 / G;
    const float step = f16_value(kv4_half(img, VALUES ? L::v_step(slot, g) : L::k_step(slot, g)));
    const float low = f16_value(kv4_half(img, VALUES ? L::v_low(slot, g) : L::k_low(slot, g)));
    uint32_t code[8];
    if constexpr (VALUES) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t y = img[L::v_byte(slot, t * 4 + e / 2)];
            code[e] = y & 15u;
            code[e + 1] = y >> 4;
        }
    } else {
        const uint32_t w = kv4_word(img, L::k_dword(slot, t));
#pragma unroll
        for (int e = 0; e < 8; ++e) code[e] = w >> (4 * ((e & 1) * 4 + (e >> 1))) & 15u;
    }
    Vec y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        T z;
        KvElem<TYPE>::put(&z, __builtin_fmaf(step, (float)code[e], low));
        y[e] = z;
    }
    if (vec)
        *reinterpret_cast<Vec*>(to + t * 8) = y;
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (t * 8 + e < dim) to[t * 8 + e] = y[e];
}

// A workgroup reads one head's rows of one chunk: the chunk to LDS, 16 bytes a
// thread, then 8 dims a lane out of it.  Bound by what it writes: the 7,485 rows
// above in 10 us (4 TB/s), 8 layers of 4,122 (177 MB) in 35 (5 TB/s).
template <int TYPE, int W, int G>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4View c, int layer0, KvSpans p, int64_t rows, int64_t row_at,
                                                  typename KvElem<TYPE>::T* __restrict__ k,
                                                  typename KvElem<TYPE>::T* __restrict__ v, Kv4Rows a) {
    typedef Kv4Lay<W, G> L;
    __shared__ __align__(16) uint8_t img[L::CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.x % c.heads;
    const int unit = blockIdx.x / c.heads, b = kv_span(p.unit0, p.n, unit, lane);
    const int first = p.pos[b], end = first + p.row0[b + 1] - p.row0[b];
    const int pos0 = ((first >> 5) + unit - p.unit0[b]) << 5, lo = max(first - pos0, 0), hi = min(end - 1 - pos0, 31);
    const int pg = kv_page(c, p.seq[b], pos0);
    if (pg < 0) return;
    const uint8_t* from = kv4_block(c, pg, layer0 + (int)blockIdx.y, head) + (uint32_t)((pos0 & (c.page() - 1)) >> 5) * L::CHUNK;
    for (uint32_t i = tid; i < L::CHUNK / 16; i += 256)
        reinterpret_cast<uint4*>(img)[i] = reinterpret_cast<const uint4*>(from)[i];
    __syncthreads();
    const int64_t row = (int64_t)blockIdx.y * rows + row_at + p.row0[b] + (pos0 - first);  // of slot 0
    for (int i = tid; i < (hi - lo + 1) * (W / 8); i += 256) {
        const int slot = lo + i / (W / 8), t = i % (W / 8);
        const int64_t at = (row + slot) * c.heads + head;
        if (t * 8 < c.dk) kv4_unpack8<TYPE, W, G, false>(img, slot, t, k + at * c.dk, c.dk, a.veck);
        if (t * 8 < c.dv) kv4_unpack8<TYPE, W, G, true>(img, slot, t, v + at * c.dv, c.dv, a.vecv);
    }
}

template <int TYPE, int G>
static hipError_t read_typed(const Kv4View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                             hipStream_t s) {
    typedef typename KvElem<TYPE>::T* P;
    const Kv4Rows a{0, 0, can_take8<TYPE>(k, c.dk, c.dk), can_take8<TYPE>(v, c.dv, c.dv), 0};
    const int64_t blocks = (int64_t)p.unit0[p.n] * c.heads;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    auto kern = c.width == 64 ? k_kv4_read<TYPE, 64, G> : c.width == 128 ? k_kv4_read<TYPE, 128, G> : k_kv4_read<TYPE, 256, G>;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks, layer < 0 ? c.layers : 1), dim3(256), 0, s, c, layer < 0 ? 0 : layer, p,
                       rows, row, (P)k, (P)v, a);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t read_typed(const Kv4View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                             hipStream_t s) {
    return c.group == 32 ? read_typed<TYPE, 32>(c, layer, p, rows, row, k, v, s)
                         : read_typed<TYPE, 64>(c, layer, p, rows, row, k, v, s);
}

hipError_t launch_kv4_read(const Kv4View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s) {
    static_assert(sizeof(KvSpans) <= 3900, "the argument segment");
    return type == KV_F32   ? read_typed<KV_F32>(c, layer, p, rows, row, k, v, s)
           : type == KV_F16 ? read_typed<KV_F16>(c, layer, p, rows, row, k, v, s)
                             : read_typed<KV_BF16>(c, layer, p, rows, row, k, v, s);
}

// ------------------------------------------------------------------ pages
// A workgroup writes one run's positions of one chunk of a fresh page, for one
// (layer, head): gathered into LDS, then stored as an append stores them.  The
// fresh pages belong to this sequence alone and no position shares a byte with
// another, so the order of the moves does not matter.  3 x 1,374 rows of 8 layers
// and 8 heads (84 MB in and out) in 25 us, 3.4 TB/s; 37 us without the image.
template <int W, int G>
__global__ __launch_bounds__(128) void k_kv4_runs(Kv4View c, const int* __restrict__ state, Kv4Runs r) {
    typedef Kv4Lay<W, G> L;
    __shared__ __align__(16) uint8_t img[L::CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, l = tid & 15;
    const int unit = blockIdx.x, m = kv_span(r.unit0, r.n, unit, lane);
    const int dst = r.dst[m], pos0 = ((dst >> 5) + unit - r.unit0[m]) << 5;
    const int lo = max(dst - pos0, 0), hi = min(dst + r.count[m] - 1 - pos0, 31), src0 = r.src[m] - dst + pos0;
    const int to = state[r.fresh[m] + (pos0 >> c.page_log2)], mask = c.page() - 1;
    for (int slot = lo + (tid >> 4); slot <= hi; slot += 8) {
        const int src = src0 + slot, from = kv_page(c, r.seq[m], src);
        if (from < 0) continue;
        const uint8_t* a = kv4_block(c, from, (int)blockIdx.y, (int)blockIdx.z) + (uint32_t)((src & mask) >> 5) * L::CHUNK;
        const int s = src & 31;
#pragma unroll
        for (int t = l; t < W / 8; t += 16) kv4_word(img, L::k_dword(slot, t)) = kv4_word(a, L::k_dword(s, t));
#pragma unroll
        for (int b = 0; b < L::NB; ++b) kv4_half(img, L::v_half(slot, l, b)) = kv4_half(a, L::v_half(s, l, b));
        if (l < L::NG) {
            kv4_half(img, L::k_step(slot, l)) = kv4_half(a, L::k_step(s, l));
            kv4_half(img, L::k_low(slot, l)) = kv4_half(a, L::k_low(s, l));
            kv4_half(img, L::v_step(slot, l)) = kv4_half(a, L::v_step(s, l));
            kv4_half(img, L::v_low(slot, l)) = kv4_half(a, L::v_low(s, l));
        }
    }
    __syncthreads();
    uint8_t* z = kv4_block(c, to, (int)blockIdx.y, (int)blockIdx.z) + (uint32_t)((pos0 & mask) >> 5) * L::CHUNK;
    kv4_put_chunk<W, G, 128>(img, z, lo, hi, tid);
}

template <int G>
static hipError_t launch_runs(const Kv4View& c, const int* state, const Kv4Runs& r, hipStream_t s) {
    auto kern = c.width == 64 ? k_kv4_runs<64, G> : c.width == 128 ? k_kv4_runs<128, G> : k_kv4_runs<256, G>;
    hipLaunchKernelGGL(kern, dim3((unsigned)r.unit0[r.n], c.layers, c.heads), dim3(128), 0, s, c, state, r);
    return hipGetLastError();
}

hipError_t launch_kv4_runs(const Kv4View& c, const int* state, const Kv4Runs& r, hipStream_t s) {
    static_assert(sizeof(Kv4Runs) <= 3900, "the argument segment");
    if (r.unit0[r.n] <= 0) return hipSuccess;
    return c.group == 32 ? launch_runs<32>(c, state, r, s) : launch_runs<64>(c, state, r, s);
}

}  // namespace nh
