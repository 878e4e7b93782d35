// The 8-bit cache's rows: storing (keys and queries turned first, if asked) and
// reading them.  The layout and the format are in nh_kv8.h.
#include <algorithm>
#include <type_traits>

#include "nh_kv8_device.h"
#include "nh_rope_turn.h"

namespace nh {

// ------------------------------------------------------------------ steps
// What a block's rows do to its step: `largest` |x| of the new rows, `old` the
// step so far (0: none, or rows of nothing but 0).
struct Kv8Step {
    float step, inv;  // inv 0: every code is 0
    int down;         // the codes that were there are divided by 2^down
};
__device__ __forceinline__ Kv8Step kv8_step(float largest, float old) {
    float need = largest * __builtin_bit_cast(float, 0x3c010204u);  // f32(1/127)
    if (need < 0x1p-120f) need = 0.0f;
    Kv8Step s;
    s.down = 0;
    s.step = need;
    if (old > 0.0f) {
        s.step = old;
        if (need > old) {
            // (both are normal numbers: their exponents, and one more if that is short)
            int k = (int)(__builtin_bit_cast(uint32_t, need) >> 23) - (int)(__builtin_bit_cast(uint32_t, old) >> 23);
            if (__builtin_amdgcn_ldexpf(old, k) < need) ++k;
            s.step = __builtin_amdgcn_ldexpf(old, k);
            s.down = k;
        }
    }
    s.inv = s.step > 0.0f ? 1.0f / s.step : 0.0f;
    return s;
}
// The byte of x: 1.5 2^23 added leaves the nearest whole number, ties to even, in
// the low bits.
__device__ __forceinline__ uint32_t kv8_code(float x, float inv) {
    const float c = __builtin_amdgcn_fmed3f(x * inv, -127.0f, 127.0f) + 12582912.0f;
    return __builtin_bit_cast(uint32_t, c) + 128u;  // (its low byte)
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t x = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), y = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return x | y;
}
// Four bytes divided by 2^down, ties to even.
__device__ __forceinline__ uint32_t kv8_halved(uint32_t w, int down) {
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float c = (float)(int)((w >> (8 * e) & 255u) - 128u);
        y[e] = (uint32_t)(int)rintf(__builtin_amdgcn_ldexpf(c, -down)) + 128u;
    }
    return low_bytes(y[0], y[1], y[2], y[3]);
}

__device__ __forceinline__ float wave_max(float v, int lane) {
#pragma unroll
    for (int h = 1; h < 64; h <<= 1) v = fmaxf(v, lane_xor(v, h, lane));
    return v;
}

// Eight elements of a row from dim d, 0 past its end.
template <int TYPE>
__device__ __forceinline__ void kv8_take8(const typename KvElem<TYPE>::T* __restrict__ x, int d, int dim, bool vec, float* v) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(8)));
    if (vec) {  // (dim is a multiple of 8)
        Vec y = {};
        if (d < dim) y = *reinterpret_cast<const Vec*>(x + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)y[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = d + e < dim ? KvElem<TYPE>::get(x + d + e) : 0.0f;
    }
}

// ----------------------------------------------------------------- append
struct Kv8AppendPlan {
    int each;               // chunks of every sequence, when all have the same rows (the most), else 0
    int veck, vecv;         // rows of k, of v can be taken 8 (4) elements at a time
    int k_share, v_share, q_share;  // heads a workgroup takes
    int k_parts, v_parts, q_parts;  // workgroups a chunk
    RopePlan rope;          // of the queries
    int wide;               // .. 4 pairs a thread
};

__host__ __device__ inline int kv8_most_chunks(int rows) { return rows ? (rows + 62) / 64 + 1 : 0; }

// One block of keys by one wavefront: lane (o, kg) has position o, 16 dims of
// each 64 from 16 kg on: the bytes that it stores are one piece of its own.
template <int TYPE, int WK, int WV, int TURN>
__device__ __forceinline__ void kv8_put_keys(const typename KvElem<TYPE>::T* __restrict__ x, int dim, bool vec, uint8_t* chunk,
                                             int t, int lo, int hi, int lane, const RopeView& r, const float2* cs) {
    typedef Kv8Lay<WK, WV> L;
    const int o = lane & 15, kg = lane >> 4;
    const bool live = o >= lo && o <= hi;
    Kv8Record* rec = reinterpret_cast<Kv8Record*>(chunk + L::RECORD);
    const float old = lo ? rec->ks[t] : 0.0f;
    const uint32_t old_bad = lo ? rec->kbad[t] & ((1u << lo) - 1u) : 0u;
    float v[L::NJ][16];
#pragma unroll
    for (int j = 0; j < L::NJ; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int d = 64 * j + 16 * kg + 8 * g;
            float* y = v[j] + 8 * g;
            if (!live) {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = 0.0f;
                continue;
            }
            kv8_take8<TYPE>(x, d, dim, vec, y);
            if constexpr (TURN == 1) {  // pairs (i, i + pairs)
                if (d < 2 * r.pairs) {
                    float z[8];
                    // (eight dims on one side of the pairs, or some on each)
                    const bool whole = r.pairs % 8 == 0;
                    if (whole)
                        kv8_take8<TYPE>(x, d < r.pairs ? d + r.pairs : d - r.pairs, dim, vec, z);
                    else
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = d + e < r.pairs ? d + e + r.pairs : d + e - r.pairs;
                            z[e] = d + e < 2 * r.pairs ? KvElem<TYPE>::get(x + at) : 0.0f;
                        }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool second = d + e >= r.pairs;
                        const int i = second ? d + e - r.pairs : d + e;
                        if (i < r.pairs) {
                            const float2 w = cs[i];
                            const float2 both = second ? rope_turn(z[e], y[e], w) : rope_turn(y[e], z[e], w);
                            y[e] = second ? both.y : both.x;
                        }
                    }
                }
            } else if constexpr (TURN == 2) {  // neighbours
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const int i = (d + e) / 2;
                    if (i < r.pairs) {
                        const float2 both = rope_turn(y[e], y[e + 1], cs[i]);
                        y[e] = both.x, y[e + 1] = both.y;
                    }
                }
            }
        }
    float most = 0.0f;
    int bad = 0;
#pragma unroll
    for (int j = 0; j < L::NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            bad |= !(fabsf(v[j][e]) < __builtin_inff());
            most = fmaxf(most, fabsf(v[j][e]));
        }
    // a row with a NaN or an infinity: its four lanes
    bad |= __shfl_xor(bad, 16, 64);
    bad |= __shfl_xor(bad, 32, 64);
    const uint32_t bads = (uint32_t)__ballot(bad != 0) & 0xffffu;
    most = wave_max(bad ? 0.0f : most, lane);
    const Kv8Step s = kv8_step(most, old);
    if (live) {
#pragma unroll
        for (int j = 0; j < L::NJ; ++j) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = kv8_code(bad ? 0.0f : v[j][4 * i + e], s.inv);
                w[i] = low_bytes(y[0], y[1], y[2], y[3]);
            }
            *reinterpret_cast<u32x4*>(chunk + L::k_piece(t, j, lane)) = w;
        }
    } else if (s.down && o < lo) {
#pragma unroll
        for (int j = 0; j < L::NJ; ++j) {
            u32x4* p = reinterpret_cast<u32x4*>(chunk + L::k_piece(t, j, lane));
            u32x4 w = *p;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = kv8_halved(w[i], s.down);
            *p = w;
        }
    }
    if (lane == 0) {
        rec->ks[t] = s.step;
        rec->kbad[t] = (uint16_t)(old_bad | bads);
    }
}

// One block of values: lane (c, a) has dims 4 c .. of positions 4 a ..: turned
// four by four, its words are whole too.
template <int TYPE, int WK, int WV>
__device__ __forceinline__ void kv8_put_values(const typename KvElem<TYPE>::T* __restrict__ x, int64_t ld, int dim, bool vec,
                                               uint8_t* chunk, int t, int lo, int hi, int lane) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(4)));
    typedef Kv8Lay<WK, WV> L;
    constexpr int NB = WV / 64;
    const int c = lane & 15, a = lane >> 4;
    Kv8Record* rec = reinterpret_cast<Kv8Record*>(chunk + L::RECORD);
    const float old = lo ? rec->vs[t] : 0.0f;
    const uint32_t old_bad = lo ? rec->vbad[t] & ((1u << lo) - 1u) : 0u;
    float v[NB][4][4];  // [..][position][dim]
    float most = 0.0f;
    uint32_t bads = 0;
    bool bad[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int slot = 4 * a + r;
        const bool live = slot >= lo && slot <= hi;
        int wrong = 0;
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int d = 64 * n + 4 * c;
            const T* p = x + (int64_t)slot * ld;
            if (vec) {
                Vec y = {};
                if (live && d < dim) y = *reinterpret_cast<const Vec*>(p + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[n][r][e] = (float)y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[n][r][e] = live && d + e < dim ? KvElem<TYPE>::get(p + d + e) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                wrong |= !(fabsf(v[n][r][e]) < __builtin_inff());
                top = fmaxf(top, fabsf(v[n][r][e]));
            }
        }
        // (the row's sixteen lanes)
        const uint64_t which = __ballot(wrong != 0);
        bad[r] = (which >> (16 * a) & 0xffffu) != 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) bads |= (which >> (16 * g) & 0xffffu) ? 1u << (4 * g + r) : 0u;
        most = fmaxf(most, bad[r] ? 0.0f : top);
    }
    most = wave_max(most, lane);
    const Kv8Step s = kv8_step(most, old);
    const bool some = 4 * a <= hi && 4 * a + 3 >= lo, before = 4 * a < lo;
    if (some || (s.down && before)) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 4 * c + e;  // of 64
                uint32_t* p = reinterpret_cast<uint32_t*>(chunk + L::v_piece(4 * n + (d >> 4), 16 * a + (d & 15)) + 4 * t);
                uint32_t y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = kv8_code(bad[r] ? 0.0f : v[n][r][e], s.inv);
                uint32_t w = low_bytes(y[0], y[1], y[2], y[3]);
                if (before) {
                    uint32_t was = *p;
                    if (s.down) was = kv8_halved(was, s.down);
                    // (its bytes of positions below lo)
                    const uint32_t keep = lo - 4 * a >= 4 ? 0xffffffffu : (1u << (8 * (lo - 4 * a))) - 1u;
                    w = (was & keep) | (w & ~keep);
                }
                *p = w;
            }
    }
    if (lane == 0) {
        rec->vs[t] = s.step;
        rec->vbad[t] = (uint16_t)(old_bad | bads);
    }
}

// A workgroup takes one chunk of a sequence's new rows and some heads of the
// keys, of the values or of the queries.  A wavefront has a block: its step is a
// maximum over its own lanes, no workgroup shares a block, and no barrier is
// needed but the one behind the table of cosines and sines of the chunk's
// positions, worked out once for the workgroup's heads.
template <int TYPE, int WK, int WV, int TURN>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8View c, Kv8Append a, Kv8AppendPlan p) {
    typedef typename KvElem<TYPE>::T T;
    typedef Kv8Lay<WK, WV> L;
    extern __shared__ float2 cs[];  // [64][pairs + 1]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int parts = p.k_parts + p.v_parts + p.q_parts;
    int part = blockIdx.x % parts, unit = blockIdx.x / parts, b;
    if (p.each) {
        b = unit / p.each;
        unit -= b * p.each;
    } else
        b = kv_find(c, unit, lane, [](const KvEntry& e) { return kv8_most_chunks(e.row1 - e.row0); });
    if (b >= c.nb) return;
    const KvEntry e = kv_batch(c, b);
    const int first = e.len - (e.row1 - e.row0);  // the position of row row0
    const int pos0 = ((first >> 6) + unit) << 6, lo = max(first - pos0, 0), hi = min(e.len - 1 - pos0, 63);
    if (!kv_current(c) || first < 0 || lo > hi || e.row1 > c.rows) return;
    const int64_t row0 = (int64_t)e.row0 + pos0 - first;  // of slot 0

    if constexpr (TURN != 0) {
        if (part >= p.k_parts + p.v_parts) {
            const int h0 = (part - p.k_parts - p.v_parts) * p.q_share, h1 = min(h0 + p.q_share, a.q.heads);
            const RopeArgs q{a.r, nullptr, a.q, RopeRows{}, 0, c.dk, 0};
            for (int i = tid; i < (hi - lo + 1) * p.rope.units; i += 256) {
                const int slot = lo + i / p.rope.units, u = i % p.rope.units;
                const int64_t row = row0 + slot;
                const int pos = a.pos ? a.pos[row] : pos0 + slot;
                if (p.wide)
                    rope_rows<TYPE, 4, TURN == 2>(q, p.rope, row, u, pos, h0, h1);
                else
                    rope_rows<TYPE, 1, TURN == 2>(q, p.rope, row, u, pos, h0, h1);
            }
            return;
        }
    }
    const int pg = kv_page(c, e.seq, pos0);
    if (pg < 0) return;
    const uint32_t at = (uint32_t)((pos0 & (c.page() - 1)) >> 6) * L::CHUNK;
    const bool keys = part < p.k_parts;
    if (!keys) part -= p.k_parts;
    const int share = keys ? p.k_share : p.v_share;
    const int h0 = part * share, h1 = min(h0 + share, c.heads);
    if constexpr (TURN != 0) {
        if (keys) {
            const int n = (hi - lo + 1) * a.r.pairs;
            for (int i = tid; i < n; i += 256) {
                const int slot = lo + i / a.r.pairs, pair = i % a.r.pairs;
                cs[slot * (a.r.pairs + 1) + pair] =
                    rope_cos_sin(a.r.turns[pair], a.pos ? a.pos[row0 + slot] : pos0 + slot, a.r.amplitude);
            }
            __syncthreads();
        }
    }
    const int t = wave, blo = max(lo - 16 * t, 0), bhi = min(hi - 16 * t, 15);
    if (blo > bhi) return;
    for (int h = h0; h < h1; ++h) {
        uint8_t* chunk = kv8_block(c, pg, a.layer, h) + at;
        if (keys) {
            const int slot = 16 * t + (lane & 15);
            const T* x = reinterpret_cast<const T*>(a.k) + (row0 + slot) * a.ldk + (int64_t)h * c.dk;
            kv8_put_keys<TYPE, WK, WV, TURN>(x, c.dk, p.veck, chunk, t, blo, bhi, lane, a.r, cs + slot * (a.r.pairs + 1));
        } else {
            const T* x = reinterpret_cast<const T*>(a.v) + (row0 + 16 * t) * a.ldv + (int64_t)h * c.dv;
            kv8_put_values<TYPE, WK, WV>(x, a.ldv, c.dv, p.vecv, chunk, t, blo, bhi, lane);
        }
    }
}

template <int TYPE, int WK, int WV>
static hipError_t append_typed(const Kv8View& c, const int* row0, const Kv8Append& a, hipStream_t s) {
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    Kv8AppendPlan p;
    p.each = kv8_most_chunks(c.each);
    int64_t units = (int64_t)p.each * c.nb;
    if (!p.each)
        for (int b = 0; b < c.nb; ++b) units += kv8_most_chunks(row0[b + 1] - row0[b]);
    p.veck = c.dk % 8 == 0 && (uintptr_t)a.k % 16 == 0 && a.ldk * es % 16 == 0 && c.dk * es % 16 == 0;
    p.vecv = c.dv % 4 == 0 && (uintptr_t)a.v % (4 * es) == 0 && a.ldv % 4 == 0;
    const bool turn = a.r.turns != nullptr;
    p.k_share = p.v_share = 1;
    p.q_share = 0;
    p.k_parts = (c.heads + p.k_share - 1) / p.k_share;
    p.v_parts = (c.heads + p.v_share - 1) / p.v_share;
    p.q_parts = 0;
    p.rope = RopePlan{};
    p.wide = 0;
    if (turn && a.q.heads) {
        const RopeArgs q{a.r, nullptr, a.q, RopeRows{}, 0, c.dk, 0};
        p.wide = rope_takes4(q, es);
        p.rope = rope_plan(q, p.wide ? 4 : 1);
        p.q_share = std::min(a.q.heads, 8);
        p.q_parts = (a.q.heads + p.q_share - 1) / p.q_share;
    }
    const int64_t blocks = units * (p.k_parts + p.v_parts + p.q_parts);
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    const size_t lds = turn ? (size_t)64 * (a.r.pairs + 1) * sizeof(float2) : 0;
    auto kern = !turn              ? k_kv8_append<TYPE, WK, WV, 0>
                : a.r.interleaved ? k_kv8_append<TYPE, WK, WV, 2>
                                  : k_kv8_append<TYPE, WK, WV, 1>;
    if (lds > 65536) {
        // (more than a kernel may have without being asked for it)
        if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds))
            return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), lds, s, c, a, p);
    return hipGetLastError();
}

// ------------------------------------------------------------------- read
// A workgroup reads one head's rows of one chunk, a wavefront a block: keys as
// their lanes hold them, values four positions by four dims.
template <int TYPE, int WK, int WV>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8View c, int layer0, KvSpans p, int64_t rows, int64_t row_at,
                                                  typename KvElem<TYPE>::T* __restrict__ k,
                                                  typename KvElem<TYPE>::T* __restrict__ v, int veck, int vecv) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec8 __attribute__((ext_vector_type(8)));
    typedef T Vec4 __attribute__((ext_vector_type(4)));
    typedef Kv8Lay<WK, WV> L;
    const int tid = threadIdx.x, lane = tid & 63, o = lane & 15, kg = lane >> 4;
    const int t = __builtin_amdgcn_readfirstlane(tid >> 6), head = blockIdx.x % c.heads;
    const int unit = blockIdx.x / c.heads, b = kv_span(p.unit0, p.n, unit, lane);
    const int first = p.pos[b], end = first + p.row0[b + 1] - p.row0[b];
    const int pos0 = ((first >> 6) + unit - p.unit0[b]) << 6, lo = max(first - pos0, 0), hi = min(end - 1 - pos0, 63);
    const int pg = kv_page(c, p.seq[b], pos0);
    if (pg < 0) return;
    const uint8_t* chunk = kv8_block(c, pg, layer0 + (int)blockIdx.y, head) + (uint32_t)((pos0 & (c.page() - 1)) >> 6) * L::CHUNK;
    const Kv8Record* rec = reinterpret_cast<const Kv8Record*>(chunk + L::RECORD);
    const int64_t row = (int64_t)blockIdx.y * rows + row_at + p.row0[b] + (pos0 - first);  // of slot 0
    if (16 * t > hi || 16 * t + 15 < lo) return;
    const float nan = __builtin_nanf("");
    {
        const int slot = 16 * t + o;
        if (slot >= lo && slot <= hi) {
            const float step = rec->kbad[t] >> o & 1 ? nan : rec->ks[t];
            T* to = k + ((row + slot) * c.heads + head) * c.dk;
#pragma unroll
            for (int j = 0; j < L::NJ; ++j) {
                const int d = 64 * j + 16 * kg;
                if (d >= c.dk) continue;
                const u32x4 w = *reinterpret_cast<const u32x4*>(chunk + L::k_piece(t, j, lane));
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    Vec8 y;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t u = w[2 * g + e / 4] >> (8 * (e % 4)) & 255u;
                        y[e] = (T)((float)((int)u - 128) * step);
                    }
                    if (veck) {
                        if (d + 8 * g < c.dk) *reinterpret_cast<Vec8*>(to + d + 8 * g) = y;
                    } else
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (d + 8 * g + e < c.dk) to[d + 8 * g + e] = y[e];
                }
            }
        }
    }
    const int cc = o, a = kg;
    if (16 * t + 4 * a > hi || 16 * t + 4 * a + 3 < lo) return;
#pragma unroll
    for (int n = 0; n < WV / 64; ++n) {
        const int d = 64 * n + 4 * cc;
        if (d >= c.dv) continue;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = *reinterpret_cast<const uint32_t*>(chunk + L::v_piece(4 * n + (cc >> 2), 16 * a + 4 * (cc & 3) + e) + 4 * t);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int in = 4 * a + r, slot = 16 * t + in;
            if (slot < lo || slot > hi) continue;
            const float step = rec->vbad[t] >> in & 1 ? nan : rec->vs[t];
            T* to = v + ((row + slot) * c.heads + head) * c.dv + d;
            Vec4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)((float)((int)(w[e] >> (8 * r) & 255u) - 128) * step);
            if (vecv)
                *reinterpret_cast<Vec4*>(to) = y;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < c.dv) to[e] = y[e];
        }
    }
}

template <int TYPE, int WK, int WV>
static hipError_t read_typed(const Kv8View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                             hipStream_t s) {
    typedef typename KvElem<TYPE>::T T;
    const int veck = c.dk % 8 == 0 && (uintptr_t)k % 16 == 0, vecv = c.dv % 4 == 0 && (uintptr_t)v % (4 * sizeof(T)) == 0;
    const int64_t blocks = (int64_t)p.unit0[p.n] * c.heads;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_kv8_read<TYPE, WK, WV>), dim3((unsigned)blocks, layer < 0 ? c.layers : 1), dim3(256), 0, s, c,
                       layer < 0 ? 0 : layer, p, rows, row, (T*)k, (T*)v, veck, vecv);
    return hipGetLastError();
}

// f(type, wk, wv) as constants of the view's widths and the type.
template <int TYPE, class F>
static hipError_t by_width(const Kv8View& c, F f) {
    return c.wk == 64    ? f(std::integral_constant<int, TYPE>(), std::integral_constant<int, 64>(), std::integral_constant<int, 64>())
           : c.wk == 128 ? f(std::integral_constant<int, TYPE>(), std::integral_constant<int, 128>(), std::integral_constant<int, 128>())
           : c.wk == 192 ? f(std::integral_constant<int, TYPE>(), std::integral_constant<int, 192>(), std::integral_constant<int, 128>())
                         : f(std::integral_constant<int, TYPE>(), std::integral_constant<int, 256>(), std::integral_constant<int, 256>());
}
template <class F>
static hipError_t by_type(const Kv8View& c, int type, F f) {
    return type == KV_F32 ? by_width<KV_F32>(c, f) : type == KV_F16 ? by_width<KV_F16>(c, f) : by_width<KV_BF16>(c, f);
}

hipError_t launch_kv8_append(const Kv8View& c, const int* row0, const Kv8Append& a, int type, hipStream_t s) {
    return by_type(c, type, [&](auto T, auto K, auto V) { return append_typed<T.value, K.value, V.value>(c, row0, a, s); });
}

hipError_t launch_kv8_read(const Kv8View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s) {
    return by_type(c, type, [&](auto T, auto K, auto V) {
        return read_typed<T.value, K.value, V.value>(c, layer, p, rows, row, k, v, s);
    });
}

}  // namespace nh
