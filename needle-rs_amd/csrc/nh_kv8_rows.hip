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
    int blocks_each, chunks_each;  // blocks of 16 and chunks of 64 of every sequence, when all have the same rows (the most), else 0
    int veck, vecv;                // rows of k can be taken 8, rows of v 4 elements at a time
    int k_parts, q_parts;          // workgroups a block for the heads of the keys, of the queries
    int q_share;                   // query heads a workgroup takes
    int k_grid, v_grid, grid;      // workgroups of the keys, of the values, of all: the queries' come after them
    RopePlan rope;                 // of the queries
    int wide, widek;               // .. and of the keys: four pairs a thread
};
constexpr int KV8_HEADS = 4;  // of the keys a workgroup takes, a wavefront each

// The most blocks (chunks) of 2^LOG positions that rows of a sequence can lie in.
template <int LOG>
__host__ __device__ inline int kv8_most(int rows) {
    return rows ? ((rows + (1 << LOG) - 2) >> LOG) + 1 : 0;
}

// Unit `unit` of all sequences' blocks of 2^LOG positions: the new rows in it.
struct Kv8Unit {
    bool some;
    int seq, pos0, lo, hi;  // slots lo .. hi of the block from pos0 on
    int64_t row0;           // the row of slot 0
};
template <int LOG>
__device__ __forceinline__ Kv8Unit kv8_unit(const Kv8View& c, int unit, int each, int lane) {
    Kv8Unit u;
    u.some = false;
    int b;
    if (each) {
        b = unit / each;
        unit -= b * each;
    } else
        b = kv_find(c, unit, lane, [](const KvEntry& e) { return kv8_most<LOG>(e.row1 - e.row0); });
    if (b >= c.nb) return u;
    const KvEntry e = kv_batch(c, b);
    const int first = e.len - (e.row1 - e.row0);  // the position of row row0
    u.seq = e.seq;
    u.pos0 = ((first >> LOG) + unit) << LOG;
    u.lo = max(first - u.pos0, 0);
    u.hi = min(e.len - 1 - u.pos0, (1 << LOG) - 1);
    u.row0 = (int64_t)e.row0 + u.pos0 - first;
    u.some = kv_current(c) && first >= 0 && u.lo <= u.hi && e.row1 <= c.rows;
    return u;
}

// One block of keys by one wavefront: lane (o, kg) has position o, 16 dims of
// each 64 from 16 kg on (v, 0 where there is none): the bytes that it stores are
// one piece of its own.
template <int WK, int WV>
__device__ __forceinline__ void kv8_put_keys(float (&v)[WK / 64][16], uint8_t* chunk, int t, int lo, int hi, int lane) {
    typedef Kv8Lay<WK, WV> L;
    const int o = lane & 15;
    const bool live = o >= lo && o <= hi;
    Kv8Record* rec = reinterpret_cast<Kv8Record*>(chunk + L::RECORD);
    const float old = lo ? rec->ks[t] : 0.0f;
    const uint32_t old_bad = lo ? rec->kbad[t] & ((1u << lo) - 1u) : 0u;
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
// four by four, its words are whole too.  A whole chunk's go to `img`, which its
// workgroup stores 16 bytes a lane.
template <int TYPE, int WK, int WV>
__device__ __forceinline__ void kv8_put_values(const typename KvElem<TYPE>::T* __restrict__ x, int64_t ld, int dim, bool vec,
                                               uint8_t* chunk, uint8_t* img, int t, int lo, int hi, int lane) {
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
        const T* p = x + (int64_t)slot * ld;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int d = 64 * n + 4 * c;
            if (vec) {
                Vec y = {};
                if (live && d < dim) y = *reinterpret_cast<const Vec*>(p + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[n][r][e] = (float)y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[n][r][e] = live && d + e < dim ? KvElem<TYPE>::get(p + d + e) : 0.0f;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        int wrong = 0;
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                wrong |= !(fabsf(v[n][r][e]) < __builtin_inff());
                top = fmaxf(top, fabsf(v[n][r][e]));
            }
        // (the row's sixteen lanes)
        const uint64_t which = __ballot(wrong != 0);
        bad[r] = (which >> (16 * a) & 0xffffu) != 0;
        if (which) {
#pragma unroll
            for (int g = 0; g < 4; ++g) bads |= (which >> (16 * g) & 0xffffu) ? 1u << (4 * g + r) : 0u;
        }
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
                const uint32_t at = L::v_piece(4 * n + (d >> 4), 16 * a + (d & 15)) + 4 * t;
                uint32_t y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = kv8_code(bad[r] ? 0.0f : v[n][r][e], s.inv);
                uint32_t w = low_bytes(y[0], y[1], y[2], y[3]);
                if (img) {
                    *reinterpret_cast<uint32_t*>(img + at - L::VALUES) = w;
                    continue;
                }
                uint32_t* p = reinterpret_cast<uint32_t*>(chunk + at);
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

// How keys find the other of a pair: interleaved, both are a lane's; in halves too
// where there are 64 or 128 pairs; else by LDS.
constexpr int KV8_APART = 1, KV8_NEIGHBOURS = 2, KV8_HALVES = 3;

// The cosines and sines of a block's new rows, shared out over the threads:
// [16][kv8_angles_ld] (rows apart by 16 bytes of the banks).
__host__ __device__ __forceinline__ int kv8_angles_ld(int pairs) { return pairs + 2 - (pairs & 1); }
__device__ __forceinline__ void kv8_angles(const Kv8Append& a, const Kv8Unit& u, float2* cs) {
    const int pairs = a.r.pairs, ld = kv8_angles_ld(pairs);
    for (int i = threadIdx.x; i < (u.hi - u.lo + 1) * pairs; i += 256) {
        const int slot = u.lo + i / pairs, pair = i % pairs;
        cs[slot * ld + pair] = rope_cos_sin(a.r.turns[pair], a.pos ? a.pos[u.row0 + slot] : u.pos0 + slot, a.r.amplitude);
    }
}

// Rows of some heads' keys turned into LDS, f32 [head][16][LD]: a thread takes V
// pairs (i, i + pairs) (or V dims behind them) of one row, for all the heads.
template <int TYPE, int V, int LD>
__device__ __forceinline__ void kv8_turn_keys(const typename KvElem<TYPE>::T* __restrict__ k, int64_t ld, int dim, int heads,
                                              const Kv8Unit& u, int pairs, const float2* cs, float* to) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef float Out __attribute__((ext_vector_type(V)));
    const int turned = pairs / V, units = turned + (dim - 2 * pairs) / V;
    for (int i = threadIdx.x; i < (u.hi - u.lo + 1) * units; i += 256) {
        const int slot = u.lo + i / units, n = i % units;
        const bool turns = n < turned;
        const int d0 = turns ? n * V : 2 * pairs + (n - turned) * V, d1 = turns ? d0 + pairs : d0;
        const T* x = k + (u.row0 + slot) * ld;
        float* y = to + slot * LD;
        Vec x0[KV8_HEADS], x1[KV8_HEADS];
#pragma unroll
        for (int h = 0; h < KV8_HEADS; ++h) {
            x0[h] = *reinterpret_cast<const Vec*>(x + (int64_t)min(h, heads - 1) * dim + d0);
            x1[h] = *reinterpret_cast<const Vec*>(x + (int64_t)min(h, heads - 1) * dim + d1);
        }
        float2 w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = turns ? cs[slot * kv8_angles_ld(pairs) + n * V + e] : float2{1.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < KV8_HEADS; ++h) {
            Out y0, y1;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 z = rope_turn((float)x0[h][e], (float)x1[h][e], w[e]);
                y0[e] = turns ? z.x : (float)x0[h][e], y1[e] = z.y;
            }
            *reinterpret_cast<Out*>(y + h * 16 * LD + d0) = y0;
            if (turns) *reinterpret_cast<Out*>(y + h * 16 * LD + d1) = y1;
        }
    }
}

// A workgroup takes
//   a block of 16 positions and four heads of the keys, a wavefront a head.  Turned
//   keys: the block's cosines and sines through LDS, shared out over the threads;
//   where a pair's dims are not one lane's, the heads' rows go through LDS too;
//   a chunk of 64 positions and one head of the values, a wavefront a block;
//   a block of 16 positions and some heads of the queries.
// A block's step is a maximum over one wavefront's lanes, and no two workgroups
// share a block, so rows that join one are stored by reading, halving and writing
// it.
// Bytes bound it: 7,490 rows of three prompts, 8 heads of 128 + 128 turned with 32
// query heads, bf16 (169 MB) 34 to 37 us, 4.6 to 5 TB/s; their keys and values alone (46
// MB) 13.5, turned 18, where a copy would take 8.9: a wavefront has one block's rows in
// flight and then their codes to work out; a row of each of 8 sequences 5.1 us, latency.  All three roles in one workgroup kept 386 scalar registers spilled
// and took twice as long; keys' rows through LDS where a lane holds both of a pair cost
// 4 us of the 34.
template <int TYPE, int WK, int WV, int TURN>
__global__ __launch_bounds__(256) void k_kv8_append(Kv8View c, Kv8Append a, Kv8AppendPlan p) {
    typedef typename KvElem<TYPE>::T T;
    typedef Kv8Lay<WK, WV> L;
    constexpr int LD = WK + 4;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bid = blockIdx.y * gridDim.x + blockIdx.x;
    if (bid >= p.grid) return;
    if (bid < p.k_grid) {
        const int h0 = bid % p.k_parts * KV8_HEADS, heads = min(KV8_HEADS, c.heads - h0);
        const Kv8Unit u = kv8_unit<4>(c, bid / p.k_parts, p.blocks_each, lane);
        if (!u.some) return;
        const int pg = kv_page(c, u.seq, u.pos0);
        if (pg < 0) return;
        const T* k = reinterpret_cast<const T*>(a.k) + (int64_t)h0 * c.dk;
        float v[L::NJ][16];
        const int o = lane & 15, kg = lane >> 4;
        const bool live = o >= u.lo && o <= u.hi;
        if constexpr (TURN == KV8_APART) {
            float* rows = reinterpret_cast<float*>(lds);
            float2* cs = reinterpret_cast<float2*>(rows + KV8_HEADS * 16 * LD);
            kv8_angles(a, u, cs);
            __syncthreads();
            if (p.widek)
                kv8_turn_keys<TYPE, 4, LD>(k, a.ldk, c.dk, heads, u, a.r.pairs, cs, rows);
            else
                kv8_turn_keys<TYPE, 1, LD>(k, a.ldk, c.dk, heads, u, a.r.pairs, cs, rows);
            __syncthreads();
            if (wave >= heads) return;
            const float* x = rows + (wave * 16 + o) * LD;
#pragma unroll
            for (int j = 0; j < L::NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 64 * j + 16 * kg + 4 * i;
                    const f32x4 y = *reinterpret_cast<const f32x4*>(x + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[j][4 * i + e] = live && d + e < c.dk ? y[e] : 0.0f;
                }
        } else {
            const T* x = k + (u.row0 + o) * a.ldk + (int64_t)min(wave, heads - 1) * c.dk;
#pragma unroll
            for (int j = 0; j < L::NJ; ++j)
#pragma unroll
                for (int g = 0; g < 2; ++g) kv8_take8<TYPE>(x, 64 * j + 16 * kg + 8 * g, live ? c.dk : 0, p.veck, v[j] + 8 * g);
            if constexpr (TURN != 0) {
                float2* cs = reinterpret_cast<float2*>(lds);
                kv8_angles(a, u, cs);
                __syncthreads();
                const float2* w = cs + o * kv8_angles_ld(a.r.pairs);
                if (live) {
                    if constexpr (TURN == KV8_NEIGHBOURS) {
#pragma unroll
                        for (int j = 0; j < L::NJ; ++j)
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                const int i = (64 * j + 16 * kg + e) / 2;
                                if (i < a.r.pairs) {
                                    const float2 z = rope_turn(v[j][e], v[j][e + 1], w[i]);
                                    v[j][e] = z.x, v[j][e + 1] = z.y;
                                }
                            }
                    } else {  // (KV8_HALVES: pairs is a multiple of 64, so both of a pair are this lane's)
                        const auto turn = [&](float (&y)[16], float (&z)[16], int j) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float2 both = rope_turn(y[e], z[e], w[64 * j + 16 * kg + e]);
                                y[e] = both.x, z[e] = both.y;
                            }
                        };
                        if (a.r.pairs == 64) {
                            if constexpr (L::NJ >= 2) turn(v[0], v[1], 0);
                        } else if constexpr (L::NJ >= 4) {
                            turn(v[0], v[2], 0);
                            turn(v[1], v[3], 1);
                        }
                    }
                }
            }
            if (wave >= heads) return;
        }
        uint8_t* chunk = kv8_block(c, pg, a.layer, h0 + wave) + (uint32_t)((u.pos0 & (c.page() - 1)) >> 6) * L::CHUNK;
        kv8_put_keys<WK, WV>(v, chunk, u.pos0 >> 4 & 3, u.lo, u.hi, lane);
        return;
    }
    bid -= p.k_grid;
    if (bid < p.v_grid) {
        const int h = bid % c.heads;
        const Kv8Unit u = kv8_unit<6>(c, bid / c.heads, p.chunks_each, lane);
        if (!u.some) return;
        const int pg = kv_page(c, u.seq, u.pos0);
        if (pg < 0) return;
        uint8_t* chunk = kv8_block(c, pg, a.layer, h) + (uint32_t)((u.pos0 & (c.page() - 1)) >> 6) * L::CHUNK;
        const bool whole = u.lo == 0 && u.hi == 63;
        const int t = wave, lo = max(u.lo - 16 * t, 0), hi = min(u.hi - 16 * t, 15);
        if (lo <= hi) {
            const T* x = reinterpret_cast<const T*>(a.v) + (u.row0 + 16 * t) * a.ldv + (int64_t)h * c.dv;
            kv8_put_values<TYPE, WK, WV>(x, a.ldv, c.dv, p.vecv, chunk, whole ? lds : nullptr, t, lo, hi, lane);
        }
        if (whole) {
            __syncthreads();
            for (int i = tid; i < 4 * WV; i += 256)
                reinterpret_cast<u32x4*>(chunk + L::VALUES)[i] = reinterpret_cast<const u32x4*>(lds)[i];
        }
        return;
    }
    if constexpr (TURN != 0) {
        bid -= p.v_grid;
        const int h0 = bid % p.q_parts * p.q_share, h1 = min(h0 + p.q_share, a.q.heads);
        const Kv8Unit u = kv8_unit<4>(c, bid / p.q_parts, p.blocks_each, lane);
        if (!u.some) return;
        const RopeArgs q{a.r, nullptr, a.q, RopeRows{}, 0, c.dk, 0};
        for (int i = tid; i < (u.hi - u.lo + 1) * p.rope.units; i += 256) {
            const int slot = u.lo + i / p.rope.units, n = i % p.rope.units;
            const int64_t row = u.row0 + slot;
            const int pos = a.pos ? a.pos[row] : u.pos0 + slot;
            if (p.wide)
                rope_rows<TYPE, 4, TURN == KV8_NEIGHBOURS>(q, p.rope, row, n, pos, h0, h1);
            else
                rope_rows<TYPE, 1, TURN == KV8_NEIGHBOURS>(q, p.rope, row, n, pos, h0, h1);
        }
    }
}

template <int TYPE, int WK, int WV>
static hipError_t append_typed(const Kv8View& c, const int* row0, const Kv8Append& a, hipStream_t s) {
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    Kv8AppendPlan p = {};
    p.blocks_each = kv8_most<4>(c.each);
    p.chunks_each = kv8_most<6>(c.each);
    int64_t blocks = (int64_t)p.blocks_each * c.nb, chunks = (int64_t)p.chunks_each * c.nb;
    if (!c.each)
        for (int b = 0; b < c.nb; ++b) {
            blocks += kv8_most<4>(row0[b + 1] - row0[b]);
            chunks += kv8_most<6>(row0[b + 1] - row0[b]);
        }
    p.veck = c.dk % 8 == 0 && (uintptr_t)a.k % 16 == 0 && a.ldk * es % 16 == 0 && c.dk * es % 16 == 0;
    p.vecv = c.dv % 4 == 0 && (uintptr_t)a.v % (4 * es) == 0 && a.ldv % 4 == 0;
    const bool turn = a.r.turns != nullptr;
    p.k_parts = (c.heads + KV8_HEADS - 1) / KV8_HEADS;
    const int64_t k_grid = blocks * p.k_parts, v_grid = chunks * c.heads;
    if (turn) {
        const RopeArgs k{a.r, nullptr, {a.k, nullptr, a.ldk, 4, c.heads}, RopeRows{}, 0, c.dk, 0};
        p.widek = rope_takes4(k, es);
        if (a.q.heads) {
            const RopeArgs q{a.r, nullptr, a.q, RopeRows{}, 0, c.dk, 0};
            p.wide = rope_takes4(q, es);
            p.rope = rope_plan(q, p.wide ? 4 : 1);
            p.q_share = std::min(a.q.heads, 8);
            p.q_parts = (a.q.heads + p.q_share - 1) / p.q_share;
        }
    }
    const int64_t grid = k_grid + v_grid + blocks * p.q_parts;
    // (beyond the threads of a launch in x they go on in y)
    const int64_t x = grid > KV8_THREADS / 256 ? 1 << 22 : grid, y = (grid + x - 1) / x;
    if (grid > INT32_MAX - x) return hipErrorInvalidValue;
    p.k_grid = (int)k_grid;
    p.v_grid = (int)v_grid;
    p.grid = (int)grid;
    const int how = !turn ? 0 : a.r.interleaved ? KV8_NEIGHBOURS : a.r.pairs % 64 == 0 ? KV8_HALVES : KV8_APART;
    // keys' rows and angles, or a chunk's values
    const size_t angles = turn ? (size_t)16 * kv8_angles_ld(a.r.pairs) * sizeof(float2) : 0;
    const size_t lds = std::max<size_t>(64 * WV, angles + (how == KV8_APART ? (size_t)KV8_HEADS * 16 * (WK + 4) * 4 : 0));
    auto kern = how == 0                ? k_kv8_append<TYPE, WK, WV, 0>
                : how == KV8_NEIGHBOURS ? k_kv8_append<TYPE, WK, WV, KV8_NEIGHBOURS>
                                        : k_kv8_append<TYPE, WK, WV, KV8_APART>;
    if constexpr (WK >= 128)
        if (how == KV8_HALVES) kern = k_kv8_append<TYPE, WK, WV, KV8_HALVES>;
    if (lds > 65536) {
        // (more than a kernel may have without being asked for it)
        if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds))
            return e;
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)x, (unsigned)y), dim3(256), lds, s, c, a, p);
    return hipGetLastError();
}

// ------------------------------------------------------------------- read
// A workgroup reads one head's rows of one chunk, a wavefront a block: keys as
// their lanes hold them, values four positions by four dims, their pieces 16 bytes
// a lane by LDS.  The 7,490 rows above (46 MB) 12 us, 3.8 TB/s; 8 rows 4.5.
// Few spans are few arguments: a launch's are read from host memory (3.9 KB of them
// make a microsecond of a read of 8 rows).
struct Kv8FewSpans {
    static constexpr int MAX = 16;
    int n;
    int seq[MAX], pos[MAX], row0[MAX + 1], unit0[MAX + 1];
};

template <int TYPE, int WK, int WV, class Spans>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8View c, int layer0, Spans p, int64_t rows, int64_t row_at,
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
    __shared__ __align__(16) uint8_t img[64 * WV];
    for (int i = tid; i < 4 * WV; i += 256)
        reinterpret_cast<u32x4*>(img)[i] = reinterpret_cast<const u32x4*>(chunk + L::VALUES)[i];
    __syncthreads();
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
            w[e] = *reinterpret_cast<const uint32_t*>(img + L::v_piece(4 * n + (cc >> 2), 16 * a + 4 * (cc & 3) + e) - L::VALUES + 4 * t);
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
    if (blocks > KV8_THREADS / 256) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, layer < 0 ? c.layers : 1);
    if (p.n <= Kv8FewSpans::MAX) {
        Kv8FewSpans few;
        few.n = p.n;
        for (int i = 0; i < p.n; ++i) few.seq[i] = p.seq[i], few.pos[i] = p.pos[i];
        for (int i = 0; i <= p.n; ++i) few.row0[i] = p.row0[i], few.unit0[i] = p.unit0[i];
        hipLaunchKernelGGL((k_kv8_read<TYPE, WK, WV, Kv8FewSpans>), grid, dim3(256), 0, s, c, layer < 0 ? 0 : layer, few, rows, row,
                           (T*)k, (T*)v, veck, vecv);
    } else
        hipLaunchKernelGGL((k_kv8_read<TYPE, WK, WV, KvSpans>), grid, dim3(256), 0, s, c, layer < 0 ? 0 : layer, p, rows, row, (T*)k,
                           (T*)v, veck, vecv);
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
