// Attention of a batch's rows over the 4-bit cache (the layout: nh_kv4.h).
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= i of row i's
//   sequence; with a ring also j < sink or j > i - ring.
//
// With k_j = low + step c_j per group g, and the same of v_j:
//   scale q . k_j = cq sum_g step_jg (q_g . c_jg) + sum_g low_jg (scale sum q_g)
//   o = (sum_g sum_j (p_j step_jg) c_jg + sum_j p_j low_jg) / sum_j p_j
// The two sums over low are matrix products of their own, with the lows as they
// are stored: of the queries' sums (two f16 parts, 22 bits) and of the weights,
// so the codes themselves are the matrix operands: a code 0 .. 15 under a
// 16-bit mask is the f16 subnormal c 2^-24 (under the next nibble's mask 16 c
// 2^-24), which the f16 MFMAs take exactly; unpacking is one AND for two
// codes, and no value is dequantized.  The powers of two go into q and the
// result.  The products are transposed, keys (or dims) by rows: S^T = K Q^T
// leaves lane (row = lane % 16, kg = lane / 16) the scores of its row's keys 4 kg
// + 0..3 of each 16, which is the operand that O^T = V^T P^T wants of that lane
// (the order of the summed keys is free), so a weight never leaves its lane, and
// a row's maximum, sum and correction are one lane's scalars.
//
// Bound by the codes' bytes where keys are many: 64 sequences of 4,096 to 8,192
// keys, 8 kv heads of 128 under 32, bf16 (511 MB): 110 us, 4.65 TB/s, what a
// large copy reaches.  A wavefront's 32 keys cost about 300 vector instructions
// (masks, steps, exponentials) beside 19 MFMAs, 0.87 us a SIMD, so where one
// sequence has all the keys the two are about equal: 131,072 keys (151 MB, f16) 41
// us with the join.  Few keys are latency: 374 of them 7.8 us.
#include <algorithm>
#include <type_traits>

#include "nh_kv4_device.h"

namespace nh {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int KA_CHUNK = 32;   // keys of a step of a wavefront; a page holds whole chunks
constexpr float KA_LOG2E = 1.44269504088896340736f;

// The value of lane `I` of each row of 16 lanes (DPP row_newbcast).
template <int I>
__device__ __forceinline__ float row_bcast(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + I, 0xF, 0xF, true));
}
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

template <int I, int N, class F>
__device__ __forceinline__ void static_for(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>());
        static_for<I + 1, N>(f);
    }
}

struct KaPlan {
    int splits;      // key ranges of a sequence; more than one: partial results go to the workspace
    int tiles_each;  // row tiles of every sequence when they are equal, else 0
    int aligned;     // rows of q can be read 8 elements at a time
    int out_aligned; // rows of out can be written 4 elements at a time
};

// The chunks that a tile of rows at positions lo .. hi sees: [0, ns) and [w, n).
struct KaSpan {
    int ns, w, n;
    __device__ __forceinline__ KaSpan(int lo, int hi, int sink, int ring) {
        n = hi / KA_CHUNK + 1;
        ns = 0, w = 0;
        if (ring) {
            ns = min((int)(((int64_t)sink + KA_CHUNK - 1) / KA_CHUNK), n);
            w = max(ns, max(0, lo - ring + 1) / KA_CHUNK);
        }
    }
    __device__ __forceinline__ int count() const { return ns + n - w; }
    __device__ __forceinline__ int at(int i) const { return i < ns ? i : i - ns + w; }
};

// What a lane loads of a chunk: two tiles of 16 keys.
template <int W, int NG>
struct KaChunk {
    static constexpr int NS = (4 * NG + 15) / 16;
    static constexpr int NL = (NG + 1) / 2;  // dwords of a key's lows
    uint32_t k[2][W / 32], v[2][W / 32], kl[2][NL], vl[2][2];
    uint16_t ks[2][NS], vs[2][NS];
};

// NW wavefronts a workgroup, each every NW-th chunk of the range; RT tiles of 16 rows.
template <int TYPE, int W, int G, int RT, int NW>
__global__ __launch_bounds__(NW * 64, W <= 128 ? 2 : 1) void k_kv4_attend(Kv4View c, Kv4AttendArgs a, KaPlan plan) {
    typedef typename Kv4Elem<TYPE>::T T;
    constexpr int NG = W / G, NB = W / 64, NJ = W / 32, GJ = G / 32, GI = G / 16;
    constexpr int PARTS = TYPE == KV4_F32 ? 2 : 1;   // f16 halves of a query element
    // ..  and of a weight.  One leaves up to three roundings of an f16 output (4.6e-4
    // of it instead of 2.1e-4, 20 keys; 131,072 keys: 38.6 us, 41.0 with two), but
    // a tenth of a bf16 output's one.
    constexpr int WPARTS = TYPE == KV4_BF16 ? 1 : 2;
    // The MFMAs take a subnormal as it is, but line its products up by the exponent
    // of the smallest normal number: up to 2^-17 of the largest product is cut off
    // (2^-20 with normal operands, both measured).  Calls that carry 22 bits bring
    // their codes up by 2^14 first, one more instruction for two codes.
    constexpr int UP = PARTS == 2 ? 14 : 0;
    auto operand = [](u32x4 y) {
        h8 z = __builtin_bit_cast(h8, y);
        if constexpr (PARTS == 2) z *= (_Float16)16384.0f;
        return z;
    };
    typedef KaChunk<W, NG> Chunk;
    constexpr int LD = W + 4;
    constexpr uint32_t CB = 32 * (W + 8 * NG);
    __shared__ float so[NW][16][LD];
    __shared__ float sm[NW][16], sl[NW][16], spl[NW][16][8];

    const int tid = threadIdx.x, lane = tid & 63, o = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % c.heads, per = a.heads / c.heads, split = blockIdx.y;

    // The sequence and the rows of this tile.
    int tile = blockIdx.x / c.heads, b;
    if (plan.tiles_each) {
        b = tile / plan.tiles_each;
        tile -= b * plan.tiles_each;
    } else {
        b = kv4_find(c, tile, lane, [&](const Kv4Entry& e) { return ((e.row1 - e.row0) * per + 16 * RT - 1) / (16 * RT); });
    }
    if (b >= c.nb) return;
    const Kv4Entry entry = kv4_batch(c, b);
    const int row0 = entry.row0, nrows = entry.row1 - row0, seq = entry.seq;
    const int first = entry.len - nrows, r0 = tile * 16 * RT;
    if (!kv4_current(c) || first < 0 || r0 >= nrows * per || entry.row1 > c.rows) return;
    const int r1 = min(r0 + 16 * RT, nrows * per) - 1;
    const int plo = first + r0 / per, phi = first + r1 / per;

    // The queries: f16 operands scaled by a power of two to just under 2^15,
    // elements 2, 3, 6, 7 of 8 by 1/16 for their codes' 16; the sums of each group.
    h8 q[RT][PARTS][NJ];
    h8 qs[RT];
    float cq[RT];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(r0 + rt * 16 + o, r1), t = r / per;
        pos[rt] = first + t;
        const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + t) * a.ldq + (int64_t)(kvh * per + r - t * per) * c.dk;
        float x[NJ][8], most = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int d = j * 32 + kg * 8;
            if (plan.aligned) {
                typedef T Vec __attribute__((ext_vector_type(8)));
                Vec y = {};
                if (d < c.dk) y = *reinterpret_cast<const Vec*>(src + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = (float)y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = d + e < c.dk ? Kv4Elem<TYPE>::get(src + d + e) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[j][e]));
        }
        most = groups_max(most);
        const int ef = max((int)(__builtin_bit_cast(uint32_t, most) >> 23 & 255u), 15);
        const float up = __builtin_bit_cast(float, (uint32_t)(268 - ef) << 23);
        // scores: (2^(18 - UP) sum step z + low . qs) cq, z = 2^(UP - 24) up (q . c), qs = 2^-6 up sum q
        cq[rt] = (a.scale * KA_LOG2E * 64.0f) * __builtin_bit_cast(float, (uint32_t)(ef - 14) << 23);
        qs[rt] = h8{};
        static_for<0, NG>([&](auto GG) {
            constexpr int g = GG.value;
            float s = 0.0f;
#pragma unroll
            for (int j = g * GJ; j < (g + 1) * GJ; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s += x[j][e] * up;
            s = groups_sum(s) * 0.015625f;
            const _Float16 hi = (_Float16)s, lo = (_Float16)(s - (float)hi);
            qs[rt][g] = kg == 0 ? hi : kg == 1 ? lo : (_Float16)0.0f;
        });
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = x[j][e] * up, f = e & 2 ? 0.0625f : 1.0f;
                const _Float16 hi = (_Float16)y;
                q[rt][0][j][e] = (_Float16)((float)hi * f);
                if constexpr (PARTS == 2) q[rt][1][j][e] = (_Float16)((y - (float)hi) * f);
            }
    }

    f32x4 acc[RT][W / 16];
    f32x4 accl[RT];  // 2^15 sum_j p_j low_jg: group 4 kg + r
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff();
        l[rt] = 0.0f;
        accl[rt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < W / 16; ++i) acc[rt][i] = f32x4{0, 0, 0, 0};
    }
    // The weights are kept as 2^15 p, and with their steps as the f16 operand
    // 2^15 p step / 2^eref, 2^eref above every step seen so far: at most 2^15,
    // and exact to 11 bits down to 2^-29 of it.
    int eref = -24;

    const KaSpan span(plo, phi, a.sink, a.ring);
    const int sink = a.ring ? a.sink : 0x7fffffff, ring = a.ring;
    const int per_split = max((span.count() + plan.splits - 1) / plan.splits, NW);
    const int c0 = split * per_split, c1 = min(c0 + per_split, span.count());

    const int* table = c.table + (size_t)seq * c.table_ld;
    auto page_of = [&](int i) { return i < c1 ? table[span.at(i) * KA_CHUNK >> c.page_log2] : 0; };
    const uint32_t sidx = o & (4 * NG - 1);
    auto load = [&](Chunk& x, int i, int pg) {
        const int slot = span.at(i) * KA_CHUNK & (c.page() - 1);
        // (a page id comes from the cache's own table; a bad one is not followed)
        const uint8_t* blk = kv4_block(c, (unsigned)pg < (unsigned)c.pages ? pg : 0, a.layer, kvh);
        blk += (uint32_t)(slot >> 5) * CB;
        // (the lane's 2 W / 32 dwords of each, 16 bytes a piece)
#pragma unroll
        for (int u = 0; u < 2 * NJ; u += 4) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(blk + (u >> 2) * 1024 + lane * 16);
            const u32x4 v = *reinterpret_cast<const u32x4*>(blk + 16 * W + (u >> 2) * 1024 + lane * 16);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                x.k[(u + n) / NJ][(u + n) % NJ] = k[n];
                x.v[(u + n) / NJ][(u + n) % NJ] = v[n];
            }
        }
        const uint8_t* scales = blk + 32 * W;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t so = ((uint32_t)(16 * t + 4 * kg) * NG + sidx) * 2;
#pragma unroll
            for (int n = 0; n < Chunk::NS; ++n) {
                x.ks[t][n] = kv4_half(scales, so + 32 * n);
                x.vs[t][n] = kv4_half(scales, 128 * NG + so + 32 * n);
            }
            const uint32_t kl = 64 * NG + (uint32_t)(16 * t + o) * NG * 2;
            if constexpr (NG == 1)
                x.kl[t][0] = kv4_half(scales, kl);
            else
#pragma unroll
                for (int n = 0; n < NG / 2; ++n) x.kl[t][n] = kv4_word(scales, kl + 4 * n);
            const uint32_t vl = 192 * NG + ((uint32_t)(4 * t + kg) * NG + (o & (NG - 1))) * 8;
#pragma unroll
            for (int n = 0; n < 2; ++n) x.vl[t][n] = kv4_word(scales, vl + 4 * n);
        }
    };

    auto compute = [&](const Chunk& x, int i) {
        const int key0 = span.at(i) * KA_CHUNK;
        const bool whole = key0 + KA_CHUNK - 1 <= plo &&
                           (key0 + KA_CHUNK - 1 < sink || key0 > phi - ring);
        // The steps' reference: raised (a wavefront at a time) when a step passes it.
        uint32_t top = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < Chunk::NS; ++n) {
                const uint32_t s = x.vs[t][n];
                const int key = key0 + 16 * t + 4 * kg + (int)(sidx & 3);
                if (s < 0x7c00u && key <= phi) top = max(top, s);
            }
        // step < 2^(e - 14) for the f16 exponent field e (subnormals below 2^-14)
        if (__any((int)(top >> 10) - 14 > eref)) {
            int e = (int)(top >> 10) - 14;
#pragma unroll
            for (int h = 1; h < 64; h <<= 1) e = max(e, __shfl_xor(e, h, 64));
            const float down = pow2i(max(eref - e, -126));
            eref = __builtin_amdgcn_readfirstlane(e);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < W / 16; ++k) acc[rt][k] *= down;
        }
        const float wscale = pow2i(-eref);
        float kstep[2][Chunk::NS], vstep[2][Chunk::NS];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < Chunk::NS; ++n) {
                kstep[t][n] = f16_value(x.ks[t][n]) * pow2i(18 - UP);
                vstep[t][n] = f16_value(x.vs[t][n]) * wscale;
            }
        h8 ka[2][NJ];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t w = x.k[t][j], z = w >> 8;
                const u32x4 y = {w & 0x000f000fu, w & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u};
                ka[t][j] = operand(y);
            }
        h8 pw[RT][NG][WPARTS];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const bool fresh = m[rt] == -__builtin_inff();  // no key seen yet
            const float base = fresh ? 0.0f : m[rt];
            float s[2][4];  // 15 + log2 of the weight against the maximum so far
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                u32x4 y = {};
#pragma unroll
                for (int n = 0; n < Chunk::NL; ++n) y[n] = x.kl[t][n];
                f32x4 lows = {0, 0, 0, 0};
                lows = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, y), qs[rt], lows, 0, 0, 0);
                f32x4 z[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    z[g] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = g * GJ; j < (g + 1) * GJ; ++j)
#pragma unroll
                        for (int p = 0; p < PARTS; ++p)
                            z[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t][j], q[rt][p][j], z[g], 0, 0, 0);
                }
                static_for<0, 4>([&](auto R) {
                    constexpr int r = R.value;
                    float sum = lows[r];
                    static_for<0, NG>([&](auto GG) {
                        constexpr int g = GG.value, at = r * NG + g;
                        sum = __builtin_fmaf(row_bcast<at % 16>(kstep[t][at / 16]), z[g][r], sum);
                    });
                    s[t][r] = __builtin_fmaf(sum, cq[rt], 15.0f - base);
                });
            }
            bool seen[2][4];
            if (!whole) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = key0 + 16 * t + 4 * kg + r;
                        seen[t][r] = (j <= pos[rt]) & ((j < sink) | (j > pos[rt] - ring));
                        s[t][r] = seen[t][r] ? s[t][r] : -__builtin_inff();
                    }
            }
            float most = s[0][0];
#pragma unroll
            for (int k = 1; k < 8; ++k) most = fmaxf(most, s[k / 4][k % 4]);
            most = groups_max(most);
            if (__any(most > 15.0f || fresh)) {
                // A new maximum (the first: whatever it is).
                const float over = most == -__builtin_inff() ? 0.0f : fresh ? most - 15.0f : fmaxf(most - 15.0f, 0.0f);
                const float keep = fresh ? 0.0f : __builtin_amdgcn_exp2f(-over);
                m[rt] = fresh && most == -__builtin_inff() ? m[rt] : base + over;
                l[rt] *= keep;
                accl[rt] *= keep;
#pragma unroll
                for (int k = 0; k < W / 16; ++k) acc[rt][k] *= keep;
#pragma unroll
                for (int k = 0; k < 8; ++k) s[k / 4][k % 4] -= over;
            }
            float p[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                p[k] = __builtin_amdgcn_exp2f(s[k / 4][k % 4]);
                l[rt] += p[k];
            }
            // Two numbers to f16 at a time; f32 and f16 calls carry what that rounds off.
            auto halves = [&](const float* w, h8* to) {
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const f32x2 y = {w[k], w[k + 1]};
                    const h2 hi = __builtin_convertvector(y, h2);
                    to[0][k] = hi[0], to[0][k + 1] = hi[1];
                    if constexpr (WPARTS == 2) {
                        to[1][k] = (_Float16)(w[k] - (float)hi[0]);
                        to[1][k + 1] = (_Float16)(w[k + 1] - (float)hi[1]);
                    }
                }
            };
            h8 pp[WPARTS];
            halves(p, pp);
            const u32x4 vl = {x.vl[0][0], x.vl[0][1], x.vl[1][0], x.vl[1][1]};
#pragma unroll
            for (int k = 0; k < WPARTS; ++k)
                accl[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, vl), pp[k], accl[rt], 0, 0, 0);
            static_for<0, NG>([&](auto GG) {
                constexpr int g = GG.value;
                float w[8];
                static_for<0, 8>([&](auto K) {
                    constexpr int k = K.value, at = g * 4 + k % 4;
                    w[k] = p[k] * row_bcast<at % 16>(vstep[k / 4][at / 16]);
                });
                if (!whole)  // (a step may be NaN: a hidden key's weight is none)
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = seen[k / 4][k % 4] ? w[k] : 0.0f;
                halves(w, pw[rt][g]);
            });
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            // dword (token pair, n) of each quad: dims 64 n + 32 (i / 2) + 2 o + i % 2
            const uint32_t w[4] = {x.v[0][n], x.v[0][NB + n], x.v[1][n], x.v[1][NB + n]};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u32x4 y;
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = (i & 2 ? w[k] >> 8 : w[k]) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
                const h8 va = operand(y);
                const int d = 4 * n + i;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int p = 0; p < WPARTS; ++p)
                        acc[rt][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pw[rt][d / GI][p], acc[rt][d], 0, 0, 0);
            }
        }
    };

    // The loads of the next two chunks are in flight during this one's
    // arithmetic, the page id of the third is on its way.
    {
        Chunk x[3];
        int i = c0 + wave;
        auto fetch = [&](Chunk& to, int at, int pg) {
            if (at < c1) load(to, at, pg);
        };
        int p0 = page_of(i), p1 = page_of(i + NW), p2 = page_of(i + 2 * NW);
        fetch(x[0], i, p0);
        fetch(x[1], i + NW, p1);
        while (i < c1) {
#pragma unroll
            for (int k = 0; k < 3; ++k, i += NW) {
                if (i >= c1) break;
                fetch(x[(k + 2) % 3], i + 2 * NW, p2);
                p2 = page_of(i + 3 * NW);
                compute(x[k], i);
            }
        }
    }

    // The wavefronts' sums joined, 16 rows at a time.
    const float unit = pow2i(24 - 15 - UP + eref);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = groups_sum(l[rt]);
        if (l[rt] != l[rt]) m[rt] = l[rt];  // NaN scores: the row's, whatever other ranges hold
        if (rt) __syncthreads();
        if (kg == 0) sm[wave][o] = m[rt], sl[wave][o] = l[rt] * 0x1p-15f;
        if (4 * kg < NG) *reinterpret_cast<f32x4*>(&spl[wave][o][4 * kg]) = accl[rt] * 0x1p-15f;
        __syncthreads();
        float most = sm[0][o];
#pragma unroll
        for (int w = 1; w < NW; ++w) most = fmaxf(most, sm[w][o]);
        const float base = most == -__builtin_inff() ? 0.0f : most;
        const float f = __builtin_amdgcn_exp2f(m[rt] - base);
#pragma unroll
        for (int i = 0; i < W / 16; i += 2) {
            // products i, i + 1: dims 16 i + 8 kg + 2 r, and the ones after them
            const float low = spl[wave][o][i / GI];
            f32x4 y, z;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                y[2 * r] = (acc[rt][i][r] * unit + low) * f;
                y[2 * r + 1] = (acc[rt][i + 1][r] * (unit * 0.0625f) + low) * f;
                z[2 * r] = (acc[rt][i][r + 2] * unit + low) * f;
                z[2 * r + 1] = (acc[rt][i + 1][r + 2] * (unit * 0.0625f) + low) * f;
            }
            *reinterpret_cast<f32x4*>(&so[wave][o][16 * i + 8 * kg]) = y;
            *reinterpret_cast<f32x4*>(&so[wave][o][16 * i + 8 * kg + 4]) = z;
        }
        __syncthreads();
        for (int x = tid; x < 16 * W; x += NW * 64) {
            const int rr = x / W, d = x % W, r = r0 + rt * 16 + rr;
            if (r > r1 || d >= c.dv) continue;
            float top = sm[0][rr];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, sm[w][rr]);
            const float zero = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f, v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                sum = __builtin_fmaf(sl[w][rr], __builtin_amdgcn_exp2f(sm[w][rr] - zero), sum);
                v += so[w][rr][d];
            }
            const int t = r / per, head = kvh * per + r - t * per;
            const int64_t row = row0 + t;
            if (plan.splits == 1) {
                Kv4Elem<TYPE>::put(reinterpret_cast<T*>(a.out) + row * a.ldo + (int64_t)head * c.dv + d, v / sum);
                if (a.lse && d == 0) a.lse[row * a.heads + head] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
            } else {
                const int64_t at = ((int64_t)split * c.rows + row) * a.heads + head;
                float* ml = reinterpret_cast<float*>(a.ws);
                ml[2 * ((int64_t)plan.splits * c.rows * a.heads) + at * c.dv + d] = v;
                if (d == 0) ml[2 * at] = sum == sum ? top : sum, ml[2 * at + 1] = sum;
            }
        }
    }
}

// ------------------------------------------------------------------ prompts
// Many rows: a workgroup of eight wavefronts takes 256 rows, 32 a wavefront, and
// the chunks' codes are turned into f16 operands once for all of them, through
// LDS, two chunks in turn.  Keys and values are kept as step x code there,
// rounded to 11 bits, their lows go through the same small products as above, so
// the rounding is relative to a group's range and not to its offset.  A code
// under a mask and 0x6400 is the f16 number 1024 + c; one fused multiply-add
// with the step and -1024 steps leaves step x code, for two codes at a time (an
// AND-OR and the multiply-add).  The power of two over the largest step of the
// range is 2^6 there, so that 1024 steps and 240 steps are f16 numbers: steps down
// to 2^-20 of that power keep their 11 bits, smaller ones leave step x code good
// to 2^-27 of it.  (Codes as subnormals times steps lose bits from 2^-5 on: a row
// 10,000 times the others took 5 % off every result that did not see it, for 1 %
// of the time.)
// 32 x 32 MFMAs: a lane holds 16 scores of its row, the other half of
// them is 32 lanes away.  The weights' sum is one more row of the lows' product.
//
// Two sequences' 2,000 rows after 6,000 keys, 32 heads over 8 of 128, bf16 (427
// GFLOP): 573 us, 745 TFLOP/s (up to 591 by card); the kernel above takes 1,450,
// an operand's masks, steps and lows serving 16 rows there and 256 here.  A large
// library product runs at 1,130 to 1,180.  The matrix cores are busy 37 % of the
// time, the vector units (exponentials, maxima, weights to f16) 43 %, one wavefront's chain of
// scores, maximum, weights and sums being what neither hides from the other.
constexpr int KP_WAVES = 8;
constexpr int KP_ROWS = 32 * KP_WAVES;
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float halves_max(float v) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
}

template <int TYPE, int W, int G>
__global__ __launch_bounds__(KP_WAVES * 64) void k_kv4_prompt(Kv4View c, Kv4AttendArgs a, KaPlan plan) {
    typedef typename Kv4Elem<TYPE>::T T;
    typedef Kv4Lay<W, G> L;
    constexpr int NG = L::NG, NJ = W / 32, NX = W / 16, ND = W / 32;
    struct Image {  // a chunk's operands, 16 bytes a lane each
        u32x4 k[NX][64], kl[64], v[ND][2][64], vl[2][64];
    };
    __shared__ Image img[2][2];

    const int tid = threadIdx.x, lane = tid & 63, o = lane & 15, kg = lane >> 4, half = lane >> 5, m32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % c.heads, per = a.heads / c.heads, split = blockIdx.y;
    int tile = blockIdx.x / c.heads, b;
    if (plan.tiles_each) {
        b = tile / plan.tiles_each;
        tile = plan.tiles_each - 1 - (tile - b * plan.tiles_each);  // the longest first
    } else
        b = kv4_find(c, tile, lane, [&](const Kv4Entry& e) { return ((e.row1 - e.row0) * per + KP_ROWS - 1) / KP_ROWS; });
    if (b >= c.nb) return;
    const Kv4Entry entry = kv4_batch(c, b);
    const int row0 = entry.row0, nrows = entry.row1 - row0, first = entry.len - nrows, r0 = tile * KP_ROWS;
    if (!kv4_current(c) || first < 0 || r0 >= nrows * per || entry.row1 > c.rows) return;
    const int r1 = min(r0 + KP_ROWS, nrows * per) - 1;
    const int plo = first + r0 / per, phi = first + r1 / per;
    const int w0 = min(r0 + wave * 32, r1), w1 = min(w0 + 31, r1);  // this wavefront's rows
    const int wlo = first + w0 / per, whi = first + w1 / per;
    const int sink = a.ring ? a.sink : 0x7fffffff, ring = a.ring;

    const int r = min(r0 + wave * 32 + m32, r1), token = r / per, pos = first + token;
    f32x16 acc[ND], accl = {};
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    float m = -__builtin_inff();

    const KaSpan span(plo, phi, a.sink, a.ring);
    const int per_split = (span.count() + plan.splits - 1) / plan.splits;
    const int c0 = split * per_split, c1 = min(c0 + per_split, span.count());
    const int* table = c.table + (size_t)entry.seq * c.table_ld;
    const uint8_t* layer = kv4_block(c, 0, a.layer, kvh);
    const size_t page_bytes = c.page_bytes();
    const int mask = c.page() - 1;
    auto page_of = [&](int i) { return i < c1 ? table[span.at(i) * KA_CHUNK >> c.page_log2] : 0; };
    auto chunk_at = [&](int i, int pg) {
        const int slot = span.at(i) * KA_CHUNK & mask;
        return layer + ((unsigned)pg < (unsigned)c.pages ? pg : 0) * page_bytes + (uint32_t)(slot >> 5) * L::CHUNK;
    };

    // The references: powers of two, 2^ref above every step of the keys (and values)
    // of this range, and whether a value is NaN.  One look at the steps ahead of
    // the loop: inside it they took a third of the instructions.  The operands' units are
    // 2^unit: 64 steps of the largest's size, fewer where the format's smallest
    // step, 2^-24, keeps its bits without (so that the queries' sums fit, below).
    int kunit, vunit;
    bool nan;
    {
        const uint32_t x2 = 2 * (lane & (16 * NG - 1));  // two steps a lane
        uint32_t top[2] = {0, 0};
        bool bad = false;
        constexpr int DEEP = 8;
        for (int i0 = c0 + wave; i0 < c1; i0 += DEEP * KP_WAVES) {
            // (past the end: the last chunk again, so that every load is in flight at once)
            int pg[DEEP];
            uint32_t w[DEEP][2];
#pragma unroll
            for (int x = 0; x < DEEP; ++x) pg[x] = page_of(min(i0 + x * KP_WAVES, c1 - 1));
#pragma unroll
            for (int x = 0; x < DEEP; ++x) {
                const uint8_t* p = chunk_at(min(i0 + x * KP_WAVES, c1 - 1), pg[x]);
                w[x][0] = kv4_word(p, 32 * W + 2 * x2);
                w[x][1] = kv4_word(p, 32 * W + 128 * NG + 2 * x2);
            }
#pragma unroll
            for (int x = 0; x < DEEP; ++x) {
                const int key0 = span.at(min(i0 + x * KP_WAVES, c1 - 1)) * KA_CHUNK;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const uint32_t k = w[x][0] >> (16 * t) & 0xffffu, v = w[x][1] >> (16 * t) & 0xffffu;
                    const int kkey = key0 + (int)(x2 + t) / NG, vkey = key0 + (int)(x2 / (4 * NG)) * 4 + (int)((x2 + t) & 3);
                    top[0] = max(top[0], (kkey <= phi) & (k < 0x7c00u) ? k : 0u);
                    top[1] = max(top[1], (vkey <= phi) & (v < 0x7c00u) ? v : 0u);
                    bad |= (vkey <= phi) & (v >= 0x7c00u);
                }
            }
        }
        __shared__ uint32_t st[2][KP_WAVES];
        __shared__ int sbad[KP_WAVES];
#pragma unroll
        for (int h = 1; h < 64; h <<= 1) {
            top[0] = max(top[0], (uint32_t)__shfl_xor((int)top[0], h, 64));
            top[1] = max(top[1], (uint32_t)__shfl_xor((int)top[1], h, 64));
        }
        const bool any = __any(bad);
        if (lane == 0) st[0][wave] = top[0], st[1][wave] = top[1], sbad[wave] = any;
        __syncthreads();
        int bads = 0;
#pragma unroll
        for (int w = 0; w < KP_WAVES; ++w) {
            top[0] = max(top[0], st[0][w]);
            top[1] = max(top[1], st[1][w]);
            bads |= sbad[w];
        }
        const int kref = __builtin_amdgcn_readfirstlane((int)(top[0] >> 10)) - 14;
        const int vref = __builtin_amdgcn_readfirstlane((int)(top[1] >> 10)) - 14;
        kunit = max(kref - 6, -10);
        vunit = max(vref - 6, -10);
        nan = __builtin_amdgcn_readfirstlane(bads) != 0;
    }
    const float kmul = pow2i(-kunit), vmul = pow2i(-vunit);

    // The queries, scaled to just under 2^a, and their sums in units that make the
    // lows' product another term of the scores' own accumulator: scores are z cz,
    // z = up (q . step c) 2^-unit + low (up sum q 2^-unit).  The sum of 64 is just under
    // 2^(a + 6 - unit): a takes it to 2^15, so that its two f16 parts hold 22 bits of it,
    // and is -1 at least (unit >= -10), where elements down to 2^-8 of the row's largest
    // keep 11 bits (smaller ones are good to 2^-20 of it).
    h8 q[NX], qs = {};
    float cz;
    {
        const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + token) * a.ldq + (int64_t)(kvh * per + r - token * per) * c.dk;
        float most = 0.0f, sums[NG] = {};
        T x[NX][8];
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const int d = 16 * j + 8 * half;
            typedef T Vec __attribute__((ext_vector_type(8)));
            if (plan.aligned) {
                Vec y = {};
                if (d < c.dk) y = *reinterpret_cast<const Vec*>(src + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = d + e < c.dk ? src[d + e] : (T)0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf((float)x[j][e]));
        }
        most = halves_max(most);
        const int ef = max((int)(__builtin_bit_cast(uint32_t, most) >> 23 & 255u), 15);
        const int size = min(9 + kunit, 15);  // (a)
        const int up = size + 126 - ef;
        cz = __builtin_amdgcn_ldexpf(a.scale * KA_LOG2E, kunit - up);
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = __builtin_amdgcn_ldexpf((float)x[j][e], up);
                sums[j * 16 / G] += y;
                q[j][e] = (_Float16)(y * (e & 2 ? 0.0625f : 1.0f));
            }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float s = (sums[g] + __shfl_xor(sums[g], 32, 64)) * pow2i(-kunit);
            const _Float16 hi = (_Float16)s, lo = (_Float16)(s - (float)hi);
            qs[g] = half == 0 ? hi : lo;
        }
    }

    // What this wavefront turns into operands: key dword (kt, kj), value dwords
    // (vt, vn) under nibbles 2 vi, 2 vi + 1; a few wavefronts also the lows.
    constexpr int UNITS = W == 128 ? 8 : 4;
    const bool does_k = W == 128 || wave < UNITS, does_v = W == 128 || wave >= UNITS;
    const int ku = wave % UNITS, kt = ku / NJ, kj = ku % NJ;
    const int vt = ku & 1, vn = W == 128 ? ku >> 1 & 1 : 0, vi = W == 128 ? ku >> 2 : ku >> 1;
    const uint32_t at_k = L::lane_dword(lane, kt * NJ + kj), at_ks = L::k_step(16 * kt + o, kj * 32 / G);
    const uint32_t at_v = 16 * W + L::lane_dword(lane, vt * NJ + vn);
    const uint32_t at_vs = L::v_step(16 * vt + 4 * kg, (64 * vn + 32 * vi) / G);
    // value lows of keys 16 y + 8 w + 4 half .., y = wave / 2, w = wave % 2; key lows by wavefront 4
    const uint32_t at_low = wave < 4 ? L::v_low(16 * (wave >> 1) + 8 * (wave & 1) + 4 * half, m32 & (NG - 1)) : L::k_low(m32, 0);
    struct Raw {
        uint32_t k, v[2], vs[2], low[2];
        uint16_t ks;
    };
    auto load = [&](Raw& x, int i, int pg) {
        const uint8_t* p = chunk_at(i, pg);
        if (does_k) {
            x.k = kv4_word(p, at_k);
            x.ks = kv4_half(p, at_ks);
        }
        if (does_v) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                x.v[t] = kv4_word(p, at_v + 4 * t * L::NB);
                x.vs[t] = kv4_word(p, at_vs + 4 * t);
            }
        }
        if (wave < 5) {
            if constexpr (NG == 4) {
                x.low[0] = kv4_word(p, at_low);
                x.low[1] = kv4_word(p, at_low + 4);
            } else {
                // (a key's lows take 2 NG bytes)
                x.low[0] = NG == 1 && wave == 4 ? kv4_half(p, at_low) : kv4_word(p, at_low);
                x.low[1] = wave < 4 ? kv4_word(p, at_low + 4) : 0;
            }
        }
    };
    // Codes under a mask times scaled steps s (16 c s under the upper mask), two at a
    // time: (1024 + c) s - 1024 s, rounded once.  (Two literals do not fit an
    // AND-OR: the second one stays in a register, which the empty asm keeps it in.)
    uint32_t k1024 = 0x64006400u;
    asm("" : "+v"(k1024));
    auto times = [&](uint32_t codes, h2 steps) {
        const h2 y = __builtin_elementwise_fma(__builtin_bit_cast(h2, codes | k1024), steps, steps * (_Float16)-1024.0f);
        return __builtin_bit_cast(uint32_t, y);
    };
    auto unpack = [&](const Raw& x, int i, Image& to) {
        const int key0 = span.at(i) * KA_CHUNK;
        if (does_k) {
            float s = f16_value(x.ks) * kmul;
            s = s > 63.96875f ? 63.96875f : s;  // (a hidden key's; NaN stays, a key's reader has to see it)
            const h2 sw = {(_Float16)s, (_Float16)s};
            const uint32_t w = x.k, z = w >> 8;
            const u32x4 y = {times(w & 0x000f000fu, sw), times(w & 0x00f000f0u, sw), times(z & 0x000f000fu, sw),
                             times(z & 0x00f000f0u, sw)};
            to.k[2 * kj + (kg >> 1)][(kg & 1) * 32 + 16 * kt + o] = y;
        }
        if (does_v) {
            float s[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) s[t] = f16_value(x.vs[t >> 1] >> (16 * (t & 1))) * vmul;
            // (hidden keys' steps, and NaN, count as 0: what a NaN does to its readers comes after the products)
            if (nan || key0 + KA_CHUNK - 1 > phi) {
#pragma unroll
                for (int t = 0; t < 4; ++t) s[t] = key0 + 16 * vt + 4 * kg + t <= phi && s[t] == s[t] ? s[t] : 0.0f;
            }
            h2 sw[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const f32x2 y = {s[2 * t], s[2 * t + 1]};
                sw[t] = __builtin_convertvector(y, h2);
            }
            const uint32_t w0 = vi ? x.v[0] >> 8 : x.v[0], w1 = vi ? x.v[1] >> 8 : x.v[1];
            const uint2 even = {times(w0 & 0x000f000fu, sw[0]), times(w1 & 0x000f000fu, sw[1])};
            const uint2 odd = {times(w0 & 0x00f000f0u, sw[0]), times(w1 & 0x00f000f0u, sw[1])};
            uint2* out = reinterpret_cast<uint2*>(&to.v[2 * vn + vi][vt][(kg & 1) * 32 + 2 * o]) + (kg >> 1);
            out[0] = even;
            out[2] = odd;
        }
        if (wave < 4) {
            const bool one = m32 == 8;
            const uint2 y = {one ? 0x3c003c00u : x.low[0], one ? 0x3c003c00u : x.low[1]};
            reinterpret_cast<uint2*>(&to.vl[wave >> 1][lane])[wave & 1] = y;
        } else if (wave == 4) {
            const u32x4 y = {x.low[0], NG == 4 ? x.low[1] : 0, 0, 0};
            to.kl[lane] = y;
        }
    };

    // Two chunks a step.  Their loads run two steps ahead, their operands one: a
    // step's images are written while the one before is used, one barrier a step.
    // The second chunk's scores are started before the first one's weights are
    // worked out, and so on, so that the matrix unit has work under the vector
    // unit's.  Past the end the last chunk is loaded and written again (its keys
    // count as hidden), so that fewer branches cut the instructions in pieces.
    if (c0 < c1) {
        Raw x[2];
        const int end = c1 - 1;
        int pg[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            load(x[u], min(c0 + u, end), page_of(min(c0 + u, end)));
            unpack(x[u], min(c0 + u, end), img[0][u]);
            load(x[u], min(c0 + 2 + u, end), page_of(min(c0 + 2 + u, end)));
            pg[u] = page_of(min(c0 + 4 + u, end));
        }
        __syncthreads();
        int turn = 0;
        for (int i = c0; i < c1; i += 2, turn ^= 1) {
            f32x16 z[2];
            auto scores = [&](int u) {
                const Image& now = img[turn][u];
                z[u] = f32x16{};
                z[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, now.kl[lane]), qs, z[u], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NX; ++j)
                    z[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, now.k[j][lane]), q[j], z[u], 0, 0, 0);
            };
            auto next = [&](int u) {
                unpack(x[u], min(i + 2 + u, end), img[turn ^ 1][u]);
                load(x[u], min(i + 4 + u, end), pg[u]);
                pg[u] = page_of(min(i + 6 + u, end));
            };
            auto weigh = [&](int u) {
                const Image& now = img[turn][u];
                const int key0 = span.at(min(i + u, end)) * KA_CHUNK;
                const bool live = i + u < c1;
                const bool fresh = m == -__builtin_inff();
                const float zero = fresh ? 0.0f : m;
                float s[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_fmaf(z[u][e], cz, 15.0f - zero);
                if (!(live && key0 + KA_CHUNK - 1 <= wlo && (key0 + KA_CHUNK - 1 < sink || key0 > whi - ring))) {
                    const int top = live ? pos : -1;
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = key0 + 8 * (e >> 2) + 4 * half + (e & 3);
                        s[e] = (j <= top) & ((j < sink) | (j > pos - ring)) ? s[e] : -__builtin_inff();
                    }
                }
                float most = s[0];
#pragma unroll
                for (int e = 1; e < 16; ++e) most = fmaxf(most, s[e]);
                most = halves_max(most);
                if (__any(most > 15.0f || fresh)) {
                    const float over = most == -__builtin_inff() ? 0.0f : fresh ? most - 15.0f : fmaxf(most - 15.0f, 0.0f);
                    const float keep = fresh ? 0.0f : __builtin_amdgcn_exp2f(-over);
                    m = fresh && most == -__builtin_inff() ? m : zero + over;
                    accl *= keep;
#pragma unroll
                    for (int d = 0; d < ND; ++d) acc[d] *= keep;
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] -= over;
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    h8 p;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const f32x2 w = {__builtin_amdgcn_exp2f(s[8 * y + e]), __builtin_amdgcn_exp2f(s[8 * y + e + 1])};
                        const h2 w2 = __builtin_convertvector(w, h2);
                        p[e] = w2[0], p[e + 1] = w2[1];
                    }
                    accl = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, now.vl[y][lane]), p, accl, 0, 0, 0);
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, now.v[d][y][lane]), p, acc[d], 0, 0, 0);
                }
                // (each half's operands are read under its exponentials: 592 -> 582 us)
                __builtin_amdgcn_sched_group_barrier(0x100, ND + 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x402, 12, 1);
                __builtin_amdgcn_sched_group_barrier(0x8, ND + 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x100, ND + 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x402, 12, 1);
                __builtin_amdgcn_sched_group_barrier(0x8, ND + 1, 1);
            };
            scores(0);
            next(0);
            scores(1);
            weigh(0);
            next(1);
            weigh(1);
            __syncthreads();
        }
    }
    if (nan) {
        // NaN values: the rows that see one are NaN in its group.
        int hit[NG] = {};
        for (int i = c0; i < c1; ++i) {
            const int key0 = span.at(i) * KA_CHUNK;
            const uint8_t* at = chunk_at(i, page_of(i));
            for (int e = 0; e < 16; ++e) {
                const int j = 16 * half + e, key = key0 + j;
                if (key <= pos && (key < sink || key > pos - ring))
#pragma unroll
                    for (int g = 0; g < NG; ++g) hit[g] |= (kv4_half(at, L::v_step(j, g)) & 0x7fffu) > 0x7c00u;
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            hit[g] |= __shfl_xor(hit[g], 32, 64);
            const float add = hit[g] ? __builtin_nanf("") : 0.0f;
#pragma unroll
            for (int d = g * (G / 32); d < (g + 1) * (G / 32); ++d) acc[d] += add;
        }
    }

    // Row `m32` of the lows' product is in reg m % 4 + 4 (m / 8) of half m / 4 % 2.
    const float l = __shfl(accl[4], m32, 64);  // m = 8
    if (l != l) m = l;
    const float unit = pow2i(vunit);
    if (r0 + wave * 32 + m32 > r1) return;
    const int64_t row = row0 + token, head = kvh * per + r - token * per;
    const bool last = plan.splits == 1;
    const float scale = last ? 1.0f / l : 0x1p-15f;
    T* out = reinterpret_cast<T*>(a.out) + row * a.ldo + head * c.dv;
    const int64_t at = ((int64_t)split * c.rows + row) * a.heads + head;
    float* ml = reinterpret_cast<float*>(a.ws);
    float* po = ml + 2 * ((int64_t)plan.splits * c.rows * a.heads) + at * c.dv;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        constexpr int GD = G / 32;
        const float low = __shfl(accl[d / GD], m32, 64);  // (NG <= 4: m = d / GD is in the lower half)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int dim = 32 * d + 8 * (e >> 2) + 4 * half;
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = (acc[d][e + k] * (k & 1 ? unit * 0.0625f : unit) + low) * scale;
            if (last) {
                typedef T Vec4 __attribute__((ext_vector_type(4)));
                if (plan.out_aligned && dim + 4 <= c.dv) {
                    Vec4 z;
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[k] = (T)y[k];
                    *reinterpret_cast<Vec4*>(out + dim) = z;
                } else
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (dim + k < c.dv) out[dim + k] = (T)y[k];
            } else
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (dim + k < c.dv) po[dim + k] = y[k];
        }
    }
    if (half == 0) {
        if (last) {
            if (a.lse) a.lse[row * a.heads + head] = (m + __builtin_amdgcn_logf(l * 0x1p-15f)) * 0.69314718055994530942f;
        } else
            ml[2 * at] = l == l ? m : l, ml[2 * at + 1] = l * 0x1p-15f;
    }
}

// The key ranges' partial results of one (row, head), joined by a workgroup: the
// ranges' factors first, then a wavefront every fourth range, eight loads at a
// time (one wavefront in turn over the 256 ranges of a long sequence took 170 us).
constexpr int KA_SPLITS = 512;
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4View c, Kv4AttendArgs a, int splits) {
    typedef typename Kv4Elem<TYPE>::T T;
    __shared__ float f[KA_SPLITS], sv[4][256], st[4], ss[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t n = (int64_t)c.rows * a.heads, at = blockIdx.x;
    const float* ml = reinterpret_cast<const float*>(a.ws);
    const float* po = ml + 2 * n * splits + at * c.dv;
    float top = -__builtin_inff();
    for (int s = tid; s < splits; s += 256) {
        f[s] = ml[2 * (s * n + at)];
        top = fmaxf(top, f[s]);
    }
#pragma unroll
    for (int h = 1; h < 64; h <<= 1) top = fmaxf(top, lane_xor(top, h, lane));
    if (lane == 0) st[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]));
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
    for (int s = tid; s < splits; s += 256) {
        // -1: a range without keys, which wrote no sums.  NaN: scores were, and the row's results are.
        const float g = f[s] == -__builtin_inff() ? -1.0f : __builtin_amdgcn_exp2f(f[s] - zero);
        f[s] = g;
        sum += g < 0.0f ? 0.0f : ml[2 * (s * n + at) + 1] * g;
    }
#pragma unroll
    for (int h = 1; h < 64; h <<= 1) sum += lane_xor(sum, h, lane);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    for (int x = 0; x * 64 < c.dv; ++x) {
        const int d = x * 64 + lane;
        float v = 0.0f;
        for (int s0 = wave; s0 < splits; s0 += 32) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = s0 + 4 * k < splits && d < c.dv ? po[(s0 + 4 * k) * n * c.dv + d] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float g = s0 + 4 * k < splits ? f[s0 + 4 * k] : -1.0f;
                v = g < 0.0f ? v : __builtin_fmaf(y[k], g, v);
            }
        }
        sv[wave][d & 255] = v;
    }
    __syncthreads();
    if (tid < c.dv) {
        T* out = reinterpret_cast<T*>(a.out) + at / a.heads * a.ldo + at % a.heads * c.dv;
        Kv4Elem<TYPE>::put(out + tid, ((sv[0][tid] + sv[1][tid]) + (sv[2][tid] + sv[3][tid])) / sum);
    }
    if (a.lse && tid == 0) a.lse[at] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

// The same for few ranges, a thread an element of the output: many rows are many
// elements, and a workgroup a (row, head) would mostly wait for its barriers (32,768
// of two ranges).
constexpr int KA_FEW = 8;
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv4_join_few(Kv4View c, Kv4AttendArgs a, int splits) {
    typedef typename Kv4Elem<TYPE>::T T;
    const int64_t n = (int64_t)c.rows * a.heads, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * c.dv) return;
    const int64_t at = i / c.dv;
    const int d = (int)(i - at * c.dv);
    const float* ml = reinterpret_cast<const float*>(a.ws);
    const float* po = ml + 2 * n * splits + i;
    float m[KA_FEW], l[KA_FEW], v[KA_FEW], top = -__builtin_inff();
#pragma unroll
    for (int s = 0; s < KA_FEW; ++s) {
        const int64_t x = s < splits ? s : 0;
        m[s] = s < splits ? ml[2 * (x * n + at)] : -__builtin_inff();
        l[s] = ml[2 * (x * n + at) + 1];
        v[s] = po[x * n * c.dv];
        top = fmaxf(top, m[s]);
    }
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int s = 0; s < KA_FEW; ++s) {
        const float g = __builtin_amdgcn_exp2f(m[s] - zero);
        const bool some = m[s] != -__builtin_inff();  // (a range without keys wrote no sums)
        sum = some ? __builtin_fmaf(l[s], g, sum) : sum;
        o = some ? __builtin_fmaf(v[s], g, o) : o;
    }
    Kv4Elem<TYPE>::put(reinterpret_cast<T*>(a.out) + at / a.heads * a.ldo + at % a.heads * c.dv + d, o / sum);
    if (a.lse && d == 0) a.lse[at] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

// The shape of a call: which kernel, its rows a tile and wavefronts, key ranges.
struct KaShape {
    bool prompt;
    int rows, waves, tiles_each, splits;
    int64_t tiles;
};

static void tiles_of(const Kv4View& c, const int* row0, int per, int rows, KaShape& s) {
    s.rows = rows;
    s.tiles_each = 0;
    s.tiles = 0;
    if (c.each) {
        s.tiles_each = (int)(((int64_t)c.each * per + rows - 1) / rows);
        s.tiles = (int64_t)s.tiles_each * c.nb;
    } else
        for (int b = 0; b < c.nb; ++b) s.tiles += ((int64_t)(row0[b + 1] - row0[b]) * per + rows - 1) / rows;
}

// Which kernel is the quicker depends on the rows, the keys and how both fill the
// chip, so both are estimated, in us, from what was measured of each at 128 (64)
// dims of bf16:
//  rows   4 in all and 4 a round of 512 workgroups of four wavefronts (256 of
//         eight), 1.74 (1.8) a step of a wavefront: 32 keys of 16 (32) rows
//  prompt 18 in all (the references, the first images), 1.3 (1.0) for 32 keys of
//         256 rows, a workgroup a CU
//  join   4, and the partial results' bytes there and back at 2 TB/s
// One sequence of 4,000 keys and 32 heads over 8, 128 dims, rows / prompt: 128 rows
// 33 / 63, 256 60 / 71, 512 112 / 98, 1,024 224 / 162, 2,048 480 / 265; 16 sequences'
// 32 rows 110 / 109, 64 rows 204 / 139; 500 keys' 1,024 rows 80 / 80, 2,048 190 / 124.
static double ka_join_us(const Kv4View& c, int heads, int64_t splits) {
    return splits > 1 ? 4.0 + (double)c.rows * heads * (double)splits * (c.dv + 2) * 8 / 2e6 : 0.0;
}

static KaShape shape_of(const Kv4View& c, const int* row0, int type, int heads, int sink, int ring, int longest) {
    const int per = heads / c.heads;
    const int64_t tokens = c.nb ? (c.rows + c.nb - 1) / c.nb : 0, mean = c.nb ? (int64_t)c.rows * per / c.nb : 0;
    // The chunks that a tile of `rows` rows sees: the last tile's, and a middle one's.
    auto chunks_of = [&](int rows, bool middle) -> int64_t {
        const int64_t keys = longest - (middle ? tokens / 2 : 0), wide = std::min<int64_t>(tokens, rows / per + 1);
        return ((ring ? std::min<int64_t>(keys, (int64_t)sink + ring + wide + 2 * KA_CHUNK) : keys) + KA_CHUNK - 1) / KA_CHUNK;
    };
    KaShape s;
    s.prompt = false;
    // Two tiles of rows a wavefront where their sums fit the registers beside the
    // loads, and there are tiles for every CU's eight wavefronts without it (2 kv
    // heads, 4000 keys: 96 tiles of 16 17.6 us, half as many of 32 21.3; 384 36.4 and
    // 47.3; 1024 about the same).
    tiles_of(c, row0, per, 16, s);
    if (c.width == 64 && mean > 16 && s.tiles * c.heads > 512) tiles_of(c, row0, per, 32, s);
    const int64_t base = s.tiles * c.heads;
    s.waves = s.rows == 16 && c.width <= 128 && base <= 256 ? 8 : 4;
    // The workgroups that run at once: eight wavefronts a CU, as many as their
    // registers let run (four at 256 dims).  Eight of one workgroup meet in LDS and
    // not in the workspace, so half as many ranges are joined: 1060 keys of 256 tiles
    // 15.4 us for 27.9, 131,072 keys of 8 38.7 for 41.5 (weights of one part).  With more than 256 tiles
    // every CU has its eight without it.
    const int64_t slots = s.waves == 8 || c.width == 256 ? 256 : 512;
    const int64_t chunks = chunks_of(s.rows, false);
    // Ranges as the slots allow: a second round for some costs more than slots that
    // stay empty (240 tiles of 1000 keys, 8 wavefronts: 14.9 us, in two ranges each
    // 22.7; 400 of 4000 keys, 4 wavefronts: 56 and 64; 192 of 256 dims 62 and 84), but
    // for long keys where hardly half of them are taken (304 tiles of 4000 keys: 57 and
    // 54, of 64 dims 39 and 33; of 1000 keys 22 and 26).  A wavefront of eight has two
    // steps at least (8 tiles of 4000 keys 12.4 us, with four 16.7; 16000 keys 14.3 and
    // 17.1), of four, whose join is larger beside its work, four.
    int64_t want = base ? std::max<int64_t>(1, slots / base) : 1;
    if (slots == 512 && want == 1 && base * 8 < slots * 5 && chunks >= 64) want = 2;  // (two workgroups share a CU)
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, KA_SPLITS), chunks / ((s.waves == 8 ? 2 : 4) * s.waves)));

    // f32 calls keep 22 bits of a weight, which the prompt kernel does not; at
    // 256 dims its sums do not fit the registers.
    if (type == KV4_F32 || c.width > 128 || c.kernel == 1 || base == 0) return s;
    const int64_t steps = (chunks_of(s.rows, true) + s.splits * s.waves - 1) / (s.splits * s.waves);
    const double step = s.rows == 32 ? 1.8 : c.width == 64 ? 0.9 : 1.74;
    const double plain = 4.0 + std::max(1.0, (double)(base * s.splits) / (double)slots) * (4.0 + (double)steps * step) +
                         ka_join_us(c, heads, s.splits);
    KaShape p;
    p.prompt = true;
    p.waves = KP_WAVES;
    tiles_of(c, row0, per, KP_ROWS, p);
    const int64_t most = chunks_of(KP_ROWS, false), middle = chunks_of(KP_ROWS, true);
    const double each = c.width == 64 ? 1.0 : 1.3;
    double best = 0.0;
    for (int64_t n = 1; n <= KA_FEW * 4 && (n == 1 || most / n >= 16); ++n) {
        const int64_t rounds = (p.tiles * c.heads * n + 255) / 256;
        const double us = 18.0 + (double)rounds * (double)(((rounds == 1 ? most : middle) + n - 1) / n) * each + ka_join_us(c, heads, n);
        if (n == 1 || us < best) best = us, p.splits = (int)n;
    }
    return best < plain || c.kernel == 2 ? p : s;
}

size_t kv4_attend_ws(const Kv4View& c, const int* row0, int heads, int sink, int ring, int longest) {
    // (enough for a call of any type)
    const int s = std::max(shape_of(c, row0, KV4_F32, heads, sink, ring, longest).splits,
                           shape_of(c, row0, KV4_F16, heads, sink, ring, longest).splits);
    return s > 1 ? (size_t)s * c.rows * heads * (c.dv + 2) * 4 : 0;
}

template <int TYPE, int W, int G>
static hipError_t attend_shaped(const Kv4View& c, const int* row0, const Kv4AttendArgs& a, int longest, hipStream_t s) {
    const KaShape shape = shape_of(c, row0, TYPE, a.heads, a.sink, a.ring, longest);
    const size_t es = sizeof(typename Kv4Elem<TYPE>::T);
    KaPlan plan;
    plan.tiles_each = shape.tiles_each;
    plan.splits = shape.splits;
    plan.aligned = c.dk % 8 == 0 && (uintptr_t)a.q % 16 == 0 && a.ldq * es % 16 == 0 && c.dk * es % 16 == 0;
    plan.out_aligned = c.dv % 4 == 0 && (uintptr_t)a.out % 16 == 0 && a.ldo * es % 16 == 0;
    if (shape.tiles * c.heads > 0x7fffffff || (int64_t)c.rows * a.heads > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(shape.tiles * c.heads), plan.splits);
    bool done = false;
    if constexpr (W <= 128 && TYPE != KV4_F32)
        if (shape.prompt) {
            hipLaunchKernelGGL((k_kv4_prompt<TYPE, W, G>), grid, dim3(KP_WAVES * 64), 0, s, c, a, plan);
            done = true;
        }
    if (!done) {
        auto kern = k_kv4_attend<TYPE, W, G, 1, 4>;
        if constexpr (W <= 128)
            if (shape.waves == 8) kern = k_kv4_attend<TYPE, W, G, 1, 8>;
        if constexpr (W == 64)
            if (shape.rows == 32) kern = k_kv4_attend<TYPE, W, G, 2, 4>;
        hipLaunchKernelGGL(kern, grid, dim3(shape.waves * 64), 0, s, c, a, plan);
    }
    if (plan.splits > KA_FEW)
        hipLaunchKernelGGL(k_kv4_join<TYPE>, dim3((unsigned)(c.rows * a.heads)), dim3(256), 0, s, c, a, plan.splits);
    else if (plan.splits > 1)
        hipLaunchKernelGGL(k_kv4_join_few<TYPE>, dim3((unsigned)(((int64_t)c.rows * a.heads * c.dv + 255) / 256)), dim3(256), 0, s, c, a,
                           plan.splits);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t attend_typed(const Kv4View& c, const int* row0, const Kv4AttendArgs& a, int longest, hipStream_t s) {
    if (c.group == 32)
        return c.width == 64    ? attend_shaped<TYPE, 64, 32>(c, row0, a, longest, s)
               : c.width == 128 ? attend_shaped<TYPE, 128, 32>(c, row0, a, longest, s)
                                : attend_shaped<TYPE, 256, 32>(c, row0, a, longest, s);
    return c.width == 64    ? attend_shaped<TYPE, 64, 64>(c, row0, a, longest, s)
           : c.width == 128 ? attend_shaped<TYPE, 128, 64>(c, row0, a, longest, s)
                            : attend_shaped<TYPE, 256, 64>(c, row0, a, longest, s);
}

hipError_t launch_kv4_attend(const Kv4View& c, const int* row0, const Kv4AttendArgs& a, int longest, hipStream_t s) {
    return a.type == KV4_F32   ? attend_typed<KV4_F32>(c, row0, a, longest, s)
           : a.type == KV4_F16 ? attend_typed<KV4_F16>(c, row0, a, longest, s)
                               : attend_typed<KV4_BF16>(c, row0, a, longest, s);
}

}  // namespace nh
