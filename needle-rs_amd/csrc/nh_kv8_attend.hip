// Attention of a batch's rows over the 8-bit cache (the layout: nh_kv8.h).
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= i of row i's
//   sequence; with a ring also j < sink or j > i - ring; of a batch that asks all
//   keys of its sequence.
//
// A key is step x code with one step for 16 positions, so a score is scale step
// (q . c): the codes themselves are the matrix operands, and the step is one
// factor of 16 x 16 scores.  In the same way a weight takes its value's step, and
// the second product's operands are codes too.  A byte c + 128 under 0x64 is the
// f16 number 1152 + c (one byte permutation for two), from which one packed
// addition takes 1152: exact.  That is done to the values; a key's byte alone is the
// f16 subnormal (128 + c) 2^-24, and the products' sums start at -128 2^-24 times the
// query's own sum: 30.0 us became 28.6 in the last example below.  (Sums of weights and
// values would lose to the offset what their signs cancel.)  f32 queries go the other
// way: their rows as whole numbers of 23 bits in three signed digits of 8, times the
// codes in the i8 MFMAs, which are exact and take the bytes as they are.
// The products are transposed, keys (or dims) by rows: S^T = K Q^T leaves lane (o,
// kg) the scores of its row o with keys 16 t + 4 kg + 0..3, and a lane's 16 bytes
// of values are of those very keys, so a weight never leaves its lane, and a
// row's maximum, sum and correction are one lane's scalars.
//
// One row a head is bound by the cache's bytes: 64 sequences of up to 8,192 keys, 32
// heads over 8 of 128, bf16 (818 MB) 155 us, 5.2 TB/s, as a large copy; one of 131,072
// keys (269 MB) 50 to 60 with the 4.5 of its join.  The 64 at other dims and in f32: 192 +
// 128 dims 184 (f32 191), 256 + 256 290 (303), 128 + 128 f32 154, 5.3 to 5.6 TB/s.  Few keys are bound by latency (374 of
// them 6.5 us on the GPU), so the first chunk's loads start before the queries are
// operands.  More rows are bound by vector instructions, some 250 for 64 keys of 16
// rows at 64 dims, 96 of them for codes turned into f16: four sequences' 448 rows over
// 1,500 keys, 16 heads of 64, 28.6 us with the vector units three quarters busy.  512 rows
// after 4,000 keys, 32 heads over 8 (the only kernel for f32, and for more than 128 dims, at
// one wavefront a SIMD): 128 dims f32 89, 192 + 128 bf16 118 (f32 145), 256 + 256 177 (232).
#include <algorithm>

#include "nh_kv8_device.h"

namespace nh {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// What a lane loads of a chunk.
template <int WK, int WV>
struct Ka8Chunk {
    u32x4 k[4][WK / 64], v[WV / 16];
    f32x4 ks, vs;
    u32x4 bad;  // 4 u16 of the keys, 4 of the values
};

// NW wavefronts a workgroup, each every NW-th chunk of the range.
template <int TYPE, int WK, int WV, int NW>
__global__ __launch_bounds__(NW * 64, WK <= 128 ? 2 : 1) void k_kv8_attend(Kv8View c, Kv8AttendArgs a, KaPlan plan) {
    typedef typename KvElem<TYPE>::T T;
    typedef Kv8Lay<WK, WV> L;
    typedef Ka8Chunk<WK, WV> Chunk;
    constexpr int NJ = L::NJ, NV = L::NV;
    constexpr bool DIGITS = TYPE == KV_F32;
    // f16 parts of a weight: f32 and f16 calls carry what the first rounds off.
    constexpr int WPARTS = TYPE == KV_BF16 ? 1 : 2;
    constexpr int LD = WV + 4;
    __shared__ float so[NW][16][LD];
    __shared__ float sm[NW][16], sl[NW][16];

    const int tid = threadIdx.x, lane = tid & 63, o = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % c.heads, per = a.heads / c.heads, split = blockIdx.y;

    // The sequence and the rows of this tile.
    int tile = blockIdx.x / c.heads, b;
    if (plan.tiles_each) {
        b = tile / plan.tiles_each;
        tile -= b * plan.tiles_each;
    } else {
        b = kv_find(c, tile, lane, [&](const KvEntry& e) { return ((e.row1 - e.row0) * per + 15) / 16; });
    }
    // (the entry and the shape in one wait, no branch between them)
    const KvEntry entry = kv_batch(c, min(b, c.nb - 1));
    const bool current = kv_current(c);
    const int row0 = entry.row0, nrows = entry.row1 - row0, seq = entry.seq;
    const int first = entry.len - (c.ask ? 1 : nrows), r0 = tile * 16;
    if ((b >= c.nb) | !current | (!c.ask & (first < 0)) | (r0 >= nrows * per) | (entry.row1 > c.rows)) return;
    const int r1 = min(r0 + 16, nrows * per) - 1;
    const int plo = first + (c.ask ? 0 : r0 / per), phi = first + (c.ask ? 0 : r1 / per);

    const Ka8Span span(plo, phi, a.sink, a.ring);
    const int sink = a.ring ? a.sink : 0x7fffffff, ring = a.ring;
    const int per_split = max((span.count() + plan.splits - 1) / plan.splits, NW);
    const int c0 = split * per_split, c1 = min(c0 + per_split, span.count());
    const int* table = c.table + (size_t)seq * c.table_ld;
    auto page_of = [&](int i) { return i < c1 ? table[span.at(i) * KV8_CHUNK >> c.page_log2] : 0; };
    int chunk = c0 + wave, p0 = page_of(chunk), p1 = page_of(chunk + NW);

    // The queries: f16 operands scaled by a power of two to just under 2^15, or digits.
    h8 q[NJ][2];
    i32x4 qd[3][NJ];
    float cq, offset = 0.0f;
    const int r = min(r0 + o, r1), token = r / per, pos = first + (c.ask ? 0 : token);
    const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + token) * a.ldq + (int64_t)(kvh * per + r - token * per) * c.dk;
    T raw[NJ][16];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int d = j * 64 + kg * 16 + g * 8;
            if (plan.aligned) {
                typedef T Vec __attribute__((ext_vector_type(8)));
                Vec y = {};
                if (d < c.dk) y = *reinterpret_cast<const Vec*>(src + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) raw[j][8 * g + e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) raw[j][8 * g + e] = d + e < c.dk ? src[d + e] : (T)0.0f;
            }
        }

    // (the first chunk is on its way while the queries are turned into operands)
    auto load = [&](Chunk& to, int i, int pg) {
        if (i >= c1) return;
        const int slot = span.at(i) * KV8_CHUNK & (c.page() - 1);
        // (a page id comes from the cache's own table; a bad one is not followed)
        const uint8_t* p = kv8_block(c, (unsigned)pg < (unsigned)c.pages ? pg : 0, a.layer, kvh) + (uint32_t)(slot >> 6) * L::CHUNK;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) to.k[t][j] = *reinterpret_cast<const u32x4*>(p + L::k_piece(t, j, lane));
        to.ks = *reinterpret_cast<const f32x4*>(p + L::RECORD);
        to.vs = *reinterpret_cast<const f32x4*>(p + L::RECORD + 16);
        to.bad = *reinterpret_cast<const u32x4*>(p + L::RECORD + 32);
#pragma unroll
        for (int n = 0; n < NV; ++n) to.v[n] = *reinterpret_cast<const u32x4*>(p + L::v_piece(n, lane));
    };
    Chunk two[2];
    load(two[0], chunk, p0);

    float x[NJ][16], most = 0.0f;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[j][e] = (float)raw[j][e];
            most = fmaxf(most, fabsf(x[j][e]));
            nan |= x[j][e] != x[j][e];
        }
    if constexpr (DIGITS) {
        most = nan ? __builtin_inff() : most;
        most = groups_max(most);
        // |x| <= most, as a whole number of at most 127 (2^16 + 2^8 + 1)
        const float full = 8355711.0f;
        const bool fine = most < __builtin_inff(), some = most > 0x1p-100f;
        const float up = fine && some ? full / most : 0.0f;
        // z = 2^-8 of the sum of whole numbers x codes
        cq = fine ? (a.scale * KA_LOG2E) * (some ? most * (256.0f / full) : 0.0f) : __builtin_nanf("");
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t d0 = 0, d1 = 0, d2 = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = (int)rintf(__builtin_amdgcn_fmed3f(x[j][4 * w + e] * up, -full, full));
                    const int lo = (int8_t)n, n1 = (n - lo) >> 8, mid = (int8_t)n1, hi = (n1 - mid) >> 8;
                    d0 |= (uint32_t)(uint8_t)hi << (8 * e);
                    d1 |= (uint32_t)(uint8_t)mid << (8 * e);
                    d2 |= (uint32_t)(uint8_t)lo << (8 * e);
                }
                qd[0][j][w] = (int)d0;
                qd[1][j][w] = (int)d1;
                qd[2][j][w] = (int)d2;
            }
    } else {
        most = groups_max(most);
        const int ef = max((int)(__builtin_bit_cast(uint32_t, most) >> 23 & 255u), 15);
        const float up = __builtin_bit_cast(float, (uint32_t)(268 - ef) << 23);
        cq = (a.scale * KA_LOG2E) * __builtin_bit_cast(float, (uint32_t)(ef - 14) << 23);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) q[j][e / 8][e % 8] = (_Float16)(x[j][e] * up);
        // what the keys' 128 too many make of a row's scores
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) offset += (float)q[j][e / 8][e % 8];
        offset = groups_sum(offset) * -0x1p-17f;
    }

    f32x4 acc[NV];
    float m, l;
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = f32x4{0, 0, 0, 0};
    // The weights are kept as 2^15 p, and with their steps as the f16 operand 2^15 p
    // step / 2^eref, 2^eref above every step seen so far: at most 2^15, and exact to
    // 11 bits down to 2^-29 of it.
    int eref = -126;

    auto compute = [&](const Chunk& x, int i) {
        const int key0 = span.at(i) * KV8_CHUNK;
        const bool whole = key0 + KV8_CHUNK - 1 <= plo && (key0 + KV8_CHUNK - 1 < sink || key0 > phi - ring);
        const uint32_t bad0 = __builtin_amdgcn_readfirstlane((int)(x.bad[0] | x.bad[2]));
        const uint32_t bad1 = __builtin_amdgcn_readfirstlane((int)(x.bad[1] | x.bad[3]));
        const bool plain = whole && !(bad0 | bad1);
        // The steps' reference: raised when a step passes it (of a block that the tile sees;
        // others' steps, past the rows or under no window, count as 0).
        f32x4 vs = x.vs;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 4; ++t) vs[t] = ka8_sees(key0 + 16 * t, plo, phi, sink, ring) ? vs[t] : 0.0f;
        }
        const float top = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
        const int et = __builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, top) >> 23)) - 126;
        if (et > eref) {
            const float down = pow2i(max(eref - et, -126));
            eref = et;
#pragma unroll
            for (int k = 0; k < NV; ++k) acc[k] *= down;
        }
        const float wscale = pow2i(-eref);
        float vstep[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) vstep[t] = vs[t] * wscale;
        f32x4 z[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (DIGITS) {
                i32x4 n[3] = {};
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const i32x4 k = __builtin_bit_cast(i32x4, x.k[t][j] ^ 0x80808080u);
#pragma unroll
                    for (int d = 0; d < 3; ++d) n[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, qd[d][j], n[d], 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    z[t][r] = __builtin_fmaf((float)n[2][r], 0x1p-8f, (float)(n[0][r] * 256 + n[1][r]));
            } else {
                z[t] = f32x4{offset, offset, offset, offset};
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const h8 k = bytes8(x.k[t][j][2 * g], x.k[t][j][2 * g + 1]);
                        z[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[j][g], z[t], 0, 0, 0);
                    }
            }
        }
        h8 pw[2][WPARTS];
        const bool fresh = m == -__builtin_inff();  // no key seen yet
        const float base = fresh ? 0.0f : m;
        float s[4][4];  // 15 + log2 of the weight against the maximum so far
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float f = DIGITS ? cq * x.ks[t] : cq * x.ks[t] * 0x1p24f;
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][r] = __builtin_fmaf(z[t][r], f, 15.0f - base);
        }
        if (!plain) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t bad = (t & 2 ? bad1 : bad0) >> (16 * (t & 1)) >> (4 * kg);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = key0 + 16 * t + 4 * kg + r;
                    const bool seen = (j <= pos) & ((j < sink) | (j > pos - ring));
                    s[t][r] = !seen ? -__builtin_inff() : bad >> r & 1 ? __builtin_nanf("") : s[t][r];
                }
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int k = 1; k < 16; ++k) most = fmaxf(most, s[k / 4][k % 4]);
        most = groups_max(most);
        if (__any(most > 15.0f || fresh)) {
            // A new maximum (the first: whatever it is).
            const float over = most == -__builtin_inff() ? 0.0f : fresh ? most - 15.0f : fmaxf(most - 15.0f, 0.0f);
            const float keep = fresh ? 0.0f : __builtin_amdgcn_exp2f(-over);
            m = fresh && most == -__builtin_inff() ? m : base + over;
            l *= keep;
#pragma unroll
            for (int k = 0; k < NV; ++k) acc[k] *= keep;
#pragma unroll
            for (int k = 0; k < 16; ++k) s[k / 4][k % 4] -= over;
        }
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            const f32x2 p = {__builtin_amdgcn_exp2f(s[k / 4][k % 4]), __builtin_amdgcn_exp2f(s[k / 4][k % 4 + 1])};
            l += p[0];
            l += p[1];
            const f32x2 w = {p[0] * vstep[k / 4], p[1] * vstep[k / 4]};
            const h2 hi = __builtin_convertvector(w, h2);
            pw[k / 8][0][k % 8] = hi[0], pw[k / 8][0][k % 8 + 1] = hi[1];
            if constexpr (WPARTS == 2) {
                const f32x2 rest = {w[0] - (float)hi[0], w[1] - (float)hi[1]};
                const h2 lo = __builtin_convertvector(rest, h2);
                pw[k / 8][1][k % 8] = lo[0], pw[k / 8][1][k % 8 + 1] = lo[1];
            }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const h8 v = codes8(x.v[n][2 * h], x.v[n][2 * h + 1]);
#pragma unroll
                for (int p = 0; p < WPARTS; ++p)
                    acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pw[h][p], acc[n], 0, 0, 0);
            }
    };

    // The loads of the next chunk are in flight during this one's arithmetic, the
    // page id of the one after it is on its way.
    while (chunk < c1) {
#pragma unroll
        for (int k = 0; k < 2; ++k, chunk += NW) {
            if (chunk >= c1) break;
            load(two[k ^ 1], chunk + NW, p1);
            p1 = page_of(chunk + 2 * NW);
            compute(two[k], chunk);
        }
    }

    // The wavefronts' sums joined.
    const float unit = pow2i(eref);
    l = groups_sum(l);
    if (l != l) m = l;  // NaN scores: the row's, whatever other ranges hold
    if (kg == 0) sm[wave][o] = m, sl[wave][o] = l * 0x1p-15f;
    __syncthreads();
    float high = sm[0][o];
#pragma unroll
    for (int w = 1; w < NW; ++w) high = fmaxf(high, sm[w][o]);
    const float base = high == -__builtin_inff() ? 0.0f : high;
    const float f = __builtin_amdgcn_exp2f(m - base) * 0x1p-15f;
#pragma unroll
    for (int n = 0; n < NV; ++n) *reinterpret_cast<f32x4*>(&so[wave][o][16 * n + 4 * kg]) = acc[n] * f * unit;
    __syncthreads();
    // (four dims of a row a thread)
    for (int at = tid; at < 4 * WV; at += NW * 64) {
        const int rr = at / (WV / 4), d = 4 * (at % (WV / 4));
        if (r0 + rr > r1 || d >= c.dv) continue;
        float top = sm[0][rr];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, sm[w][rr]);
        const float zero = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f;
        f32x4 v = {};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            sum = __builtin_fmaf(sl[w][rr], __builtin_amdgcn_exp2f(sm[w][rr] - zero), sum);
            v += *reinterpret_cast<const f32x4*>(&so[w][rr][d]);
        }
        const int t = (r0 + rr) / per, head = kvh * per + r0 + rr - t * per;
        const int64_t row = row0 + t;
        if (plan.splits == 1) {
            T* out = reinterpret_cast<T*>(a.out) + row * a.ldo + (int64_t)head * c.dv + d;
            v *= sum == 0.0f ? 0.0f : 1.0f / sum;  // (no key seen: 0)
            if (plan.out_aligned) {
                typedef T Vec4 __attribute__((ext_vector_type(4)));
                *reinterpret_cast<Vec4*>(out) = __builtin_convertvector(v, Vec4);
            } else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < c.dv) out[e] = (T)v[e];
            if (a.lse && d == 0) a.lse[row * a.heads + head] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
        } else {
            const int64_t part = ((int64_t)split * c.rows + row) * a.heads + head;
            float* ml = reinterpret_cast<float*>(a.ws);
            float* out = ml + 2 * ((int64_t)plan.splits * c.rows * a.heads) + part * c.dv + d;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < c.dv) out[e] = v[e];
            if (d == 0) ml[2 * part] = sum == sum ? top : sum, ml[2 * part + 1] = sum;
        }
    }
}

// The shape of a call: which kernel, its rows a tile and wavefronts, key ranges.
struct Ka8Shape {
    bool prompt;
    int rows, waves, tiles_each, splits;
    int64_t tiles;
};

static void tiles_of(const Kv8View& c, const int* row0, int per, int rows, Ka8Shape& s) {
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
//  rows   4 in all and 5 (3) a round of 512 workgroups of four wavefronts, 2.2 (1.4) a
//         step of a wavefront: 64 keys of 16 rows
//  prompt 4 in all and 8 (6) a round of a workgroup a CU, 2.0 (1.75) for 64 keys of
//         256 rows
//  join   4, and the partial results' bytes there and back at 2 TB/s
// 32 heads over 8 of 128 dims, rows / prompt: a sequence of 4,000 keys 512 rows 75 / 74,
// 1,024 130 / 110, 2,048 220 / 135; four of 1,500 keys 128 rows 37 / 62, 256 67 / 56; 16
// of 2,000 keys 32 rows 46 / 63, 64 rows 85 / 71.  16 heads of 64: 16 sequences of 2,000
// keys 128 rows 53 / 58, 256 92 / 64; four of 1,500 512 rows 39 / 49, 1,024 62 / 51.
// (Both kernels were swept at these two head shapes, causal and of even batches alone, before
// the first one's keys became subnormals, which took 2 to 4 percent off it.)
static double ka_join_us(const Kv8View& c, int heads, int64_t splits) {
    return splits > 1 ? 4.0 + (double)c.rows * heads * (double)splits * (c.dv + 2) * 8 / 2e6 : 0.0;
}

static Ka8Shape shape_of(const Kv8View& c, const int* row0, int type, int heads, int sink, int ring, int longest) {
    const int per = heads / c.heads;
    const int64_t tokens = c.nb ? (c.rows + c.nb - 1) / c.nb : 0;
    // The chunks that a tile of `rows` rows sees: the last tile's, and a middle one's.
    auto chunks_of = [&](int rows, bool middle) -> int64_t {
        const int64_t keys = longest - (middle && !c.ask ? tokens / 2 : 0), wide = c.ask ? 1 : std::min<int64_t>(tokens, rows / per + 1);
        return ((ring ? std::min<int64_t>(keys, (int64_t)sink + ring + wide + 2 * KV8_CHUNK) : keys) + KV8_CHUNK - 1) / KV8_CHUNK;
    };
    Ka8Shape s;
    s.prompt = false;
    tiles_of(c, row0, per, 16, s);
    const int64_t base = s.tiles * c.heads;
    // Eight wavefronts where the tiles leave CUs idle (one of 4,000 keys of 8 tiles: 23 us
    // for 27): they meet in LDS and not in the workspace.
    s.waves = c.wk <= 128 && base <= 256 ? 8 : 4;
    // Ranges of keys until every CU has its eight wavefronts (four at more than 128 dims,
    // by their registers), a chunk each at least; two ranges are not worth the join (8
    // tiles of 1,000 keys 10.7 us, in two 12.1; 4,000 keys in seven 12.1 for 23, 16,000 in
    // 31 14.5 for 71).
    const int64_t slots = s.waves == 8 || c.wk > 128 ? 256 : 512;
    const int64_t chunks = chunks_of(s.rows, false);
    const int64_t most = std::min<int64_t>(std::min<int64_t>(base ? std::max<int64_t>(1, slots / base) : 1, KV_SPLITS), chunks / s.waves);
    s.splits = most < 2 || (chunks < 4 * s.waves && most < 3) ? 1 : (int)most;

    // f32 calls keep 22 bits of a weight, which the prompt kernel does not; at more than
    // 128 dims its sums do not fit the registers, and it counts a page's bytes in 32 bits.
    if (type == KV_F32 || c.wk > 128 || c.kernel == 1 || base == 0) return s;
    if ((uint64_t)c.block() * c.heads * c.layers >> 32) return s;
    const bool wide = c.wk == 128;
    const double steps = (double)((chunks_of(s.rows, true) + s.splits * s.waves - 1) / (s.splits * s.waves));
    const double plain = 4.0 + std::max(1.0, (double)(base * s.splits) / (double)slots) * (wide ? 5.0 + 2.2 * steps : 3.0 + 1.4 * steps) +
                         ka_join_us(c, heads, s.splits);
    Ka8Shape p;
    p.prompt = true;
    p.waves = 0;
    tiles_of(c, row0, per, KP8_ROWS, p);
    const int64_t last = chunks_of(KP8_ROWS, false), middle = chunks_of(KP8_ROWS, true);
    double best = 0.0;
    for (int64_t n = 1; n <= KV_FEW * 4 && (n == 1 || last / n >= 8); ++n) {
        const int64_t rounds = (p.tiles * c.heads * n + 255) / 256;
        const double each = (double)(((rounds == 1 ? last : middle) + n - 1) / n);
        const double us = 4.0 + (double)rounds * (wide ? 8.0 + 2.0 * each : 6.0 + 1.75 * each) + ka_join_us(c, heads, n);
        if (n == 1 || us < best) best = us, p.splits = (int)n;
    }
    return best < plain || c.kernel == 2 ? p : s;
}

size_t kv8_attend_ws(const Kv8View& c, const int* row0, int heads, int sink, int ring, int longest) {
    // (enough for a call of any type)
    const int s = std::max(shape_of(c, row0, KV_F32, heads, sink, ring, longest).splits,
                           shape_of(c, row0, KV_F16, heads, sink, ring, longest).splits);
    return s > 1 ? (size_t)s * c.rows * heads * (c.dv + 2) * 4 : 0;
}

static hipError_t joined(const Kv8View& c, const Kv8AttendArgs& a, const KaPlan& plan, int type, hipStream_t s) {
    if (const hipError_t e = hipGetLastError()) return e;
    if (plan.splits == 1) return hipSuccess;
    return launch_kv_join({a.out, a.lse, reinterpret_cast<const float*>(a.ws), (int64_t)c.rows * a.heads, a.ldo, a.heads, c.dv, plan.splits},
                          type, s);
}

template <int TYPE, int WK, int WV>
static hipError_t attend_shaped(const Kv8View& c, const int* row0, const Kv8AttendArgs& a, int longest, hipStream_t s) {
    const Ka8Shape shape = shape_of(c, row0, TYPE, a.heads, a.sink, a.ring, longest);
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    KaPlan plan;
    plan.tiles_each = shape.tiles_each;
    plan.splits = shape.splits;
    plan.aligned = c.dk % 8 == 0 && (uintptr_t)a.q % 16 == 0 && a.ldq * es % 16 == 0 && c.dk * es % 16 == 0;
    plan.out_aligned = c.dv % 4 == 0 && (uintptr_t)a.out % 16 == 0 && a.ldo * es % 16 == 0;
    if (shape.tiles * c.heads > KV8_THREADS / 512 || (int64_t)c.rows * a.heads > 0x7fffff00) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(shape.tiles * c.heads), plan.splits);
    if constexpr (WK <= 128 && TYPE != KV_F32)
        if (shape.prompt) {
            if (const hipError_t e = launch_kv8_prompt(c, a, plan, shape.tiles * c.heads, s)) return e;
            return joined(c, a, plan, TYPE, s);
        }
    auto kern = k_kv8_attend<TYPE, WK, WV, 4>;
    if constexpr (WK <= 128)
        if (shape.waves == 8) kern = k_kv8_attend<TYPE, WK, WV, 8>;
    hipLaunchKernelGGL(kern, grid, dim3(shape.waves * 64), 0, s, c, a, plan);
    return joined(c, a, plan, TYPE, s);
}

template <int TYPE>
static hipError_t attend_typed(const Kv8View& c, const int* row0, const Kv8AttendArgs& a, int longest, hipStream_t s) {
    return c.wk == 64    ? attend_shaped<TYPE, 64, 64>(c, row0, a, longest, s)
           : c.wk == 128 ? attend_shaped<TYPE, 128, 128>(c, row0, a, longest, s)
           : c.wk == 192 ? attend_shaped<TYPE, 192, 128>(c, row0, a, longest, s)
                         : attend_shaped<TYPE, 256, 256>(c, row0, a, longest, s);
}

hipError_t launch_kv8_attend(const Kv8View& c, const int* row0, const Kv8AttendArgs& a, int longest, hipStream_t s) {
    return a.type == KV_F32   ? attend_typed<KV_F32>(c, row0, a, longest, s)
           : a.type == KV_F16 ? attend_typed<KV_F16>(c, row0, a, longest, s)
                              : attend_typed<KV_BF16>(c, row0, a, longest, s);
}

}  // namespace nh
