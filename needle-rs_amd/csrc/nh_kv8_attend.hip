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
// addition takes 1152: exact.  f32 queries go the other way: their rows as whole
// numbers of 23 bits in three signed digits of 8, times the codes in the i8
// MFMAs, which are exact and take the bytes as they are.
// The products are transposed, keys (or dims) by rows: S^T = K Q^T leaves lane (o,
// kg) the scores of its row o with keys 16 t + 4 kg + 0..3, and a lane's 16 bytes
// of values are of those very keys, so a weight never leaves its lane, and a
// row's maximum, sum and correction are one lane's scalars.
#include <algorithm>

#include "nh_kv8_device.h"

namespace nh {

typedef int i32x4_ __attribute__((ext_vector_type(4)));

// What a lane loads of a chunk.
template <int WK, int WV>
struct Ka8Chunk {
    u32x4 k[4][WK / 64], v[WV / 16];
    f32x4 ks, vs;
    u32x4 bad;  // 4 u16 of the keys, 4 of the values
};

// NW wavefronts a workgroup, each every NW-th chunk of the range; RT tiles of 16 rows.
template <int TYPE, int WK, int WV, int RT, int NW>
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
        b = kv_find(c, tile, lane, [&](const KvEntry& e) { return ((e.row1 - e.row0) * per + 16 * RT - 1) / (16 * RT); });
    }
    if (b >= c.nb) return;
    const KvEntry entry = kv_batch(c, b);
    const int row0 = entry.row0, nrows = entry.row1 - row0, seq = entry.seq;
    const int first = entry.len - (c.ask ? 1 : nrows), r0 = tile * 16 * RT;
    if (!kv_current(c) || (!c.ask && first < 0) || r0 >= nrows * per || entry.row1 > c.rows) return;
    const int r1 = min(r0 + 16 * RT, nrows * per) - 1;
    const int plo = first + (c.ask ? 0 : r0 / per), phi = first + (c.ask ? 0 : r1 / per);

    // The queries: f16 operands scaled by a power of two to just under 2^15, or digits.
    h8 q[RT][NJ][2];
    i32x4_ qd[RT][3][NJ];
    float cq[RT];
    int pos[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(r0 + rt * 16 + o, r1), t = r / per;
        pos[rt] = first + (c.ask ? 0 : t);
        const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + t) * a.ldq + (int64_t)(kvh * per + r - t * per) * c.dk;
        float x[NJ][16], most = 0.0f;
        bool nan = false;
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
                    for (int e = 0; e < 8; ++e) x[j][8 * g + e] = (float)y[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[j][8 * g + e] = d + e < c.dk ? KvElem<TYPE>::get(src + d + e) : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    most = fmaxf(most, fabsf(x[j][8 * g + e]));
                    nan |= x[j][8 * g + e] != x[j][8 * g + e];
                }
            }
        if constexpr (DIGITS) {
            most = nan ? __builtin_inff() : most;
            most = groups_max(most);
            // |x| <= most, as a whole number of at most 127 (2^16 + 2^8 + 1)
            const float full = 8355711.0f;
            const bool fine = most < __builtin_inff(), some = most > 0x1p-100f;
            const float up = fine && some ? full / most : 0.0f;
            // z = 2^-8 of the sum of whole numbers x codes
            cq[rt] = fine ? (a.scale * KA_LOG2E) * (some ? most * (256.0f / full) : 0.0f) : __builtin_nanf("");
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
                    qd[rt][0][j][w] = (int)d0;
                    qd[rt][1][j][w] = (int)d1;
                    qd[rt][2][j][w] = (int)d2;
                }
        } else {
            most = groups_max(most);
            const int ef = max((int)(__builtin_bit_cast(uint32_t, most) >> 23 & 255u), 15);
            const float up = __builtin_bit_cast(float, (uint32_t)(268 - ef) << 23);
            cq[rt] = (a.scale * KA_LOG2E) * __builtin_bit_cast(float, (uint32_t)(ef - 14) << 23);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) q[rt][j][e / 8][e % 8] = (_Float16)(x[j][e] * up);
        }
    }

    f32x4 acc[RT][NV];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff();
        l[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[rt][i] = f32x4{0, 0, 0, 0};
    }
    // The weights are kept as 2^15 p, and with their steps as the f16 operand 2^15 p
    // step / 2^eref, 2^eref above every step seen so far: at most 2^15, and exact to
    // 11 bits down to 2^-29 of it.
    int eref = -126;

    const Ka8Span span(plo, phi, a.sink, a.ring);
    const int sink = a.ring ? a.sink : 0x7fffffff, ring = a.ring;
    const int per_split = max((span.count() + plan.splits - 1) / plan.splits, NW);
    const int c0 = split * per_split, c1 = min(c0 + per_split, span.count());

    const int* table = c.table + (size_t)seq * c.table_ld;
    auto page_of = [&](int i) { return i < c1 ? table[span.at(i) * KV8_CHUNK >> c.page_log2] : 0; };
    auto load = [&](Chunk& x, int i, int pg) {
        const int slot = span.at(i) * KV8_CHUNK & (c.page() - 1);
        // (a page id comes from the cache's own table; a bad one is not followed)
        const uint8_t* p = kv8_block(c, (unsigned)pg < (unsigned)c.pages ? pg : 0, a.layer, kvh) + (uint32_t)(slot >> 6) * L::CHUNK;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j) x.k[t][j] = *reinterpret_cast<const u32x4*>(p + L::k_piece(t, j, lane));
        x.ks = *reinterpret_cast<const f32x4*>(p + L::RECORD);
        x.vs = *reinterpret_cast<const f32x4*>(p + L::RECORD + 16);
        x.bad = *reinterpret_cast<const u32x4*>(p + L::RECORD + 32);
#pragma unroll
        for (int n = 0; n < NV; ++n) x.v[n] = *reinterpret_cast<const u32x4*>(p + L::v_piece(n, lane));
    };

    auto compute = [&](const Chunk& x, int i) {
        const int key0 = span.at(i) * KV8_CHUNK;
        const bool whole = key0 + KV8_CHUNK - 1 <= plo && (key0 + KV8_CHUNK - 1 < sink || key0 > phi - ring);
        const uint32_t bad0 = __builtin_amdgcn_readfirstlane((int)(x.bad[0] | x.bad[2]));
        const uint32_t bad1 = __builtin_amdgcn_readfirstlane((int)(x.bad[1] | x.bad[3]));
        const bool plain = whole && !(bad0 | bad1);
        // The steps' reference: raised when a step passes it (of a block that the tile sees).
        float top = x.vs[0];
#pragma unroll
        for (int t = 1; t < 4; ++t) top = fmaxf(top, key0 + 16 * t <= phi ? x.vs[t] : 0.0f);
        const int et = __builtin_amdgcn_readfirstlane((int)(__builtin_bit_cast(uint32_t, top) >> 23)) - 126;
        if (et > eref) {
            const float down = pow2i(max(eref - et, -126));
            eref = et;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < NV; ++k) acc[rt][k] *= down;
        }
        const float wscale = pow2i(-eref);
        float vstep[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) vstep[t] = key0 + 16 * t <= phi ? x.vs[t] * wscale : 0.0f;
        f32x4 z[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if constexpr (DIGITS) {
                i32x4_ n[RT][3] = {};
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const i32x4_ k = __builtin_bit_cast(i32x4_, x.k[t][j] ^ 0x80808080u);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int d = 0; d < 3; ++d) n[rt][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, qd[rt][d][j], n[rt][d], 0, 0, 0);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        z[rt][t][r] = __builtin_fmaf((float)n[rt][2][r], 0x1p-8f, (float)(n[rt][0][r] * 256 + n[rt][1][r]));
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) z[rt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const h8 k = codes8(x.k[t][j][2 * g], x.k[t][j][2 * g + 1]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) z[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rt][j][g], z[rt][t], 0, 0, 0);
                    }
            }
        }
        h8 pw[RT][2][WPARTS];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const bool fresh = m[rt] == -__builtin_inff();  // no key seen yet
            const float base = fresh ? 0.0f : m[rt];
            float s[4][4];  // 15 + log2 of the weight against the maximum so far
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float f = cq[rt] * x.ks[t];
#pragma unroll
                for (int r = 0; r < 4; ++r) s[t][r] = __builtin_fmaf(z[rt][t][r], f, 15.0f - base);
            }
            if (!plain) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t bad = (t & 2 ? bad1 : bad0) >> (16 * (t & 1)) >> (4 * kg);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = key0 + 16 * t + 4 * kg + r;
                        const bool seen = (j <= pos[rt]) & ((j < sink) | (j > pos[rt] - ring));
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
                m[rt] = fresh && most == -__builtin_inff() ? m[rt] : base + over;
                l[rt] *= keep;
#pragma unroll
                for (int k = 0; k < NV; ++k) acc[rt][k] *= keep;
#pragma unroll
                for (int k = 0; k < 16; ++k) s[k / 4][k % 4] -= over;
            }
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const f32x2 p = {__builtin_amdgcn_exp2f(s[k / 4][k % 4]), __builtin_amdgcn_exp2f(s[k / 4][k % 4 + 1])};
                l[rt] += p[0];
                l[rt] += p[1];
                const f32x2 w = {p[0] * vstep[k / 4], p[1] * vstep[k / 4]};
                const h2 hi = __builtin_convertvector(w, h2);
                pw[rt][k / 8][0][k % 8] = hi[0], pw[rt][k / 8][0][k % 8 + 1] = hi[1];
                if constexpr (WPARTS == 2) {
                    const f32x2 rest = {w[0] - (float)hi[0], w[1] - (float)hi[1]};
                    const h2 lo = __builtin_convertvector(rest, h2);
                    pw[rt][k / 8][1][k % 8] = lo[0], pw[rt][k / 8][1][k % 8 + 1] = lo[1];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const h8 v = codes8(x.v[n][2 * h], x.v[n][2 * h + 1]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int p = 0; p < WPARTS; ++p)
                        acc[rt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pw[rt][h][p], acc[rt][n], 0, 0, 0);
            }
    };

    // The loads of the next chunk are in flight during this one's arithmetic, the
    // page id of the one after it is on its way.
    {
        Chunk x[2];
        int i = c0 + wave;
        auto fetch = [&](Chunk& to, int at, int pg) {
            if (at < c1) load(to, at, pg);
        };
        int p0 = page_of(i), p1 = page_of(i + NW);
        fetch(x[0], i, p0);
        while (i < c1) {
#pragma unroll
            for (int k = 0; k < 2; ++k, i += NW) {
                if (i >= c1) break;
                fetch(x[k ^ 1], i + NW, p1);
                p1 = page_of(i + 2 * NW);
                compute(x[k], i);
            }
        }
    }

    // The wavefronts' sums joined, 16 rows at a time.
    const float unit = pow2i(eref);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = groups_sum(l[rt]);
        if (l[rt] != l[rt]) m[rt] = l[rt];  // NaN scores: the row's, whatever other ranges hold
        if (rt) __syncthreads();
        if (kg == 0) sm[wave][o] = m[rt], sl[wave][o] = l[rt] * 0x1p-15f;
        __syncthreads();
        float most = sm[0][o];
#pragma unroll
        for (int w = 1; w < NW; ++w) most = fmaxf(most, sm[w][o]);
        const float base = most == -__builtin_inff() ? 0.0f : most;
        const float f = __builtin_amdgcn_exp2f(m[rt] - base) * 0x1p-15f;
#pragma unroll
        for (int n = 0; n < NV; ++n) *reinterpret_cast<f32x4*>(&so[wave][o][16 * n + 4 * kg]) = acc[rt][n] * f * unit;
        __syncthreads();
        for (int x = tid; x < 16 * WV; x += NW * 64) {
            const int rr = x / WV, d = x % WV, r = r0 + rt * 16 + rr;
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
                // (no key seen: 0)
                KvElem<TYPE>::put(reinterpret_cast<T*>(a.out) + row * a.ldo + (int64_t)head * c.dv + d, sum == 0.0f ? 0.0f : v / sum);
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

static Ka8Shape shape_of(const Kv8View& c, const int* row0, int type, int heads, int sink, int ring, int longest) {
    const int per = heads / c.heads;
    const int64_t tokens = c.nb ? (c.rows + c.nb - 1) / c.nb : 0;
    Ka8Shape s;
    s.prompt = false;
    if (type != KV_F32 && c.wk <= 128 && c.kernel != 1 && c.nb && ((int64_t)c.rows * per / c.nb >= 128 || c.kernel == 2)) {
        s.prompt = true;
        s.waves = 0;
        s.splits = 1;
        tiles_of(c, row0, per, 128, s);
        if (s.tiles * c.heads > 256) tiles_of(c, row0, per, 256, s);
        return s;
    }
    tiles_of(c, row0, per, 16, s);
    const int64_t base = s.tiles * c.heads;
    s.waves = c.wk <= 128 && base <= 256 ? 8 : 4;
    const int64_t slots = s.waves == 8 || c.wk > 128 ? 256 : 512;
    const int64_t wide = std::min<int64_t>(tokens, s.rows / per + 1);
    const int64_t keys = ring ? std::min<int64_t>(longest, (int64_t)sink + ring + wide + 2 * KV8_CHUNK) : longest;
    const int64_t chunks = (keys + KV8_CHUNK - 1) / KV8_CHUNK;
    const int64_t want = base ? std::max<int64_t>(1, slots / base) : 1;
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, KV_SPLITS), chunks / (2 * s.waves)));
    return s;
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
    if (shape.tiles * c.heads > 0x7fffffff || (int64_t)c.rows * a.heads > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(shape.tiles * c.heads), plan.splits);
    if constexpr (WK <= 128 && TYPE != KV_F32)
        if (shape.prompt) {
            if (const hipError_t e = launch_kv8_prompt(c, a, plan, shape.tiles * c.heads, shape.rows, s)) return e;
            return joined(c, a, plan, TYPE, s);
        }
    auto kern = k_kv8_attend<TYPE, WK, WV, 1, 4>;
    if constexpr (WK <= 128)
        if (shape.waves == 8) kern = k_kv8_attend<TYPE, WK, WV, 1, 8>;
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
