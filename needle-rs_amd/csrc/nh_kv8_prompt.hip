// Attention of many rows over the 8-bit cache (the layout: nh_kv8.h; the mathematics
// and the kernel of few rows: nh_kv8_attend.hip).
#include "nh_kv8_device.h"

namespace nh {

// Many rows: a workgroup of eight wavefronts takes 32 rows a wavefront, and the
// chunks' codes are turned into f16 operands once for all of them, through
// LDS.  32 x 32 MFMAs: a lane holds 16 of its row's scores with 32 keys, the other
// half of them is 32 lanes away.
//
// A value's step goes into the exponent: p' = 2^(score + log2 step - reference) is
// the weight x step that the second product wants of that key, and the sum of the
// weights themselves is that of p' / step, 16 keys at a time.  The reference is the
// row's largest score + log2 step (within 2^7, so that it is hardly ever moved), so
// a row's weights x steps keep their 11 bits down to 2^-22 of the largest of them.  A
// step below 2^-60 of the largest that the rows see counts as that (2^-125 where that
// is more), so 1 / step passes what a row was given its reference at by 2^60 at most.
// The sum is held in a unit 2^-e of the row's own, chosen anew where its reference
// moves, as the sum or the largest new weight is then: steps of any size before and
// after one another leave it within f32.  (A unit fixed by the first 64 keys lost it
// where later steps were 2^120 times as large.)
//
// 2 x 2,000 rows after 6,000 keys, 32 heads over 8 of 128 (427 GFLOP), bf16: 440 to 470
// us, 910 to 970 TFLOP/s, where a large product reaches 1,320 to 1,370.  The matrix
// cores are busy for half of the cycles: a row's 32 exponentials, and as many sums and
// products, are vector work for nearly as long as its products, and two wavefronts a SIMD
// do not overlap them whole.  With the turning of the codes and the records taken out
// the loop takes 380, with the reference's tests out too 345, and 255 of that without the
// operands' reads from LDS.  Slower were 64 rows a wavefront (669 to 917: the
// accumulators pass the registers), halves that alternate by barriers (563), four
// wavefronts on images of 32 keys (530), sums by dot products (477), two chunks of
// loads in registers (463) and exponentials put off by half a chunk (453 for 452).
// At 64 dims there are half as many products for as many exponentials: 16 x 512 rows
// over 2,000 keys, 16 heads, 112 to 138 us; a wavefront alone takes 3,000 cycles for 64
// keys, and more than two a SIMD have no registers (four wavefronts, three a SIMD: 154).
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int KP8_WAVES = 8;
static_assert(KP8_ROWS == 32 * KP8_WAVES, "32 rows a wavefront");

template <int W>
struct Kp8Image {  // a chunk's operands, 16 bytes a lane each
    u32x4 k[2][W / 16][64], v[W / 32][4][64];
    float ks[4], lv[4], rv[4];  // the keys' steps; log2 of the values' (inf: a marked row among them), 1 over them
    float marked_lv[4];         // log2 of the steps of blocks with marked rows too
    uint32_t marks[2];          // rows of the keys or the values, a bit each
    int pad[2];
};

template <int TYPE, int W>
__global__ __launch_bounds__(KP8_WAVES * 64, 2) void k_kv8_prompt(Kv8View c, Kv8AttendArgs a, KaPlan plan) {
    typedef typename KvElem<TYPE>::T T;
    typedef Kv8Lay<W, W> L;
    typedef Kp8Image<W> Image;
    constexpr int NX = W / 16, ND = W / 32, ROWS = KP8_ROWS, NW = KP8_WAVES;
    // A wavefront turns a piece of the keys and one of the values, or (APART) one of either.
    constexpr bool APART = NX < NW;
    static_assert(APART ? 2 * NX == NW : NX == NW, "every piece is turned once");
    extern __shared__ __align__(16) uint8_t lds8[];
    Image* img = reinterpret_cast<Image*>(lds8);

    const int tid = threadIdx.x, lane = tid & 63, o = lane & 15, kg = lane >> 4, half = lane >> 5, m32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % c.heads, per = a.heads / c.heads, split = blockIdx.y;
    int tile = blockIdx.x / c.heads, b;
    if (plan.tiles_each) {
        b = tile / plan.tiles_each;
        tile = plan.tiles_each - 1 - (tile - b * plan.tiles_each);  // the longest first
    } else
        b = kv_find(c, tile, lane, [&](const KvEntry& e) { return ((e.row1 - e.row0) * per + ROWS - 1) / ROWS; });
    if (b >= c.nb) return;
    const KvEntry entry = kv_batch(c, b);
    const int row0 = entry.row0, nrows = entry.row1 - row0, first = entry.len - (c.ask ? 1 : nrows), r0 = tile * ROWS;
    if (!kv_current(c) || (!c.ask && first < 0) || r0 >= nrows * per || entry.row1 > c.rows) return;
    const int r1 = min(r0 + ROWS, nrows * per) - 1;
    const int plo = first + (c.ask ? 0 : r0 / per), phi = first + (c.ask ? 0 : r1 / per);
    const int w0 = min(r0 + wave * 32, r1), w1 = min(w0 + 31, r1);  // this wavefront's rows
    const int wlo = first + (c.ask ? 0 : w0 / per), whi = first + (c.ask ? 0 : w1 / per);
    const int sink = a.ring ? a.sink : 0x7fffffff, ring = a.ring;

    const int r = min(r0 + wave * 32 + m32, r1), token = r / per, pos = first + (c.ask ? 0 : token);
    h8 q[NX];
    float cq, m = -__builtin_inff(), l = 0.0f, unit = 1.0f;  // (l: the weights' sum x unit, 2^e)
    f32x16 acc[ND];
    {
        const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(row0 + token) * a.ldq + (int64_t)(kvh * per + r - token * per) * c.dk;
        T x[NX][8];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < NX; ++j) {
            const int d = 16 * j + 8 * half;
            if (plan.aligned) {
                typedef T Vec __attribute__((ext_vector_type(8)));
                Vec y = {};
                if (d < c.dk) y = *reinterpret_cast<const Vec*>(src + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = y[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = d + e < c.dk ? src[d + e] : (T)0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)x[j][e]));
        }
        // (scaled by a power of two to just under 2^15, as above)
        top = halves_max(top);
        const int ef = max((int)(__builtin_bit_cast(uint32_t, top) >> 23 & 255u), 15);
        const float up = __builtin_bit_cast(float, (uint32_t)(268 - ef) << 23);
        cq = (a.scale * KA_LOG2E) * __builtin_bit_cast(float, (uint32_t)(ef - 14) << 23);
#pragma unroll
        for (int j = 0; j < NX; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) q[j][e] = (_Float16)((float)x[j][e] * up);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    }

    const Ka8Span span(plo, phi, a.sink, a.ring);
    const int per_split = (span.count() + plan.splits - 1) / plan.splits;
    const int c0 = split * per_split, c1 = min(c0 + per_split, span.count());
    const int* table = c.table + (size_t)entry.seq * c.table_ld;
    const int last = c1 - 1;
    // (page ids by vector loads: a scalar one in flight makes every wait for LDS a wait for all of it)
    int lane0 = 0;
    asm volatile("" : "+v"(lane0));
    const int page_log2 = c.page_log2, pages = c.pages, in_page = (c.page() >> 6) - 1;
    auto page_of = [&](int i) { return table[(span.at(min(i, last)) * KV8_CHUNK >> page_log2) + lane0]; };
    const uint8_t* base = kv8_block(c, 0, a.layer, kvh);
    const uint32_t page_bytes = (uint32_t)(c.block() * c.heads * c.layers);  // (below 2^32: shape_of)

    struct Raw {
        u32x4 k, v;
        uint32_t rec;  // a word of the record each lane: 4 steps of the keys, 4 of the values, 4 of marks
    };
    // Where chunk i lies (past the end: the last one again), and its loads.
    auto where = [&](int i, int pg) {
        const uint32_t known = (unsigned)pg < (unsigned)pages ? (uint32_t)pg : 0u;
        return base + (uint64_t)known * page_bytes + (uint32_t)((span.at(min(i, last)) & in_page) * L::CHUNK);
    };
    auto load = [&](Raw& x, const uint8_t* p) {
        const int n = wave & (NX - 1);
        if (!APART || wave < NX) x.k = *reinterpret_cast<const u32x4*>(p + n * 1024 + lane * 16);
        if (!APART || wave >= NX) x.v = *reinterpret_cast<const u32x4*>(p + L::v_piece(n, lane));
        x.rec = *reinterpret_cast<const uint32_t*>(p + L::RECORD + 4 * (lane & 15));
    };
    // Step `step` of six of turning: two of a piece of the keys, four of one of the values.
    auto turn = [&](const Raw& x, Image& to, int step) {
        const int n = wave & (NX - 1);
        if (step < 2) {
            // piece (t, j), 16 dims of position 16 t + o: the halves of the product's step 4 j + kg
            const int t = n / L::NJ, j = n % L::NJ;
            to.k[t >> 1][4 * j + kg][32 * step + 16 * (t & 1) + o] = __builtin_bit_cast(u32x4, codes8(x.k[2 * step], x.k[2 * step + 1]));
        } else if (step < 6) {
            // dim 16 n + o, four positions of a block
            const int t = step - 2;
            const h2 y = codes2(x.v[t], 0x04010400u), w = codes2(x.v[t], 0x04030402u);
            const uint2 both = {__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, w)};
            reinterpret_cast<uint2*>(&to.v[n >> 1][t][32 * (kg & 1) + 16 * (n & 1) + o])[kg >> 1] = both;
        }
    };
    float top = 0.0f;  // the largest step so far
    auto record = [&](const Raw& x, int i, Image& to) {
        if (wave != 0) return;
        const int key0 = span.at(min(i, last)) * KV8_CHUNK;
        // lane 4 + t: the step of block t's values, 0 of hidden ones; the quad's largest
        const float mine = __builtin_bit_cast(float, x.rec);
        const float vs = lane >= 4 && lane < 8 && ka8_sees(key0 + 16 * (lane - 4), plo, phi, sink, ring) ? mine : 0.0f;
        float most = fmaxf(vs, quad_xor1(vs));
        top = fmaxf(top, fmaxf(most, quad_xor2(most)));
        const float least = fmaxf(top * 0x1p-60f, 0x1p-125f);
        // (words 8, 9 and 10, 11: the keys' and the values' marks of two blocks each)
        const uint32_t marks = x.rec | __builtin_bit_cast(uint32_t, quad_xor2(mine));
        const uint32_t m0 = (uint32_t)__builtin_amdgcn_readlane((int)marks, 8), m1 = (uint32_t)__builtin_amdgcn_readlane((int)marks, 9);
        if (lane < 4) to.ks[lane] = mine;
        if (lane >= 4 && lane < 8) {
            const int t = lane - 4;
            const float v = fmaxf(vs, least), lv = __builtin_amdgcn_logf(v);
            to.lv[t] = (t & 2 ? m1 : m0) >> (16 * (t & 1)) & 0xffffu ? __builtin_inff() : lv;
            to.marked_lv[t] = lv;
            to.rv[t] = __builtin_amdgcn_rcpf(v);
        }
        if (lane < 2) to.marks[lane] = lane ? m1 : m0;
    };
    auto whole_turn = [&](const Raw& x, int i, Image& to) {
#pragma unroll
        for (int step = 0; step < 6; ++step)
            if (!APART || (step < 2) == (wave < NX)) turn(x, to, step);
        record(x, i, to);
    };

    auto exponent = [](float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23) - 127; };
    float s[16], limit = -__builtin_inff();  // (a score past it moves the reference; none yet: any)
    f32x16 z;
    h8 p[2], kx[NX], vx[2 * ND];
    float most;
    auto key = [&](const Image& now, int tk, int j) { return __builtin_bit_cast(h8, now.k[tk][j][lane]); };
    auto value = [&](const Image& now, int tk, int j) { return __builtin_bit_cast(h8, now.v[j >> 1][2 * tk + (j & 1)][lane]); };
    // Hidden keys and marked rows, and the reference raised where a score passes it by
    // 2^7 (or there was none).
    auto settle = [&](const Image& now, int i, int tk) {
        const int key0 = span.at(i) * KV8_CHUNK + 32 * tk;
        const bool plain = key0 + 31 <= wlo && (key0 + 31 < sink || key0 > whi - ring);
        if (plain && !__any(most > limit)) return;
        const bool fresh = m == -__builtin_inff();
        const uint32_t marks = __builtin_amdgcn_readfirstlane((int)now.marks[tk]);
        int at4 = 4 * half;
        asm volatile("" : "+v"(at4));  // (or 32 registers hold the keys' numbers and bits throughout the loop)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int at = 8 * (e >> 2) + at4 + (e & 3), j = key0 + at, t = 2 * tk + (e >> 3);
            const bool seen = (j <= pos) & ((j < sink) | (j > pos - ring));
            // (the other rows of a block with a marked one: their scores again, with its step)
            if (marks) s[e] = __builtin_fmaf(z[e], cq * now.ks[t], now.marked_lv[t] + (8.0f - (fresh ? 0.0f : m)));
            s[e] = !seen ? -__builtin_inff() : marks >> at & 1 ? __builtin_nanf("") : s[e];
        }
        most = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) most = fmaxf(most, s[e]);
        most = halves_max(most);
        if (__any(most > limit)) {
            const float over = most == -__builtin_inff() ? 0.0f : fresh ? most - 8.0f : fmaxf(most - 8.0f, 0.0f);
            const float keep = fresh ? 0.0f : __builtin_amdgcn_exp2f(-over);
            m = fresh && most == -__builtin_inff() ? m : (fresh ? 0.0f : m) + over;
            limit = m == -__builtin_inff() ? m : 15.0f;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= keep;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] -= over;
            // The sum's unit: log2 of the weights' sum so far, or of the largest weight among
            // these keys, whichever is more (-inf: no key yet).
            float of[2] = {s[0], s[8]};
#pragma unroll
            for (int e = 1; e < 8; ++e) of[0] = fmaxf(of[0], s[e]), of[1] = fmaxf(of[1], s[8 + e]);
            const float now_l = fmaxf(of[0] - now.marked_lv[2 * tk], of[1] - now.marked_lv[2 * tk + 1]);
            const int e0 = exponent(unit);
            const float was = fresh ? -__builtin_inff() : __builtin_amdgcn_logf(l) - (float)e0 - over;
            // (both halves of the row hold sums of their own, in one unit)
            const float both = halves_max(fmaxf(now_l, was));
            const int e1 = both == -__builtin_inff() ? e0 : (int)rintf(fminf(fmaxf(-both, -126.0f), 126.0f));
            l = fresh ? 0.0f : l * __builtin_amdgcn_exp2f((float)(e1 - e0) - over);
            unit = pow2i(e1);
        }
    };
    // Half `tk` of a chunk, in two parts whose instructions are written down in the
    // order in which they are to issue: with each product the read of an operand that
    // the other part wants, and vector work for about as long as the product takes.
    // The first part has the next half's scores over this one's weights, the second
    // one this half's sums over the next one's scores against the reference (and over
    // a wavefront's share of turning a later chunk's codes).
    auto weights_part = [&](const Image& now, int tk) {
        // (what is read first is there first: waits for it do not wait for the operands)
        const float rv[2] = {now.rv[2 * tk], now.rv[2 * tk + 1]};
        z = f32x16{};
        float sum[2] = {0.0f, 0.0f};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int n = j * NX / 8; n < (j + 1) * NX / 8; ++n) {
                z = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[n], q[n], z, 0, 0, 0);
                vx[n] = value(now, tk, n);
            }
            const f32x2 w = {__builtin_amdgcn_exp2f(s[2 * j]), __builtin_amdgcn_exp2f(s[2 * j + 1])};
            sum[j >> 2] += w[0];
            sum[j >> 2] += w[1];
            const h2 w2 = __builtin_convertvector(w, h2);
            p[j >> 2][2 * j % 8] = w2[0], p[j >> 2][2 * j % 8 + 1] = w2[1];
            __builtin_amdgcn_sched_barrier(0);
        }
        l = __builtin_fmaf(sum[0], rv[0] * unit, l);
        l = __builtin_fmaf(sum[1], rv[1] * unit, l);
    };
    // (scores of half `tk` of `with`, keys of half `kt` of `keys`)
    auto sums_part = [&](const Image& with, int tk, const Image& keys, int kt, auto also) {
        const float base = m == -__builtin_inff() ? 0.0f : m;
        float f[2], to[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) f[t] = cq * with.ks[2 * tk + t], to[t] = with.lv[2 * tk + t] + (8.0f - base);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int n = j * NX / 8; n < (j + 1) * NX / 8; ++n) {
                // (the sums of the first 16 keys before the others')
                const int t = n / ND, d = n % ND;
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx[2 * d + t], p[t], acc[d], 0, 0, 0);
                kx[n] = key(keys, kt, n);
            }
            s[2 * j] = __builtin_fmaf(z[2 * j], f[j >> 2], to[j >> 2]);
            s[2 * j + 1] = __builtin_fmaf(z[2 * j + 1], f[j >> 2], to[j >> 2]);
            most = j ? fmaxf(fmaxf(most, s[2 * j]), s[2 * j + 1]) : fmaxf(s[0], s[1]);
            also(j);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Three images in turn: the one after the next is written at the end of a chunk,
    // when a wavefront that is behind may still read the chunk's own and the next, and
    // the barrier in the middle of the next chunk makes it whole.  The loads run a chunk
    // ahead of that.
    if (c0 < c1) {
        Raw x;
        load(x, where(c0, page_of(c0)));
        whole_turn(x, c0, img[0]);
        load(x, where(c0 + 1, page_of(c0 + 1)));
        whole_turn(x, c0 + 1, img[1]);
        load(x, where(c0 + 2, page_of(c0 + 2)));
        int pg = page_of(c0 + 3);
        __syncthreads();
        // the first half's scores; sums of nothing over its way to the reference
        z = f32x16{};
#pragma unroll
        for (int n = 0; n < NX; ++n) {
            vx[n] = h8{};
            z = __builtin_amdgcn_mfma_f32_32x32x16_f16(key(img[0], 0, n), q[n], z, 0, 0, 0);
        }
        p[0] = p[1] = h8{};
        sums_part(img[0], 0, img[0], 1, [](int) {});
        settle(img[0], c0, 0);
        int at = 0;
        for (int i = c0; i < c1; ++i) {
            const Image& now = img[at];
            const Image& next = img[at == 2 ? 0 : at + 1];
            Image& then = img[at == 0 ? 2 : at - 1];
            at = at == 2 ? 0 : at + 1;
            weights_part(now, 0);
            __syncthreads();
            const uint8_t* p;
            sums_part(now, 1, next, 0, [&](int j) {
                if (j == 0) p = where(i + 3, pg);
                if (j == 4) pg = page_of(i + 4);
            });
            settle(now, i, 1);
            weights_part(now, 1);
            if constexpr (APART) {
                sums_part(next, 0, next, 1, [](int) {});
                whole_turn(x, i + 2, then);
            } else {
                sums_part(next, 0, next, 1, [&](int j) { turn(x, then, j); });
                record(x, i + 2, then);
            }
            load(x, p);
            if (i + 1 < c1) settle(next, i + 1, 0);
        }
    }

    const int up = exponent(unit);
    const float sum = l + __shfl_xor(l, 32, 64);
    if (r0 + wave * 32 + m32 > r1) return;
    const int64_t row = row0 + token, head = kvh * per + r - token * per;
    const bool alone = plan.splits == 1;
    // the sums are of p / step x 2^up; the reference counts the step, and 2^8
    const float at_ref = m - (float)up - 8.0f;
    const float scale = alone ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
    T* out = reinterpret_cast<T*>(a.out) + row * a.ldo + head * c.dv;
    const int64_t at = ((int64_t)split * c.rows + row) * a.heads + head;
    float* ml = reinterpret_cast<float*>(a.ws);
    float* po = ml + 2 * ((int64_t)plan.splits * c.rows * a.heads) + at * c.dv;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int dim = 32 * d + 8 * (e >> 2) + 4 * half;
            float y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = __builtin_amdgcn_ldexpf(acc[d][e + k] * scale, up);
            if (alone) {
                typedef T Vec4 __attribute__((ext_vector_type(4)));
                if (plan.out_aligned && dim + 4 <= c.dv) {
                    Vec4 w;
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = (T)y[k];
                    *reinterpret_cast<Vec4*>(out + dim) = w;
                } else
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (dim + k < c.dv) out[dim + k] = (T)y[k];
            } else
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (dim + k < c.dv) po[dim + k] = y[k];
        }
    if (half == 0) {
        if (alone) {
            if (a.lse) a.lse[row * a.heads + head] = (at_ref + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
        } else
            ml[2 * at] = sum == sum ? at_ref : sum, ml[2 * at + 1] = sum;
    }
}

template <int TYPE, int W>
static hipError_t prompt_shaped(const Kv8View& c, const Kv8AttendArgs& a, const KaPlan& plan, int64_t tiles, hipStream_t s) {
    auto kern = k_kv8_prompt<TYPE, W>;
    const int lds = 3 * (int)sizeof(Kp8Image<W>);
    // (more than a kernel may have without being asked for it)
    if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds))
        return e;
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles, plan.splits), dim3(KP8_WAVES * 64), lds, s, c, a, plan);
    return hipGetLastError();
}

hipError_t launch_kv8_prompt(const Kv8View& c, const Kv8AttendArgs& a, const KaPlan& plan, int64_t tiles, hipStream_t s) {
    if (a.type == KV_F32 || c.wk > 128) return hipErrorInvalidValue;
    if (c.wk == 64)
        return a.type == KV_F16 ? prompt_shaped<KV_F16, 64>(c, a, plan, tiles, s) : prompt_shaped<KV_BF16, 64>(c, a, plan, tiles, s);
    return a.type == KV_F16 ? prompt_shaped<KV_F16, 128>(c, a, plan, tiles, s) : prompt_shaped<KV_BF16, 128>(c, a, plan, tiles, s);
}

}  // namespace nh
