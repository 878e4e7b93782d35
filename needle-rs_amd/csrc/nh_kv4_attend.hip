// Attention of a batch's rows over the 4-bit cache (the layout: nh_kv4.h).
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys j <= i of row i's
//   sequence; with a ring also j < sink or j > i - ring.
#include "nh_kv4_device.h"

namespace nh {

// One wavefront for each (row, head), 64 keys a step: a lane a key for the
// scores, a lane a dim (and each 64th on) for the sums.
template <int TYPE, int W>
__global__ __launch_bounds__(64) void k_kv4_attend(Kv4View c, Kv4AttendArgs a) {
    typedef typename Kv4Elem<TYPE>::T T;
    __shared__ float qs[W];
    __shared__ float ps[64];
    __shared__ const uint8_t* blks[64];
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y;
    const int kvh = head / (a.heads / c.heads);
    const int b = c.each ? row / c.each : kv4_entry(c.brow0, c.nb, row, lane);
    const int seq = c.bseq[b];
    const int i = c.len[seq] - c.brow0[b + 1] + row;
    const T* q = reinterpret_cast<const T*>(a.q) + row * a.ldq + (int64_t)head * c.dk;
    for (int d = lane; d < W; d += 64) qs[d] = d < c.dk ? Kv4Elem<TYPE>::get(q + d) : 0.0f;
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f, acc[W / 64] = {};
    const int mask = c.page() - 1, ng = c.groups();
    for (int j0 = 0; j0 <= i; j0 += 64) {
        if (a.ring && j0 >= a.sink && j0 + 63 <= i - a.ring) continue;
        const int j = j0 + lane;
        const bool seen = j <= i && (!a.ring || j < a.sink || j > i - a.ring);
        float s = -__builtin_inff();
        const int pg = seen ? kv4_page(c, seq, j) : -1;
        if (pg >= 0) {
            const uint8_t* blk = kv4_block(c, pg, a.layer, kvh);
            blks[lane] = blk;
            const int slot = j & mask;
            const uint32_t* codes = reinterpret_cast<const uint32_t*>(blk) + slot * (W / 8);
            const uint32_t* scales = reinterpret_cast<const uint32_t*>(blk + c.ks_off()) + slot * ng;
            s = 0.0f;
            for (int t = 0; t * 8 < c.dk; ++t) {
                const uint32_t w = codes[(t & 3) * (W / 32) + (t >> 2)], sc = scales[t * 8 / c.group];
                for (int e = 0; e < 8; ++e) {
                    const float k = __builtin_fmaf(kv4_step(sc), (float)((w >> (4 * ((e & 1) * 4 + (e >> 1)))) & 15u), kv4_low(sc));
                    s = t * 8 + e < c.dk ? __builtin_fmaf(qs[t * 8 + e], k, s) : s;
                }
            }
            s *= a.scale;
        }
        float most = s;
        for (int h = 1; h < 64; h <<= 1) most = fmaxf(most, lane_xor(most, h, lane));
        const float next = fmaxf(m, most);
        const float keep = m == next ? 1.0f : expf(m - next);
        const float p = pg >= 0 ? expf(s - next) : 0.0f;
        m = next;
        l = l * keep + p;
        ps[lane] = p;
        __syncthreads();
        for (int x = 0; x < W / 64; ++x) {
            const int d = 64 * x + lane, o = d & 15, n = (d & 63) >> 4;
            acc[x] *= keep;
            if (d >= c.dv) continue;
            for (int y = 0; y < 64; ++y) {
                const float w = ps[y];
                if (w == 0.0f) continue;
                const int slot = (j0 + y) & mask;
                const uint16_t code = reinterpret_cast<const uint16_t*>(blks[y] + c.v_off())
                    [(((slot >> 2) * 16 + o) * 2 * (W / 64) + ((slot >> 1) & 1) * (W / 64) + x) * 2 + (slot & 1)];
                const uint32_t sc = reinterpret_cast<const uint32_t*>(blks[y] + c.vs_off())[slot * ng + d / c.group];
                acc[x] = __builtin_fmaf(w, __builtin_fmaf(kv4_step(sc), (float)(code >> (4 * n) & 15), kv4_low(sc)), acc[x]);
            }
        }
        __syncthreads();
    }
    for (int h = 1; h < 64; h <<= 1) l += lane_xor(l, h, lane);
    T* out = reinterpret_cast<T*>(a.out) + row * a.ldo + (int64_t)head * c.dv;
    const float r = 1.0f / l;
    for (int x = 0; x < W / 64; ++x)
        if (64 * x + lane < c.dv) Kv4Elem<TYPE>::put(out + 64 * x + lane, acc[x] * r);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.heads + head] = m + logf(l);
}

size_t kv4_attend_ws(const Kv4View&, int, int, int, int) { return 0; }

template <int TYPE>
static hipError_t attend_typed(const Kv4View& c, const Kv4AttendArgs& a, hipStream_t s) {
    auto kern = c.width == 64 ? k_kv4_attend<TYPE, 64> : c.width == 128 ? k_kv4_attend<TYPE, 128> : k_kv4_attend<TYPE, 256>;
    hipLaunchKernelGGL(kern, dim3(c.rows, a.heads), dim3(64), 0, s, c, a);
    return hipGetLastError();
}

hipError_t launch_kv4_attend(const Kv4View& c, const Kv4AttendArgs& a, int, hipStream_t s) {
    return a.type == KV4_F32   ? attend_typed<KV4_F32>(c, a, s)
           : a.type == KV4_F16 ? attend_typed<KV4_F16>(c, a, s)
                               : attend_typed<KV4_BF16>(c, a, s);
}

}  // namespace nh
