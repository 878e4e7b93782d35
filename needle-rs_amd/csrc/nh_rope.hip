// Rotary positions: rows of queries and keys turned, each pair of a head's first
// dims by its row's position times the pair's frequency.
//
//   y_a = x_a c - x_b s, y_b = x_b c + x_a s, (a, b) = (i, i + pairs) or
//   (2 i, 2 i + 1); transposed: s with the other sign, which is the gradient.
#include <algorithm>

#include "nh_kv_device.h"
#include "nh_rope_device.h"

namespace nh {

// A thread takes V pairs of one row (or V dims behind them, where they have to be
// copied) and works out their angles once for its share of the heads.
struct RopePlan {
    int units, turned;  // threads a row; of these the first `turned` have pairs
    int share;          // heads a thread takes
};

template <int TYPE, int V, bool INTER>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a, RopePlan p) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(V)));
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / p.units;
    const int u = (int)(i - row * p.units);
    if (row >= a.rows) return;
    const int h0 = blockIdx.y * p.share, h1 = min(h0 + p.share, a.q.heads + a.k.heads);
    const bool turns = u < p.turned;
    // The two vectors of a unit: pairs' firsts and seconds, 2 V dims in one piece, or V dims to copy.
    const int d0 = !turns ? 2 * a.r.pairs + (u - p.turned) * V : INTER ? u * 2 * V : u * V;
    const int d1 = !turns ? d0 : INTER ? d0 + V : d0 + a.r.pairs;
    float2 cs[V];
    if (turns) {
        const int pos = a.pos[row];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            cs[e] = rope_cos_sin(a.r.turns[u * V + e], pos, a.r.amplitude);
            if (a.transposed) cs[e].y = -cs[e].y;
        }
    }
    constexpr int U = 4;  // heads in flight
    for (int h = h0; h < h1; h += U) {
        Vec x0[U], x1[U];
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int hh = min(h + n, h1 - 1);
            const bool is_k = hh >= a.q.heads;
            const RopeRows& r = is_k ? a.k : a.q;
            const T* x = reinterpret_cast<const T*>(r.x) + row * r.ldx + (int64_t)(hh - (is_k ? a.q.heads : 0)) * a.dim;
            x0[n] = *reinterpret_cast<const Vec*>(x + d0);
            if (turns) x1[n] = *reinterpret_cast<const Vec*>(x + d1);
        }
#pragma unroll
        for (int n = 0; n < U; ++n) {
            const int hh = h + n;
            if (hh >= h1) break;
            const bool is_k = hh >= a.q.heads;
            const RopeRows& r = is_k ? a.k : a.q;
            T* y = reinterpret_cast<T*>(r.y) + row * r.ldy + (int64_t)(hh - (is_k ? a.q.heads : 0)) * a.dim;
            if (turns) {
                Vec y0, y1;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    // (interleaved: pair e is elements 2 e, 2 e + 1 of the two vectors in a row)
                    const T xa = !INTER ? x0[n][e] : 2 * e < V ? x0[n][(2 * e) % V] : x1[n][(2 * e) % V];
                    const T xb = !INTER ? x1[n][e] : 2 * e + 1 < V ? x0[n][(2 * e + 1) % V] : x1[n][(2 * e + 1) % V];
                    const float2 z = rope_turn((float)xa, (float)xb, cs[e]);
                    if constexpr (!INTER) {
                        y0[e] = (T)z.x, y1[e] = (T)z.y;
                    } else {
                        if (2 * e < V) y0[(2 * e) % V] = (T)z.x; else y1[(2 * e) % V] = (T)z.x;
                        if (2 * e + 1 < V) y0[(2 * e + 1) % V] = (T)z.y; else y1[(2 * e + 1) % V] = (T)z.y;
                    }
                }
                *reinterpret_cast<Vec*>(y + d0) = y0;
                *reinterpret_cast<Vec*>(y + d1) = y1;
            } else
                *reinterpret_cast<Vec*>(y + d0) = x0[n];
        }
    }
}

template <int TYPE, int V>
static hipError_t rope_wide(const RopeArgs& a, hipStream_t s) {
    const int heads = a.q.heads + a.k.heads;
    const bool copies = a.q.x != a.q.y || (a.k.heads && a.k.x != a.k.y);
    RopePlan p;
    p.turned = a.r.pairs / V;
    p.units = p.turned + (copies ? (a.dim - 2 * a.r.pairs) / V : 0);
    const int64_t threads = a.rows * p.units;
    // Heads are shared out until every SIMD has four wavefronts: angles are worked
    // out again for each share, so no further.
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>((heads + 3) / 4, 262144 / std::max<int64_t>(threads, 1)));
    p.share = (int)((heads + shares - 1) / shares);
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (heads + p.share - 1) / p.share);
    if (a.r.interleaved)
        hipLaunchKernelGGL((k_rope<TYPE, V, true>), grid, dim3(256), 0, s, a, p);
    else
        hipLaunchKernelGGL((k_rope<TYPE, V, false>), grid, dim3(256), 0, s, a, p);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t rope_typed(const RopeArgs& a, hipStream_t s) {
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    auto four = [&](const RopeRows& r) {
        return !r.heads || ((uintptr_t)r.x % (4 * es) == 0 && (uintptr_t)r.y % (4 * es) == 0 && r.ldx % 4 == 0 && r.ldy % 4 == 0);
    };
    if (a.r.pairs % 4 == 0 && a.dim % 4 == 0 && four(a.q) && four(a.k)) return rope_wide<TYPE, 4>(a, s);
    return rope_wide<TYPE, 1>(a, s);
}

hipError_t launch_rope(const RopeArgs& a, int type, hipStream_t s) {
    return type == KV_F32   ? rope_typed<KV_F32>(a, s)
           : type == KV_F16 ? rope_typed<KV_F16>(a, s)
                            : rope_typed<KV_BF16>(a, s);
}

}  // namespace nh
