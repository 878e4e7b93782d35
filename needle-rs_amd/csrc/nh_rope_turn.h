// Rows of queries and keys turned: what one thread does, for the kernel that
// turns rows alone and for the cache's append.
#pragma once

#include "nh_kv_device.h"
#include "nh_rope_device.h"

namespace nh {

// A thread takes V pairs of one row (or V dims behind them, where they have to be
// copied) and works out their angles once for its share of the heads.
struct RopePlan {
    int units, turned;  // threads a row; of these the first `turned` have pairs
    int share;          // heads a thread takes
};

// Unit u of row `row`, at position pos: heads h0 .. h1 - 1 of the queries' and then the keys'.
template <int TYPE, int V, bool INTER>
__device__ __forceinline__ void rope_rows(const RopeArgs& a, const RopePlan& p, int64_t row, int u, int pos, int h0, int h1) {
    typedef typename KvElem<TYPE>::T T;
    typedef T Vec __attribute__((ext_vector_type(V)));
    const bool turns = u < p.turned;
    // The two vectors of a unit: pairs' firsts and seconds, 2 V dims in one piece, or V dims to copy.
    const int d0 = !turns ? 2 * a.r.pairs + (u - p.turned) * V : INTER ? u * 2 * V : u * V;
    const int d1 = !turns ? d0 : INTER ? d0 + V : d0 + a.r.pairs;
    float2 cs[V];
    if (turns) {
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

// Threads a row, of V pairs each.
inline RopePlan rope_plan(const RopeArgs& a, int v) {
    const bool copies = (a.q.heads && a.q.x != a.q.y) || (a.k.heads && a.k.x != a.k.y);
    RopePlan p;
    p.turned = a.r.pairs / v;
    p.units = p.turned + (copies ? (a.dim - 2 * a.r.pairs) / v : 0);
    p.share = a.q.heads + a.k.heads;
    return p;
}
// Whether rows of `es`-byte elements can be taken four pairs at a time.
inline bool rope_takes4(const RopeArgs& a, size_t es) {
    auto four = [&](const RopeRows& r) {
        return !r.heads || ((uintptr_t)r.x % (4 * es) == 0 && (uintptr_t)r.y % (4 * es) == 0 && r.ldx % 4 == 0 && r.ldy % 4 == 0);
    };
    return a.r.pairs % 4 == 0 && a.dim % 4 == 0 && four(a.q) && four(a.k);
}

}  // namespace nh
