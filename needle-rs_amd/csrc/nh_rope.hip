// Rotary positions: rows of queries and keys turned, each pair of a head's first
// dims by its row's position times the pair's frequency.
//
//   y_a = x_a c - x_b s, y_b = x_b c + x_a s, (a, b) = (i, i + pairs) or
//   (2 i, 2 i + 1); transposed: s with the other sign, which is the gradient.
//
// Bytes bound it: a thread takes four pairs of a row, works their angles out once (f64
// series, about 40 instructions a pair) and turns them in every head of its share, four
// heads' loads in flight.  6,001 rows of 32 + 8 heads of 128 in bf16 (123 MB) 25 us, 4.9
// TB/s; 4,096 rows of 24 + 24 heads of 96, 32 dims turned by neighbours, in place (76
// MB) 15.1, 5.0 TB/s; a copy of 1 GiB has 5.2.  8 rows: 3.0 to 3.4 us, a launch and
// three loads one after the other.
#include <algorithm>

#include "nh_rope_turn.h"

namespace nh {

template <int TYPE, int V, bool INTER>
__global__ __launch_bounds__(256) void k_rope(RopeArgs a, RopePlan p) {
    const int64_t i = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x, row = i / p.units;
    const int u = (int)(i - row * p.units);
    if (row >= a.rows) return;
    const int h0 = blockIdx.y * p.share;
    rope_rows<TYPE, V, INTER>(a, p, row, u, u < p.turned ? a.pos[row] : 0, h0, min(h0 + p.share, a.q.heads + a.k.heads));
}

template <int TYPE, int V>
static hipError_t rope_wide(const RopeArgs& a, hipStream_t s) {
    const int heads = a.q.heads + a.k.heads;
    RopePlan p = rope_plan(a, V);
    const int64_t threads = a.rows * p.units;
    // Heads are shared out until every SIMD has four wavefronts: angles are worked
    // out again for each share, so no further.
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(std::min((heads + 3) / 4, 65535), 262144 / std::max<int64_t>(threads, 1)));
    p.share = (int)((heads + shares - 1) / shares);
    // (a launch has fewer than 2^32 threads in x: beyond 2^30 they go on in z)
    const int64_t blocks = (threads + 255) / 256, x = std::min<int64_t>(blocks, 1 << 22);
    if (blocks > x * 65535) return hipErrorInvalidValue;
    const dim3 grid((unsigned)x, (heads + p.share - 1) / p.share, (unsigned)((blocks + x - 1) / std::max<int64_t>(x, 1)));
    if (a.r.interleaved)
        hipLaunchKernelGGL((k_rope<TYPE, V, true>), grid, dim3(256), 0, s, a, p);
    else
        hipLaunchKernelGGL((k_rope<TYPE, V, false>), grid, dim3(256), 0, s, a, p);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t rope_typed(const RopeArgs& a, hipStream_t s) {
    const size_t es = sizeof(typename KvElem<TYPE>::T);
    if (rope_takes4(a, es)) return rope_wide<TYPE, 4>(a, s);
    return rope_wide<TYPE, 1>(a, s);
}

hipError_t launch_rope(const RopeArgs& a, int type, hipStream_t s) {
    return type == KV_F32   ? rope_typed<KV_F32>(a, s)
           : type == KV_F16 ? rope_typed<KV_F16>(a, s)
                            : rope_typed<KV_BF16>(a, s);
}

}  // namespace nh
