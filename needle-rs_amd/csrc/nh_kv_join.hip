// Attention over a paged cache whose keys were taken in ranges: the ranges'
// partial results joined.
#include "nh_kv_device.h"

namespace nh {

// The key ranges' partial results of one (row, head), joined by a workgroup: the
// ranges' factors first, then a wavefront every fourth range, eight loads at a
// time (one wavefront in turn over the 256 ranges of a long sequence took 170 us).
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv_join(KvJoin a) {
    typedef typename KvElem<TYPE>::T T;
    __shared__ float f[KV_SPLITS], sv[4][256], st[4], ss[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t n = a.n, at = blockIdx.x;
    const int splits = a.splits;
    const float* ml = a.ws;
    const float* po = ml + 2 * n * splits + at * a.dv;
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
    for (int x = 0; x * 64 < a.dv; ++x) {
        const int d = x * 64 + lane;
        float v = 0.0f;
        for (int s0 = wave; s0 < splits; s0 += 32) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = s0 + 4 * k < splits && d < a.dv ? po[(s0 + 4 * k) * n * a.dv + d] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float g = s0 + 4 * k < splits ? f[s0 + 4 * k] : -1.0f;
                v = g < 0.0f ? v : __builtin_fmaf(y[k], g, v);
            }
        }
        sv[wave][d & 255] = v;
    }
    __syncthreads();
    if (tid < a.dv) {
        T* out = reinterpret_cast<T*>(a.out) + at / a.heads * a.ldo + at % a.heads * a.dv;
        const float v = (sv[0][tid] + sv[1][tid]) + (sv[2][tid] + sv[3][tid]);
        KvElem<TYPE>::put(out + tid, sum == 0.0f ? 0.0f : v / sum);  // (0: a row that sees no key)
    }
    if (a.lse && tid == 0) a.lse[at] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

// The same for few ranges, a thread an element of the output: many rows are many
// elements, and a workgroup a (row, head) would mostly wait for its barriers (32,768
// of two ranges).
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv_join_few(KvJoin a) {
    typedef typename KvElem<TYPE>::T T;
    const int splits = a.splits;
    const int64_t n = a.n, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n * a.dv) return;
    const int64_t at = i / a.dv;
    const int d = (int)(i - at * a.dv);
    const float* ml = a.ws;
    const float* po = ml + 2 * n * splits + i;
    float m[KV_FEW], l[KV_FEW], v[KV_FEW], top = -__builtin_inff();
#pragma unroll
    for (int s = 0; s < KV_FEW; ++s) {
        const int64_t x = s < splits ? s : 0;
        m[s] = s < splits ? ml[2 * (x * n + at)] : -__builtin_inff();
        l[s] = ml[2 * (x * n + at) + 1];
        v[s] = po[x * n * a.dv];
        top = fmaxf(top, m[s]);
    }
    const float zero = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int s = 0; s < KV_FEW; ++s) {
        const float g = __builtin_amdgcn_exp2f(m[s] - zero);
        const bool some = m[s] != -__builtin_inff();  // (a range without keys wrote no sums)
        sum = some ? __builtin_fmaf(l[s], g, sum) : sum;
        o = some ? __builtin_fmaf(v[s], g, o) : o;
    }
    KvElem<TYPE>::put(reinterpret_cast<T*>(a.out) + at / a.heads * a.ldo + at % a.heads * a.dv + d, sum == 0.0f ? 0.0f : o / sum);
    if (a.lse && d == 0) a.lse[at] = (top + __builtin_amdgcn_logf(sum)) * 0.69314718055994530942f;
}

hipError_t launch_kv_join(const KvJoin& a, int type, hipStream_t s) {
    const bool few = a.splits <= KV_FEW;
    const int64_t blocks = few ? (a.n * a.dv + 255) / 256 : a.n;
    if (a.splits > KV_SPLITS || blocks > 0x7fffffff) return hipErrorInvalidValue;
    auto kern = type == KV_F32   ? (few ? k_kv_join_few<KV_F32> : k_kv_join<KV_F32>)
                : type == KV_F16 ? (few ? k_kv_join_few<KV_F16> : k_kv_join<KV_F16>)
                                 : (few ? k_kv_join_few<KV_BF16> : k_kv_join<KV_BF16>);
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace nh
