// Device helpers of the paged caches' kernels, whatever the pages hold.
#pragma once

#include "nh_device.h"
#include "nh_kv.h"

namespace nh {

// Elements by type tag (KvType), widened to f32.
template <int TYPE>
struct KvElem;
template <>
struct KvElem<KV_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(const T* p) { return *p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = v; }
};
template <>
struct KvElem<KV_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = (_Float16)v; }
};
template <>
struct KvElem<KV_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(const T* p) { return (float)*p; }
    static __device__ __forceinline__ void put(T* p, float v) { *p = (__bf16)v; }
};

// The entry whose units (ascending, from first[i]) hold `unit`; the wavefront
// together, unit the same in every lane.
__device__ __forceinline__ int kv_span(const int* __restrict__ first, int n, int unit, int lane) {
    int b = 0;
    for (int i = 0; i < n; i += 64) b += __popcll(__ballot(i + lane < n && first[i + lane + 1] <= unit));
    return b < n ? b : n - 1;
}
// The batch entry whose units(entry) hold `unit`, which becomes that entry's own;
// c.nb past the last.  The wavefront together.
template <class F>
__device__ __forceinline__ int kv_find(const KvView& c, int& unit, int lane, F units) {
    int b = 0;
    for (int i = 0; i < c.nb; i += 64) {
        int sum = 0;
        if (i + lane < c.nb) {
            const int4 e = reinterpret_cast<const int4*>(c.batch)[i + lane];
            sum = units(KvEntry{e.x, e.y, e.z, e.w});
        }
#pragma unroll
        for (int h = 1; h < 64; h <<= 1) {
            const int x = __shfl_up(sum, h, 64);
            if (lane >= h) sum += x;
        }
        const int skip = __popcll(__ballot(sum <= unit && i + lane < c.nb));
        const int last = __shfl(sum, skip ? skip - 1 : 0, 64);
        b += skip;
        if (skip) unit -= last;
        if (skip < 64) break;
    }
    unit = __builtin_amdgcn_readfirstlane(unit);
    return __builtin_amdgcn_readfirstlane(b);
}
// The batch on the device is of the rows that this launch was made for: not so
// where a captured launch is replayed after an extend of other rows, or when
// the batch is over, whose grid and plan fit nothing that is there.
__device__ __forceinline__ bool kv_current(const KvView& c) {
    const int2 s = *reinterpret_cast<const int2*>(c.batch - 4);
    return (s.x == c.shape[0]) & (s.y == c.shape[1]);
}
__device__ __forceinline__ KvEntry kv_batch(const KvView& c, int b) {
    const int4 e = reinterpret_cast<const int4*>(c.batch)[b];
    return KvEntry{e.x, e.y, e.z, e.w};
}

// Where position `pos` of sequence `seq` lies: its page id, or -1 outside the
// table (a state that no extend leaves).
__device__ __forceinline__ int kv_page(const KvView& c, int seq, int pos) {
    if ((unsigned)(pos >> c.page_log2) >= (unsigned)c.table_ld) return -1;
    const int pg = c.table[(size_t)seq * c.table_ld + (pos >> c.page_log2)];
    return (unsigned)pg < (unsigned)c.pages ? pg : -1;
}

}  // namespace nh
