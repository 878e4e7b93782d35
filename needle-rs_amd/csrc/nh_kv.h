// What the paged key/value caches share whatever they hold: the view of pages
// and batch that their kernels are given, the patches of the device's state,
// whole pages copied.  The formats: nh_kv4.h, nh_kv8.h.
#pragma once

#include "nh_internal.h"

namespace nh {

enum KvType { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };  // NH_F32 ..

struct KvEntry {
    int seq, row0, row1, len;
};

struct KvView {
    uint8_t* data;       // [pages][layers][heads] blocks
    const int* table;    // [seqs][table_ld] page ids
    const int* batch;    // [nb] of (sequence, first row, end row, length): KvEntry; its shape 4 words before
    int table_ld, pages, layers, heads, dk, dv, page_log2;
    int nb, rows, each;  // the batch; each: rows of every sequence when they are equal, else 0
    int shape[2];        // names the sequences' numbers of rows, in order; (0, 0): no batch
    __host__ __device__ int page() const { return 1 << page_log2; }
};

// Values of the device's int32 state: (index, value) pairs.
struct KvPatch {
    static constexpr int MAX = 480;
    int n;
    uint32_t at[MAX];
    int v[MAX];
};
// Pages to copy whole.
struct KvPairs {
    static constexpr int MAX = 480;
    int n;
    int from[MAX], to[MAX];
};
// Rows to read: entry i is rows row0[i] .. row0[i + 1] - 1 of the output,
// positions pos[i] .. of sequence seq[i]; unit0: the first of the chunks that
// they lie in, in the launch.
struct KvSpans {
    static constexpr int MAX = 240;
    int n;
    int seq[MAX], pos[MAX], row0[MAX + 1], unit0[MAX + 1];
};

// Results of `splits` ranges of keys to join: ws holds, range by range, (maximum,
// sum) of each of n (row, head), base 2, then their sums of weighted values.
constexpr int KV_SPLITS = 512;  // at most
constexpr int KV_FEW = 8;       // ranges that the join takes a thread an element
struct KvJoin {
    void* out;
    float* lse;  // or null
    const float* ws;
    int64_t n, ldo;
    int heads, dv, splits;
};

hipError_t launch_kv_join(const KvJoin& a, int type, hipStream_t s);
hipError_t launch_kv_patch(int* state, const KvPatch& p, hipStream_t s);
hipError_t launch_kv_pairs(uint8_t* data, size_t page_bytes, const KvPairs& p, hipStream_t s);

}  // namespace nh
