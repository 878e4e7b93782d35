// The 4-bit key/value cache: its layout in HBM, what its kernels are given,
// and their launchers.
//
// Format.  A row of keys (or values) of one head is cut into groups of 32 or
// 64 along the head; per group low = f16(min), step = f16((max - min) *
// f32(1/15)) and codes rint((x - low) * (1 / step)) in 0 .. 15, all in f32
// without fused operations; the value held is low + step * code.  x is held
// to +-65504 (f16's range); a group with a NaN or an infinity stores step
// NaN, so it reads as NaN and touches no other group.
//
// Rows are stored `width` wide: 64, 128 or 256, the smallest that holds both
// head dims (dims past a head's own have code 0 and are never read out).
// A page holds `page` positions of every layer and head; the block of one
// (page, layer, head) is, with T = page, W = width and NG = W / group:
//   key codes    T x W / 2 bytes   dword (t, kg, j) at t W/2 + (kg W/32 + j) 4
//                                  holds dims 32 j + 8 kg + e (e = 0 .. 7) at
//                                  nibble (e % 2) 4 + e / 2
//   value codes  T x W / 2 bytes   ushort (t, o, b) holds dims 64 b + 16 i + o
//                                  (i = 0 .. 3) at nibble i; it is the half
//                                  t % 2 of dword ((t / 4) 16 + o) 2 NB +
//                                  (t / 2 % 2) NB + b, NB = W / 64
//   key steps    T x NG f16
//   key lows     T x NG f16
//   value steps  T x NG f16
//   value lows   f16 of (t, g) at (t / 4 NG + g) 4 + t % 4
// That is the order in which a wavefront's MFMA operands want them: 16 lanes
// (keys, or dims) by 4 lane groups kg, 8 codes of the summed index a dword,
// and the two codes of a 16-bit half pair are one mask away (see the attention
// kernel).  No position shares a byte with another, so rows are written
// without reading their neighbours.
#pragma once

#include "nh_internal.h"

namespace nh {

enum Kv4Type { KV4_F32 = 0, KV4_F16 = 1, KV4_BF16 = 2 };  // NH_F32 ..

constexpr int KV4_LANES = 16;

struct Kv4View {
    uint8_t* data;       // [pages][layers][heads] blocks
    const int* table;    // [seqs][table_ld] page ids
    const int* len;      // [seqs]
    const int* bseq;     // [nb] the batch's sequences
    const int* brow0;    // [nb + 1] their first rows
    int table_ld, pages, layers, heads, dk, dv, width, group, page_log2;
    int nb, rows, each;  // the batch; each: rows of every sequence when they are equal, else 0
    __host__ __device__ int page() const { return 1 << page_log2; }
    __host__ __device__ int groups() const { return width / group; }
    // bytes of one (page, layer, head)
    __host__ __device__ size_t block() const { return (size_t)page() * (width + 8 * groups()); }
    __host__ __device__ size_t page_bytes() const { return block() * heads * layers; }
    __host__ __device__ uint32_t v_off() const { return (uint32_t)page() * width / 2; }
    __host__ __device__ uint32_t ks_off() const { return (uint32_t)page() * width; }
    __host__ __device__ uint32_t kl_off() const { return (uint32_t)page() * (width + 2 * groups()); }
    __host__ __device__ uint32_t vs_off() const { return (uint32_t)page() * (width + 4 * groups()); }
    __host__ __device__ uint32_t vl_off() const { return (uint32_t)page() * (width + 6 * groups()); }
};

// Values of the device's int32 state: (index, value) pairs.
struct Kv4Patch {
    static constexpr int MAX = 480;
    int n;
    uint32_t at[MAX];
    int v[MAX];
};
// Pages to copy whole.
struct Kv4Pairs {
    static constexpr int MAX = 480;
    int n;
    int from[MAX], to[MAX];
};
// Rows to read: entry i is rows row0[i] .. row0[i + 1] - 1 of the output,
// positions pos[i] .. of sequence seq[i].
struct Kv4Spans {
    static constexpr int MAX = 255;
    int n;
    int seq[MAX], pos[MAX], row0[MAX + 1];
};
// Runs of positions to move into fresh pages: positions src .. of sequence
// seq to positions dst .. counted from fresh page 0 of that sequence, whose
// ids are at state[fresh ..]; row0: the run's first position in the launch.
struct Kv4Runs {
    static constexpr int MAX = 160;
    int n;
    int seq[MAX], src[MAX], dst[MAX], count[MAX], fresh[MAX], row0[MAX + 1];
};

struct Kv4AttendArgs {
    const void* q;
    void* out;
    float* lse;  // or null
    int type, layer, heads, sink, ring;
    int64_t ldq, ldo;  // elements from one row to the next
    float scale;
    void* ws;
};

hipError_t launch_kv4_patch(int* state, const Kv4Patch& p, hipStream_t s);
hipError_t launch_kv4_pairs(const Kv4View& c, const Kv4Pairs& p, hipStream_t s);
hipError_t launch_kv4_runs(const Kv4View& c, const int* state, const Kv4Runs& r, hipStream_t s);
hipError_t launch_kv4_append(const Kv4View& c, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int type,
                             hipStream_t s);
// layer < 0: all, [layers][rows]; `rows` rows a layer in the output, this launch's from `row`.
hipError_t launch_kv4_read(const Kv4View& c, int layer, const Kv4Spans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s);
// Bytes of workspace an attention call of the batch needs; row0: the host's copy
// of the sequences' first rows; longest: the batch's longest sequence.
size_t kv4_attend_ws(const Kv4View& c, const int* row0, int heads, int sink, int ring, int longest);
hipError_t launch_kv4_attend(const Kv4View& c, const int* row0, const Kv4AttendArgs& a, int longest, hipStream_t s);

}  // namespace nh
