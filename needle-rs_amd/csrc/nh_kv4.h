// The 4-bit key/value cache: its layout in HBM, what its kernels are given
// beside the view that the paged caches share (nh_kv.h), and their launchers.
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
// (page, layer, head) is page / 32 chunks of 32 positions, one after the other.
// A chunk, with W = width, NG = W / group and slot = position % 32, is what a
// wavefront of the attention kernel takes in one step, in the order in which its
// lanes hold it (lane = 16 kg + o, 16 bytes a lane and piece, so a piece is one
// load of 1 KiB):
//   key codes    W / 64 pieces: lane (o = slot % 16, kg), dword u = slot / 16
//                (W / 32) + j of the lane's W / 16 dwords holds dims 32 j + 8 kg + e
//                (e = 0 .. 7) at nibble (e % 2) 4 + e / 2
//   value codes  W / 64 pieces: lane (o, kg = slot / 4 % 4), half slot % 2 of dword u =
//                slot / 16 (W / 32) + (slot / 2 % 2) NB + b, NB = W / 64, holds dims
//                64 b + 32 (i / 2) + 2 o + i % 2 (i = 0 .. 3) at nibble i
//   key steps    32 x NG f16
//   key lows     32 x NG f16
//   value steps  f16 of (slot, g) at (slot / 4 NG + g) 4 + slot % 4
//   value lows   as the value steps
// Of a lane's 8 codes a dword, the two of a 16-bit half pair are one mask away
// from an MFMA operand (see the attention kernel).  No position shares a byte
// with another, so rows are written without reading their neighbours.
#pragma once

#include "nh_kv.h"

namespace nh {

constexpr int KV4_LANES = 16;

struct Kv4View : KvView {
    int width, group;
    int kernel;  // nh_kv4_debug_kernel
    __host__ __device__ int groups() const { return width / group; }
    // bytes of 32 positions, and of one (page, layer, head)
    __host__ __device__ uint32_t chunk() const { return 32u * (width + 8 * groups()); }
    __host__ __device__ size_t block() const { return (size_t)(page() / 32) * chunk(); }
    __host__ __device__ size_t page_bytes() const { return block() * heads * layers; }
};

// The chunks of 32 that positions pos .. pos + n - 1 lie in.
__host__ __device__ inline int kv4_chunks(int pos, int n) { return n ? ((pos + n - 1) >> 5) - (pos >> 5) + 1 : 0; }
// Runs of positions to move into fresh pages: positions src .. of sequence
// seq to positions dst .. counted from fresh page 0 of that sequence, whose
// ids are at state[fresh ..]; unit0: the first of the chunks that the run
// writes into, in the launch.
struct Kv4Runs {
    static constexpr int MAX = 160;
    int n;
    int seq[MAX], src[MAX], dst[MAX], count[MAX], fresh[MAX], unit0[MAX + 1];
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

hipError_t launch_kv4_runs(const Kv4View& c, const int* state, const Kv4Runs& r, hipStream_t s);
hipError_t launch_kv4_append(const Kv4View& c, const int* row0, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int type,
                             hipStream_t s);
// layer < 0: all, [layers][rows]; `rows` rows a layer in the output, this launch's from `row`.
hipError_t launch_kv4_read(const Kv4View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s);
// Bytes of workspace an attention call of the batch needs; row0: the host's copy
// of the sequences' first rows; longest: the batch's longest sequence.
size_t kv4_attend_ws(const Kv4View& c, const int* row0, int heads, int sink, int ring, int longest);
hipError_t launch_kv4_attend(const Kv4View& c, const int* row0, const Kv4AttendArgs& a, int longest, hipStream_t s);

}  // namespace nh
