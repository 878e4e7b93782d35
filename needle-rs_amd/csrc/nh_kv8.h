// The 8-bit key/value cache: its layout in HBM, what its kernels are given
// beside the view that the paged caches share (nh_kv.h), and their launchers.
//
// Format.  Keys and values are whole numbers -127 .. 127 times an f32 step for
// each block of 16 positions and head (one for the keys, one for the values):
// step = max|x| f32(1/127) of the rows that the block's first position came with,
// code = rint(x (1 / step)), all in f32; rows that join the block double the step
// until it is their own max|x| f32(1/127) at least, and the codes that were there are
// halved as often (ties to even).  A step below 2^-120 counts as 0, and so do its
// codes.  A row with a NaN or an infinity is left out of the step and marked.
//
// A power of two between two steps of a block keeps what it holds within a step
// of what was stored however often it grows (a quarter, an eighth .. of the
// half a step that each rounding may take); steps that followed the rows
// exactly would round anew, by half a step, with every growth.
//
// Rows are stored WK and WV wide, (64, 64), (128, 128), (192, 128) or (256, 256),
// the first that holds both head dims.  A page holds `page` positions of every
// layer and head; the block of one (page, layer, head) is page / 64 chunks of 64
// positions.  A chunk is what a wavefront of the attention kernel takes in one
// step, in the order in which its lanes hold it (lane = 16 kg + o, 16 bytes a lane
// and piece, so a piece is one load of 1 KiB); a byte is code + 128:
//   keys    4 WK / 64 pieces: piece t WK / 64 + j, lane (o, kg) holds position 16 t +
//           o, dims 64 j + 16 kg + 0 .. 15
//   values  WV / 16 pieces: piece n, lane (o, kg) holds dim 16 n + o of positions
//           16 t + 4 kg + r at byte 4 t + r
//   record  the blocks' steps, 4 f32 of the keys and 4 of the values, then their
//           marked rows, a bit each, 4 u16 of the keys and 4 of the values (128 bytes)
#pragma once

#include "nh_kv.h"
#include "nh_rope.h"

namespace nh {

constexpr int KV8_CHUNK = 64;
constexpr int64_t KV8_THREADS = 0xffffffff;  // that a launch can have in x

struct Kv8Record {
    float ks[4], vs[4];
    uint16_t kbad[4], vbad[4];
    uint32_t pad[20];
};

struct Kv8View : KvView {
    int wk, wv;
    int ask;     // the batch's rows are queries alone: each sees its whole sequence
    int kernel;  // nh_kv8_debug_kernel
    // bytes of 64 positions, and of one (page, layer, head)
    __host__ __device__ uint32_t chunk() const { return 64u * (wk + wv) + (uint32_t)sizeof(Kv8Record); }
    __host__ __device__ size_t block() const { return (size_t)(page() / KV8_CHUNK) * chunk(); }
};

// The chunks of 64 that positions pos .. pos + n - 1 lie in.
__host__ __device__ inline int kv8_chunks(int pos, int n) { return n ? ((pos + n - 1) >> 6) - (pos >> 6) + 1 : 0; }

struct Kv8Append {
    const void *k, *v;
    int64_t ldk, ldv;
    int layer;
    // keys turned, and queries with them (r.turns null: none)
    RopeView r;
    const int32_t* pos;  // null: the rows' positions
    RopeRows q;
};

struct Kv8AttendArgs {
    const void* q;
    void* out;
    float* lse;  // or null
    int type, layer, heads, sink, ring;
    int64_t ldq, ldo;  // elements from one row to the next
    float scale;
    void* ws;
};

hipError_t launch_kv8_append(const Kv8View& c, const int* row0, const Kv8Append& a, int type, hipStream_t s);
// layer < 0: all, [layers][rows]; `rows` rows a layer in the output, this launch's from `row`.
hipError_t launch_kv8_read(const Kv8View& c, int layer, const KvSpans& p, int64_t rows, int64_t row, void* k, void* v,
                           int type, hipStream_t s);
// Attention by the kernel of many rows (f16 and bf16, dims up to 128): `tiles`
// workgroups of KP8_ROWS rows a range of keys.
constexpr int KP8_ROWS = 256;
struct KaPlan;
hipError_t launch_kv8_prompt(const Kv8View& c, const Kv8AttendArgs& a, const KaPlan& plan, int64_t tiles, hipStream_t s);
// Bytes of workspace an attention call of the batch needs; row0: the host's copy
// of the sequences' first rows; longest: the batch's longest sequence.
size_t kv8_attend_ws(const Kv8View& c, const int* row0, int heads, int sink, int ring, int longest);
hipError_t launch_kv8_attend(const Kv8View& c, const int* row0, const Kv8AttendArgs& a, int longest, hipStream_t s);

}  // namespace nh
