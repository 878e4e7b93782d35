// Rotary positions: what the kernels that turn rows are given.
#pragma once

#include "nh_internal.h"

namespace nh {

struct RopeView {
    const uint64_t* turns;  // [pairs] turns a position, as fractions of 2^64
    double amplitude;
    int pairs, interleaved;
};

// Rows [rows][heads][dim], an element of `type`; y may be x.
struct RopeRows {
    const void* x;
    void* y;
    int64_t ldx, ldy;  // elements from one row to the next
    int heads;
};
struct RopeArgs {
    RopeView r;
    const int32_t* pos;  // [rows]
    RopeRows q, k;       // k.heads 0: q alone
    int64_t rows;
    int dim, transposed;
};

hipError_t launch_rope(const RopeArgs& a, int type, hipStream_t s);

}  // namespace nh

struct nh_rope {
    nh::RopeView v{};
    int device = 0;
    uint64_t* turns = nullptr;
};
