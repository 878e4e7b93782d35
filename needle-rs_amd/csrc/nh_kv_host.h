// The host side that the paged caches share (nh_kv4.cpp, nh_kv8.cpp): pages in
// one HBM allocation, the book of who holds them (nh_kv4_book.h) and its mirror
// on the device.
//
// The mirror is an int32 array: the sequences' page ids, and the batch (its
// shape, its sequences, their rows and lengths).  The host keeps a copy of what
// it sent and sends what changed as kernel arguments, so a step of a decoding
// loop is one small launch, no host memory has to outlive the call, and every
// kernel after it on the stream sees the new state.  Append and attention read
// the batch from the mirror: captured in a graph, they follow the state that
// an extend outside the graph leaves if it has the shape that they were
// captured at, and do nothing under any other.
#pragma once

#include <algorithm>
#include <new>
#include <string>
#include <vector>

#include "../../include/needle_hip.h"
#include "nh_kv.h"
#include "nh_kv4_book.h"

namespace nh {

struct KvHost {
    Kv4Book book;
    KvView* view = nullptr;  // the cache's own
    size_t page_bytes = 0;
    int device = 0;
    int seqs = 0;
    uint8_t* data = nullptr;
    int* state = nullptr;
    size_t n_state = 0;
    // where the mirror's parts start
    size_t o_table = 0, o_batch = 0, o_fresh = 0;
    std::vector<int> sent;  // the mirror's values but the tables' and the fresh ids'
    KvPatch patch{};        // values not sent yet
    bool asks = false;      // the batch's rows are queries alone (ask), not positions of the cache
};

namespace kv {

inline int fail(int code, const std::string& msg) {
    set_error(msg);
    return code;
}

inline int hip_fail(hipError_t e, const char* what) {
    return fail(NH_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

#define NH_TRY(call, what)                                       \
    do {                                                         \
        hipError_t e_ = (call);                                  \
        if (e_ != hipSuccess) return nh::kv::hip_fail(e_, what); \
    } while (0)

// No exception leaves an entry point.
template <class F>
int guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return fail(NH_ENOMEM, "out of host memory");
    } catch (...) {
        return fail(NH_EINVAL, "unexpected failure");
    }
}

// The handle is there and belongs to the current device.
inline int check(const KvHost* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (!ready()) return fail(NH_ESTATE, "nh_init has not been called");
    int dev = -1;
    NH_TRY(hipGetDevice(&dev), "hipGetDevice");
    if (dev != c->device) return fail(NH_EINVAL, "the cache belongs to another device than the current one");
    return NH_OK;
}

// A call that changes the book cannot be recorded: a replay would not repeat it.
inline int check_eager(hipStream_t st) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    NH_TRY(hipStreamIsCapturing(st, &s), "hipStreamIsCapturing");
    if (s != hipStreamCaptureStatusNone)
        return fail(NH_EINVAL, "the cache's pages change on the host: not in a captured graph");
    return NH_OK;
}

inline int refused(const KvHost* c, int code) { return fail(code, c->book.why); }

inline bool known_type(int t) { return t == NH_F32 || t == NH_F16 || t == NH_BF16; }

inline int flush(KvHost* c, hipStream_t st) {
    if (!c->patch.n) return NH_OK;
    const hipError_t e = launch_kv_patch(c->state, c->patch, st);
    c->patch.n = 0;
    NH_TRY(e, "cache state");
    return NH_OK;
}

inline int put(KvHost* c, size_t at, int v, hipStream_t st) {
    if (c->patch.n == KvPatch::MAX)
        if (int rc = flush(c, st)) return rc;
    c->patch.at[c->patch.n] = (uint32_t)at;
    c->patch.v[c->patch.n++] = v;
    return NH_OK;
}

// A value of the mirror that the host remembers: sent when it changed.
inline int put_changed(KvHost* c, size_t at, int v, hipStream_t st) {
    int& old = c->sent[at - c->o_batch];
    if (old == v) return NH_OK;
    old = v;
    return put(c, at, v, st);
}

// The device's table of a sequence up to date (queued; flush sends it).
inline int sync_table(KvHost* c, int s, hipStream_t st) {
    Kv4Book::Seq& q = c->book.seqs[s];
    for (; q.synced < (int)q.table.size(); ++q.synced)
        if (int rc = put(c, c->o_table + (size_t)s * c->view->table_ld + q.synced, q.table[q.synced], st)) return rc;
    return NH_OK;
}

inline int copy_pages(KvHost* c, const std::vector<std::pair<int, int>>& copies, hipStream_t st) {
    KvPairs p;
    for (size_t i = 0; i < copies.size();) {
        p.n = 0;
        while (i < copies.size() && p.n < KvPairs::MAX) {
            p.from[p.n] = copies[i].first;
            p.to[p.n++] = copies[i++].second;
        }
        NH_TRY(launch_kv_pairs(c->data, c->page_bytes, p, st), "cache page copy");
    }
    return NH_OK;
}

// The shape that the device's batch has (queued): a launch made for another
// one, replayed from a captured step, touches no page.
inline int put_shape(KvHost* c, int lo, int hi, hipStream_t st) {
    if (int rc = put_changed(c, c->o_batch, lo, st)) return rc;
    return put_changed(c, c->o_batch + 1, hi, st);
}
// Before pages are handed out under no batch (one that is over, or none).
inline int drop_batch(KvHost* c, hipStream_t st) {
    if (!c->book.batch_seq.empty()) return NH_OK;
    if (int rc = put_shape(c, 0, 0, st)) return rc;
    return flush(c, st);
}
// The shape of n sequences' rows: a 64-bit FNV-1a hash, (0, 0) left out.  Two
// shapes of one hash would share a grid, not run out of bounds: every kernel
// checks its rows and pages besides.
inline void shape_of_rows(const int* rows, int n, int* shape) {
    uint64_t h = 0xcbf29ce484222325ull;
    for (int i = 0; i < n; ++i)
        for (int k = 0; k < 32; k += 8) h = (h ^ ((uint32_t)rows[i] >> k & 255u)) * 0x100000001b3ull;
    if (!h) h = 1;
    shape[0] = (int)(uint32_t)h;
    shape[1] = (int)(uint32_t)(h >> 32);
}

// The batch of the last extend, as the kernels see it.
inline int check_batch(const KvHost* c, int layer) {
    if (layer < 0 || layer >= c->view->layers) return fail(NH_EINVAL, "no such layer");
    if (c->book.batch_seq.empty() && c->view->nb != 0)
        return fail(NH_EINVAL, "no batch: its sequences changed since the last extend");
    return NH_OK;
}
inline int longest(const KvHost* c) {
    int n = 0;
    for (int s : c->book.batch_seq) n = std::max(n, c->book.seqs[s].len);
    return n;
}

// What a new cache's sequences and pages have to satisfy, before any device work.
inline int check_new(int layers, int kv_heads, int qk_dim, int v_dim, int page, int pages, int seqs, int cap) {
    if (layers < 1 || layers > 4096 || kv_heads < 1 || kv_heads > 1024)
        return fail(NH_EINVAL, "1 to 4096 layers of 1 to 1024 key/value heads");
    if (qk_dim < 1 || qk_dim > 256 || v_dim < 1 || v_dim > 256) return fail(NH_EINVAL, "head dims are 1 to 256");
    if (pages < 1 || pages > (1 << 28)) return fail(NH_EINVAL, "1 to 2^28 pages");
    if (seqs < 1 || seqs > 65536) return fail(NH_EINVAL, "1 to 65536 sequences");
    if (cap < 1 || cap > (1 << 30)) return fail(NH_EINVAL, "a sequence's capacity is 1 to 2^30 positions");
    const int64_t ld = ((int64_t)cap + page - 1) / page;
    if (ld * seqs + 4 * (int64_t)seqs + 8 + pages > (int64_t)UINT32_MAX / 4)
        return fail(NH_EINVAL, "the sequences' page tables are too large");
    return NH_OK;
}

// The view's sizes and the memory of a cache whose page takes c->page_bytes.
inline int allocate(KvHost* c, int layers, int kv_heads, int qk_dim, int v_dim, int page, int pages, int seqs, int cap) {
    NH_TRY(hipGetDevice(&c->device), "hipGetDevice");
    KvView& v = *c->view;
    v.layers = layers, v.heads = kv_heads, v.dk = qk_dim, v.dv = v_dim;
    v.pages = pages;
    v.table_ld = (int)(((int64_t)cap + page - 1) / page);
    c->seqs = seqs;
    c->book.init(page, pages, seqs, cap);
    c->o_table = 0;
    c->o_batch = ((size_t)v.table_ld * seqs + 3) / 4 * 4;  // the shape, then the entries, 16 bytes each
    c->o_fresh = c->o_batch + 4 + 4 * (size_t)seqs;
    c->n_state = c->o_fresh + pages;
    c->sent.assign(c->o_fresh - c->o_batch, 0);
    const size_t bytes = (size_t)pages * c->page_bytes;
    hipError_t e = hipMalloc(&c->data, bytes);
    if (e == hipSuccess) e = hipMalloc(&c->state, c->n_state * 4);
    if (e == hipSuccess) e = hipMemset(c->data, 0, bytes);
    if (e == hipSuccess) e = hipMemset(c->state, 0, c->n_state * 4);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (c->data) hipFree(c->data);
        if (c->state) hipFree(c->state);
        (void)hipGetLastError();  // an allocation that failed is this call's error alone
        return fail(NH_ENOMEM, std::string("cache allocation: ") + hipGetErrorString(e));
    }
    v.data = c->data;
    v.table = c->state + c->o_table;
    v.batch = c->state + c->o_batch + 4;
    return NH_OK;
}

inline void release(KvHost* c) {
    // A cache may be collected while this thread captures a graph of other
    // work: in the relaxed mode the release does not end that capture.
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    if (c->data) hipFree(c->data);
    if (c->state) hipFree(c->state);
    if (relaxed) hipThreadExchangeStreamCaptureMode(&mode);
}

// ---- the calls on sequences, as the entry points make them ----------------
inline int64_t bytes(const KvHost* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return (int64_t)((size_t)c->view->pages * c->page_bytes + c->n_state * 4);
}

inline int free_pages(const KvHost* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return (int)c->book.free_pages.size();
}

inline int seq_new(KvHost* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    const int s = c->book.new_seq();
    return s < 0 ? refused(c, s) : s;
}

inline int seq_len(const KvHost* c, int seq) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (!c->book.live(seq)) return fail(NH_EINVAL, "no such sequence");
    return c->book.seqs[seq].len;
}

inline int seq_free(KvHost* c, int seq) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return guarded([&]() -> int {
        const int rc = c->book.free_seq(seq);
        return rc ? refused(c, rc) : NH_OK;
    });
}

inline int seq_truncate(KvHost* c, int seq, int len) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return guarded([&]() -> int {
        const int rc = c->book.truncate(seq, len);
        return rc ? refused(c, rc) : NH_OK;
    });
}

inline int seq_fork(KvHost* c, int seq, int n, int* branches) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (n < 0 || (n > 0 && !branches)) return fail(NH_EINVAL, "bad arguments");
    return guarded([&]() -> int {
        const int rc = c->book.fork(seq, n, branches);
        return rc ? refused(c, rc) : NH_OK;
    });
}

inline int seq_copy(KvHost* c, int seq, hipStream_t st) {
    if (int rc = check(c)) return rc;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        std::vector<std::pair<int, int>> copies;
        int to = -1;
        if (int rc = c->book.copy(seq, &to, &copies)) return refused(c, rc);
        int rc = drop_batch(c, st);
        if (!rc) rc = copy_pages(c, copies, st);
        if (rc) {
            c->book.free_seq(to);
            return rc;
        }
        return to;
    });
}

// The device's batch: n sequences with rows[i] rows each, as the book has it.
inline int put_batch(KvHost* c, const int* seqs, const int* rows, int n, hipStream_t st) {
    const std::vector<int>& row0 = c->book.batch_row0;
    KvView& v = *c->view;
    v.nb = n;
    v.rows = row0.back();
    v.each = n ? rows[0] : 0;
    shape_of_rows(rows, n, v.shape);
    // (a step captured for rows of the cache is no step for queries alone)
    if (c->asks) v.shape[1] = ~v.shape[1];
    if (int rc = put_shape(c, v.shape[0], v.shape[1], st)) return rc;
    for (int i = 0; i < n; ++i) {
        if (int rc = sync_table(c, seqs[i], st)) return rc;
        const int entry[4] = {seqs[i], row0[i], row0[i + 1], c->book.seqs[seqs[i]].len};
        for (int k = 0; k < 4; ++k)
            if (int rc = put_changed(c, c->o_batch + 4 + 4 * (size_t)i + k, entry[k], st)) return rc;
        if (rows[i] != rows[0]) v.each = 0;
    }
    return flush(c, st);
}

inline int extend(KvHost* c, const int* seqs, const int* rows, int n, hipStream_t st) {
    if (int rc = check(c)) return rc;
    if (n < 0 || (n > 0 && (!seqs || !rows))) return fail(NH_EINVAL, "bad arguments");
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        std::vector<std::pair<int, int>> copies;
        if (int rc = c->book.extend(seqs, rows, n, &copies)) return refused(c, rc);
        // (the book has changed: a launch that fails from here on leaves the
        // device behind, as any failed launch does, and the caller frees the cache)
        c->asks = false;
        if (int rc = copy_pages(c, copies, st)) return rc;
        return put_batch(c, seqs, rows, n, st);
    });
}

inline int rows(const KvHost* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return c->book.batch_row0.back();
}

// The rows of a read, as spans whose units(pos, rows) chunks a launch takes at
// a time; returns the rows.
template <class Units, class Launch>
int read(KvHost* c, int layer, const int* seqs, const int* pos, const int* n_rows, int n, const void* k, const void* v,
         int type, hipStream_t st, Units units, Launch launch) {
    if (int rc = check(c)) return rc;
    if (layer < -1 || layer >= c->view->layers) return fail(NH_EINVAL, "no such layer");
    if (n < 0 || (n > 0 && (!seqs || !pos || !n_rows))) return fail(NH_EINVAL, "bad arguments");
    if (!known_type(type)) return fail(NH_EINVAL, "no such type");
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (!c->book.live(seqs[i])) return fail(NH_EINVAL, "no such sequence");
        if (pos[i] < 0 || n_rows[i] < 0 || pos[i] > c->book.seqs[seqs[i]].len - n_rows[i])
            return fail(NH_EINVAL, "the positions are not within the sequence");
        total += n_rows[i];
    }
    if (total == 0) return 0;
    if (total > INT32_MAX) return fail(NH_EINVAL, "too many rows");
    if (!k || !v) return fail(NH_EINVAL, "null argument");
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        for (int i = 0; i < n; ++i)
            if (int rc = sync_table(c, seqs[i], st)) return rc;
        if (int rc = flush(c, st)) return rc;
        KvSpans p;
        int64_t row = 0;
        for (int i = 0; i < n;) {
            p.n = 0;
            p.row0[0] = p.unit0[0] = 0;
            for (; i < n && p.n < KvSpans::MAX; ++i) {
                if (!n_rows[i]) continue;
                p.seq[p.n] = seqs[i];
                p.pos[p.n] = pos[i];
                p.row0[p.n + 1] = p.row0[p.n] + n_rows[i];
                p.unit0[p.n + 1] = p.unit0[p.n] + units(pos[i], n_rows[i]);
                ++p.n;
            }
            if (!p.n) break;
            NH_TRY(launch(p, total, row), "cache read");
            row += p.row0[p.n];
        }
        return (int)total;
    });
}

// What an attention call has to satisfy.
inline int check_attend(const KvHost* c, int layer, int heads, int sink, int ring) {
    if (int rc = check_batch(c, layer)) return rc;
    if (heads < 1 || heads % c->view->heads != 0 || heads / c->view->heads > 1024)
        return fail(NH_EINVAL, "the query heads are 1 to 1024 for each key/value head");
    if (sink < 0 || ring < 0) return fail(NH_EINVAL, "sink and ring are not negative");
    return NH_OK;
}

}  // namespace kv
}  // namespace nh
