// The C ABI of the 4-bit key/value cache (include/needle_hip.h): pages in one
// HBM allocation, the book of who holds them (nh_kv4_book.h) and its mirror
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
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/needle_hip.h"
#include "nh_kv4.h"
#include "nh_kv4_book.h"

struct nh_kv4 {
    nh::Kv4Book book;
    nh::Kv4View v{};
    int device = 0;
    int seqs = 0;
    uint8_t* data = nullptr;
    int* state = nullptr;
    size_t n_state = 0;
    // where the mirror's parts start
    size_t o_table = 0, o_batch = 0, o_fresh = 0;
    std::vector<int> sent;  // the mirror's values but the tables' and the fresh ids'
    nh::Kv4Patch patch{};   // values not sent yet
};

namespace {

int fail(int code, const std::string& msg) {
    nh::set_error(msg);
    return code;
}

int hip_fail(hipError_t e, const char* what) {
    return fail(NH_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

#define NH_TRY(call, what)                               \
    do {                                                 \
        hipError_t e_ = (call);                          \
        if (e_ != hipSuccess) return hip_fail(e_, what); \
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
int check(const nh_kv4* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    int dev = -1;
    NH_TRY(hipGetDevice(&dev), "hipGetDevice");
    if (dev != c->device) return fail(NH_EINVAL, "the cache belongs to another device than the current one");
    return NH_OK;
}

// A call that changes the book cannot be recorded: a replay would not repeat it.
int check_eager(hipStream_t st) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    NH_TRY(hipStreamIsCapturing(st, &s), "hipStreamIsCapturing");
    if (s != hipStreamCaptureStatusNone)
        return fail(NH_EINVAL, "the cache's pages change on the host: not in a captured graph");
    return NH_OK;
}

int refused(const nh_kv4* c, int code) { return fail(code, c->book.why); }

bool known_type(int t) { return t == NH_F32 || t == NH_F16 || t == NH_BF16; }

int flush(nh_kv4* c, hipStream_t st) {
    if (!c->patch.n) return NH_OK;
    const hipError_t e = nh::launch_kv4_patch(c->state, c->patch, st);
    c->patch.n = 0;
    NH_TRY(e, "kv4 state");
    return NH_OK;
}

int put(nh_kv4* c, size_t at, int v, hipStream_t st) {
    if (c->patch.n == nh::Kv4Patch::MAX)
        if (int rc = flush(c, st)) return rc;
    c->patch.at[c->patch.n] = (uint32_t)at;
    c->patch.v[c->patch.n++] = v;
    return NH_OK;
}

// A value of the mirror that the host remembers: sent when it changed.
int put_changed(nh_kv4* c, size_t at, int v, hipStream_t st) {
    int& old = c->sent[at - c->o_batch];
    if (old == v) return NH_OK;
    old = v;
    return put(c, at, v, st);
}

// The device's table of a sequence up to date (queued; flush sends it).
int sync_table(nh_kv4* c, int s, hipStream_t st) {
    nh::Kv4Book::Seq& q = c->book.seqs[s];
    for (; q.synced < (int)q.table.size(); ++q.synced)
        if (int rc = put(c, c->o_table + (size_t)s * c->v.table_ld + q.synced, q.table[q.synced], st)) return rc;
    return NH_OK;
}

int copy_pages(nh_kv4* c, const std::vector<std::pair<int, int>>& copies, hipStream_t st) {
    nh::Kv4Pairs p;
    for (size_t i = 0; i < copies.size();) {
        p.n = 0;
        while (i < copies.size() && p.n < nh::Kv4Pairs::MAX) {
            p.from[p.n] = copies[i].first;
            p.to[p.n++] = copies[i++].second;
        }
        NH_TRY(nh::launch_kv4_pairs(c->v, p, st), "kv4 page copy");
    }
    return NH_OK;
}

// The shape that the device's batch has (queued): a launch made for another
// one, replayed from a captured step, touches no page.
int put_shape(nh_kv4* c, int lo, int hi, hipStream_t st) {
    if (int rc = put_changed(c, c->o_batch, lo, st)) return rc;
    return put_changed(c, c->o_batch + 1, hi, st);
}
// Before pages are handed out under no batch (one that is over, or none).
int drop_batch(nh_kv4* c, hipStream_t st) {
    if (!c->book.batch_seq.empty()) return NH_OK;
    if (int rc = put_shape(c, 0, 0, st)) return rc;
    return flush(c, st);
}
// The shape of n sequences' rows: a 64-bit FNV-1a hash, (0, 0) left out.  Two
// shapes of one hash would share a grid, not run out of bounds: every kernel
// checks its rows and pages besides.
void shape_of_rows(const int* rows, int n, int* shape) {
    uint64_t h = 0xcbf29ce484222325ull;
    for (int i = 0; i < n; ++i)
        for (int k = 0; k < 32; k += 8) h = (h ^ ((uint32_t)rows[i] >> k & 255u)) * 0x100000001b3ull;
    if (!h) h = 1;
    shape[0] = (int)(uint32_t)h;
    shape[1] = (int)(uint32_t)(h >> 32);
}

// The batch of the last extend, as the kernels see it.
int check_batch(const nh_kv4* c, int layer) {
    if (layer < 0 || layer >= c->v.layers) return fail(NH_EINVAL, "no such layer");
    if (c->book.batch_seq.empty() && c->v.nb != 0)
        return fail(NH_EINVAL, "no batch: its sequences changed since the last extend");
    return NH_OK;
}

}  // namespace

extern "C" {

int nh_kv4_new(int layers, int kv_heads, int qk_dim, int v_dim, int group, int page, int pages, int seqs, int cap,
               nh_kv4** h) {
    if (!h) return fail(NH_EINVAL, "null argument");
    *h = nullptr;
    if (layers < 1 || layers > 4096 || kv_heads < 1 || kv_heads > 1024)
        return fail(NH_EINVAL, "1 to 4096 layers of 1 to 1024 key/value heads");
    if (qk_dim < 1 || qk_dim > 256 || v_dim < 1 || v_dim > 256) return fail(NH_EINVAL, "head dims are 1 to 256");
    if (group != 32 && group != 64) return fail(NH_EINVAL, "groups are 32 or 64 values");
    if (page != 32 && page != 64 && page != 128 && page != 256)
        return fail(NH_EINVAL, "a page holds 32, 64, 128 or 256 positions");
    if (pages < 1 || pages > (1 << 28)) return fail(NH_EINVAL, "1 to 2^28 pages");
    if (seqs < 1 || seqs > 65536) return fail(NH_EINVAL, "1 to 65536 sequences");
    if (cap < 1 || cap > (1 << 30)) return fail(NH_EINVAL, "a sequence's capacity is 1 to 2^30 positions");
    const int64_t ld = ((int64_t)cap + page - 1) / page;
    if (ld * seqs + 4 * (int64_t)seqs + 8 + pages > (int64_t)UINT32_MAX / 4)
        return fail(NH_EINVAL, "the sequences' page tables are too large");
    const int wide = std::max(qk_dim, v_dim), width = wide <= 64 ? 64 : wide <= 128 ? 128 : 256;
    if ((double)pages * page * layers * kv_heads * (width + 8 * (width / group)) > 0x1p46)
        return fail(NH_EINVAL, "the pages are larger than any device's memory");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    return guarded([&]() -> int {
        auto c = std::make_unique<nh_kv4>();
        NH_TRY(hipGetDevice(&c->device), "hipGetDevice");
        nh::Kv4View& v = c->v;
        v.width = width;
        v.group = group;
        v.layers = layers, v.heads = kv_heads, v.dk = qk_dim, v.dv = v_dim;
        v.page_log2 = page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : 8;
        v.pages = pages;
        v.table_ld = (int)ld;
        c->seqs = seqs;
        c->book.init(page, pages, seqs, cap);
        c->o_table = 0;
        c->o_batch = ((size_t)ld * seqs + 3) / 4 * 4;  // the shape, then the entries, 16 bytes each
        c->o_fresh = c->o_batch + 4 + 4 * (size_t)seqs;
        c->n_state = c->o_fresh + pages;
        c->sent.assign(c->o_fresh - c->o_batch, 0);
        const size_t bytes = (size_t)pages * v.page_bytes();
        hipError_t e = hipMalloc(&c->data, bytes);
        if (e == hipSuccess) e = hipMalloc(&c->state, c->n_state * 4);
        if (e == hipSuccess) e = hipMemset(c->data, 0, bytes);
        if (e == hipSuccess) e = hipMemset(c->state, 0, c->n_state * 4);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        if (e != hipSuccess) {
            if (c->data) hipFree(c->data);
            if (c->state) hipFree(c->state);
            (void)hipGetLastError();  // an allocation that failed is this call's error alone
            return fail(NH_ENOMEM, std::string("kv4 allocation: ") + hipGetErrorString(e));
        }
        v.data = c->data;
        v.table = c->state + c->o_table;
        v.batch = c->state + c->o_batch + 4;
        *h = c.release();
        return NH_OK;
    });
}

int nh_kv4_free(nh_kv4* c) {
    if (!c) return NH_OK;
    // A cache may be collected while this thread captures a graph of other
    // work: in the relaxed mode the release does not end that capture.
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    if (c->data) hipFree(c->data);
    if (c->state) hipFree(c->state);
    if (relaxed) hipThreadExchangeStreamCaptureMode(&mode);
    delete c;
    return NH_OK;
}

int64_t nh_kv4_bytes(const nh_kv4* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return (int64_t)((size_t)c->v.pages * c->v.page_bytes() + c->n_state * 4);
}

int nh_kv4_free_pages(const nh_kv4* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return (int)c->book.free_pages.size();
}

int nh_kv4_seq_new(nh_kv4* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    const int s = c->book.new_seq();
    return s < 0 ? refused(c, s) : s;
}

int nh_kv4_seq_len(const nh_kv4* c, int seq) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (!c->book.live(seq)) return fail(NH_EINVAL, "no such sequence");
    return c->book.seqs[seq].len;
}

int nh_kv4_seq_free(nh_kv4* c, int seq) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return guarded([&]() -> int {
        const int rc = c->book.free_seq(seq);
        return rc ? refused(c, rc) : NH_OK;
    });
}

int nh_kv4_seq_truncate(nh_kv4* c, int seq, int len) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return guarded([&]() -> int {
        const int rc = c->book.truncate(seq, len);
        return rc ? refused(c, rc) : NH_OK;
    });
}

int nh_kv4_seq_fork(nh_kv4* c, int seq, int n, int* branches) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (n < 0 || (n > 0 && !branches)) return fail(NH_EINVAL, "bad arguments");
    return guarded([&]() -> int {
        const int rc = c->book.fork(seq, n, branches);
        return rc ? refused(c, rc) : NH_OK;
    });
}

int nh_kv4_seq_copy(nh_kv4* c, int seq, void* stream) {
    if (int rc = check(c)) return rc;
    hipStream_t st = (hipStream_t)stream;
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

int nh_kv4_seq_compact(nh_kv4* c, const int* seqs, int n, const int* counts, const int* ranges, void* stream) {
    if (int rc = check(c)) return rc;
    if (n < 0 || (n > 0 && (!seqs || !counts))) return fail(NH_EINVAL, "bad arguments");
    for (int i = 0; i < n; ++i)
        if (counts[i] > 0 && !ranges) return fail(NH_EINVAL, "bad arguments");
    hipStream_t st = (hipStream_t)stream;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        nh::Kv4Book::Compaction p;
        if (int rc = c->book.compact(seqs, n, counts, ranges, &p)) return refused(c, rc);
        // The sources' tables and the fresh pages' ids, then the moves.
        std::vector<int> at(n, 0);
        int rc = NH_OK, fresh = 0;
        for (int i = 0; i < n && !rc; ++i) {
            at[i] = fresh;
            if (p.fresh[i].empty()) continue;
            rc = sync_table(c, seqs[i], st);
            for (int page : p.fresh[i])
                if (!rc) rc = put(c, c->o_fresh + fresh++, page, st);
        }
        if (!rc) rc = flush(c, st);
        nh::Kv4Runs r;
        r.n = 0;
        r.unit0[0] = 0;
        for (size_t m = 0; m < p.moves.size() && !rc; ++m) {
            const nh::Kv4Book::Move& mv = p.moves[m];
            r.seq[r.n] = seqs[mv.seq];
            r.src[r.n] = mv.src;
            r.dst[r.n] = mv.dst;
            r.count[r.n] = mv.count;
            r.fresh[r.n] = (int)c->o_fresh + at[mv.seq];
            r.unit0[r.n + 1] = r.unit0[r.n] + nh::kv4_chunks(mv.dst, mv.count);
            if (++r.n == nh::Kv4Runs::MAX || m + 1 == p.moves.size() || r.unit0[r.n] > (1 << 26)) {
                const hipError_t e = nh::launch_kv4_runs(c->v, c->state, r, st);
                if (e != hipSuccess) rc = hip_fail(e, "kv4 compaction");
                r.n = 0;
            }
        }
        if (rc) {
            c->book.give_back(p);
            return rc;
        }
        c->book.compacted(seqs, n, p);
        return drop_batch(c, st);  // (over already, or by a sequence of it that got shorter)
    });
}

int nh_kv4_extend(nh_kv4* c, const int* seqs, const int* rows, int n, void* stream) {
    if (int rc = check(c)) return rc;
    if (n < 0 || (n > 0 && (!seqs || !rows))) return fail(NH_EINVAL, "bad arguments");
    hipStream_t st = (hipStream_t)stream;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        std::vector<std::pair<int, int>> copies;
        if (int rc = c->book.extend(seqs, rows, n, &copies)) return refused(c, rc);
        // (the book has changed: a launch that fails from here on leaves the
        // device behind, as any failed launch does, and the caller frees the cache)
        if (int rc = copy_pages(c, copies, st)) return rc;
        const std::vector<int>& row0 = c->book.batch_row0;
        c->v.nb = n;
        c->v.rows = row0.back();
        c->v.each = n ? rows[0] : 0;
        shape_of_rows(rows, n, c->v.shape);
        if (int rc = put_shape(c, c->v.shape[0], c->v.shape[1], st)) return rc;
        for (int i = 0; i < n; ++i) {
            if (int rc = sync_table(c, seqs[i], st)) return rc;
            const int entry[4] = {seqs[i], row0[i], row0[i + 1], c->book.seqs[seqs[i]].len};
            for (int k = 0; k < 4; ++k)
                if (int rc = put_changed(c, c->o_batch + 4 + 4 * (size_t)i + k, entry[k], st)) return rc;
            if (rows[i] != rows[0]) c->v.each = 0;
        }
        return flush(c, st);
    });
}

int nh_kv4_rows(const nh_kv4* c) {
    if (!c) return fail(NH_EINVAL, "null cache");
    return c->book.batch_row0.back();
}

int nh_kv4_append(nh_kv4* c, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int type, void* stream) {
    if (int rc = check(c)) return rc;
    if (int rc = check_batch(c, layer)) return rc;
    if (!known_type(type)) return fail(NH_EINVAL, "no such type");
    if (c->v.rows == 0) return NH_OK;
    if (!k || !v) return fail(NH_EINVAL, "null argument");
    if (ldk < (int64_t)c->v.heads * c->v.dk || ldv < (int64_t)c->v.heads * c->v.dv)
        return fail(NH_EINVAL, "rows overlap: a row holds every head");
    NH_TRY(nh::launch_kv4_append(c->v, c->book.batch_row0.data(), layer, k, v, ldk, ldv, type, (hipStream_t)stream), "kv4 append");
    return NH_OK;
}

int nh_kv4_read(nh_kv4* c, int layer, const int* seqs, const int* pos, const int* rows, int n, void* k, void* v,
                int type, void* stream) {
    if (int rc = check(c)) return rc;
    if (layer < -1 || layer >= c->v.layers) return fail(NH_EINVAL, "no such layer");
    if (n < 0 || (n > 0 && (!seqs || !pos || !rows))) return fail(NH_EINVAL, "bad arguments");
    if (!known_type(type)) return fail(NH_EINVAL, "no such type");
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        if (!c->book.live(seqs[i])) return fail(NH_EINVAL, "no such sequence");
        if (pos[i] < 0 || rows[i] < 0 || pos[i] > c->book.seqs[seqs[i]].len - rows[i])
            return fail(NH_EINVAL, "the positions are not within the sequence");
        total += rows[i];
    }
    if (total == 0) return 0;
    if (total > INT32_MAX) return fail(NH_EINVAL, "too many rows");
    if (!k || !v) return fail(NH_EINVAL, "null argument");
    hipStream_t st = (hipStream_t)stream;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        for (int i = 0; i < n; ++i)
            if (int rc = sync_table(c, seqs[i], st)) return rc;
        if (int rc = flush(c, st)) return rc;
        nh::Kv4Spans p;
        int64_t row = 0;
        for (int i = 0; i < n;) {
            p.n = 0;
            p.row0[0] = p.unit0[0] = 0;
            for (; i < n && p.n < nh::Kv4Spans::MAX; ++i) {
                if (!rows[i]) continue;
                p.seq[p.n] = seqs[i];
                p.pos[p.n] = pos[i];
                p.row0[p.n + 1] = p.row0[p.n] + rows[i];
                p.unit0[p.n + 1] = p.unit0[p.n] + nh::kv4_chunks(pos[i], rows[i]);
                ++p.n;
            }
            if (!p.n) break;
            NH_TRY(nh::launch_kv4_read(c->v, layer, p, total, row, k, v, type, st), "kv4 read");
            row += p.row0[p.n];
        }
        return (int)total;
    });
}

static int check_attend(const nh_kv4* c, int layer, int heads, int sink, int ring) {
    if (int rc = check_batch(c, layer)) return rc;
    if (heads < 1 || heads % c->v.heads != 0 || heads / c->v.heads > 1024)
        return fail(NH_EINVAL, "the query heads are 1 to 1024 for each key/value head");
    if (sink < 0 || ring < 0) return fail(NH_EINVAL, "sink and ring are not negative");
    return NH_OK;
}

static int longest(const nh_kv4* c) {
    int n = 0;
    for (int s : c->book.batch_seq) n = std::max(n, c->book.seqs[s].len);
    return n;
}

int nh_kv4_debug_kernel(nh_kv4* c, int kernel) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (kernel < 0 || kernel > 2) return fail(NH_EINVAL, "0, 1 or 2");
    c->v.kernel = kernel;
    return NH_OK;
}

int64_t nh_kv4_attend_ws_bytes(const nh_kv4* c, int heads, int sink, int ring) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (int rc = check_attend(c, 0, heads, sink, ring)) return rc;
    return (int64_t)nh::kv4_attend_ws(c->v, c->book.batch_row0.data(), heads, sink, ring, longest(c));
}

int nh_kv4_attend(const nh_kv4* c, int layer, const void* q, int64_t ldq, int heads, float scale, int sink, int ring,
                  void* out, int64_t ldo, float* lse, int type, void* ws, uint64_t ws_bytes, void* stream) {
    if (int rc = check(c)) return rc;
    if (int rc = check_attend(c, layer, heads, sink, ring)) return rc;
    if (!known_type(type)) return fail(NH_EINVAL, "no such type");
    if (!(fabsf(scale) <= 3.402823466e38f)) return fail(NH_EINVAL, "the scale is not finite");
    if (c->v.rows == 0) return NH_OK;
    if (!q || !out) return fail(NH_EINVAL, "null argument");
    if (ldq < (int64_t)heads * c->v.dk || ldo < (int64_t)heads * c->v.dv)
        return fail(NH_EINVAL, "rows overlap: a row holds every head");
    const int most = longest(c);
    const size_t need = nh::kv4_attend_ws(c->v, c->book.batch_row0.data(), heads, sink, ring, most);
    if (need && (!ws || (uintptr_t)ws % 16 != 0)) return fail(NH_EINVAL, "no 16-byte aligned workspace");
    if (ws_bytes < need) return fail(NH_ESMALL, "the workspace is too small");
    nh::Kv4AttendArgs a{q, out, lse, type, layer, heads, sink, ring, ldq, ldo, scale, ws};
    NH_TRY(nh::launch_kv4_attend(c->v, c->book.batch_row0.data(), a, most, (hipStream_t)stream), "kv4 attention");
    return NH_OK;
}

}  // extern "C"
