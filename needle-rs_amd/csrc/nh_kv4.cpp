// The C ABI of the 4-bit key/value cache (include/needle_hip.h) over the host
// side that the paged caches share (nh_kv_host.h).
#include <math.h>

#include <memory>

#include "nh_kv4.h"
#include "nh_kv_host.h"

using namespace nh::kv;

struct nh_kv4 : nh::KvHost {
    nh::Kv4View v{};
    nh_kv4() { view = &v; }
};

extern "C" {

int nh_kv4_new(int layers, int kv_heads, int qk_dim, int v_dim, int group, int page, int pages, int seqs, int cap,
               nh_kv4** h) {
    if (!h) return fail(NH_EINVAL, "null argument");
    *h = nullptr;
    if (group != 32 && group != 64) return fail(NH_EINVAL, "groups are 32 or 64 values");
    if (page != 32 && page != 64 && page != 128 && page != 256)
        return fail(NH_EINVAL, "a page holds 32, 64, 128 or 256 positions");
    if (int rc = check_new(layers, kv_heads, qk_dim, v_dim, page, pages, seqs, cap)) return rc;
    const int wide = std::max(qk_dim, v_dim), width = wide <= 64 ? 64 : wide <= 128 ? 128 : 256;
    if ((double)pages * page * layers * kv_heads * (width + 8 * (width / group)) > 0x1p46)
        return fail(NH_EINVAL, "the pages are larger than any device's memory");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    return guarded([&]() -> int {
        auto c = std::make_unique<nh_kv4>();
        nh::Kv4View& v = c->v;
        v.width = width;
        v.group = group;
        v.layers = layers, v.heads = kv_heads;
        v.page_log2 = page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : 8;
        c->page_bytes = v.page_bytes();
        if (int rc = allocate(c.get(), layers, kv_heads, qk_dim, v_dim, page, pages, seqs, cap)) return rc;
        *h = c.release();
        return NH_OK;
    });
}

int nh_kv4_free(nh_kv4* c) {
    if (!c) return NH_OK;
    release(c);
    delete c;
    return NH_OK;
}

int64_t nh_kv4_bytes(const nh_kv4* c) { return bytes(c); }
int nh_kv4_free_pages(const nh_kv4* c) { return free_pages(c); }
int nh_kv4_seq_new(nh_kv4* c) { return seq_new(c); }
int nh_kv4_seq_len(const nh_kv4* c, int seq) { return seq_len(c, seq); }
int nh_kv4_seq_free(nh_kv4* c, int seq) { return seq_free(c, seq); }
int nh_kv4_seq_truncate(nh_kv4* c, int seq, int len) { return seq_truncate(c, seq, len); }
int nh_kv4_seq_fork(nh_kv4* c, int seq, int n, int* branches) { return seq_fork(c, seq, n, branches); }
int nh_kv4_seq_copy(nh_kv4* c, int seq, void* stream) { return seq_copy(c, seq, (hipStream_t)stream); }

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
    return extend(c, seqs, rows, n, (hipStream_t)stream);
}

int nh_kv4_rows(const nh_kv4* c) { return rows(c); }

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
    hipStream_t st = (hipStream_t)stream;
    return read(c, layer, seqs, pos, rows, n, k, v, type, st, nh::kv4_chunks,
                [&](const nh::KvSpans& p, int64_t total, int64_t row) {
                    return nh::launch_kv4_read(c->v, layer, p, total, row, k, v, type, st);
                });
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
