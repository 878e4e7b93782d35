// The C ABI of the 8-bit key/value cache (include/needle_hip.h) over the host
// side that the paged caches share (nh_kv_host.h).
#include <math.h>

#include <memory>

#include "nh_kv8.h"
#include "nh_kv_host.h"

using namespace nh::kv;

struct nh_kv8 : nh::KvHost {
    nh::Kv8View v{};
    bool captured = false;  // a graph holds an append
    nh_kv8() { view = &v; }
};

extern "C" {

int nh_kv8_new(int layers, int kv_heads, int qk_dim, int v_dim, int page, int pages, int seqs, int cap, nh_kv8** h) {
    if (!h) return fail(NH_EINVAL, "null argument");
    *h = nullptr;
    if (page != 64 && page != 128 && page != 256) return fail(NH_EINVAL, "a page holds 64, 128 or 256 positions");
    if (int rc = check_new(layers, kv_heads, qk_dim, v_dim, page, pages, seqs, cap)) return rc;
    static const int widths[4][2] = {{64, 64}, {128, 128}, {192, 128}, {256, 256}};
    const int* w = widths[0];
    while (qk_dim > w[0] || v_dim > w[1]) w += 2;
    if ((double)pages * page * layers * kv_heads * (w[0] + w[1] + 2) > 0x1p46)
        return fail(NH_EINVAL, "the pages are larger than any device's memory");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    return guarded([&]() -> int {
        auto c = std::make_unique<nh_kv8>();
        nh::Kv8View& v = c->v;
        v.wk = w[0], v.wv = w[1];
        v.page_log2 = page == 64 ? 6 : page == 128 ? 7 : 8;
        c->page_bytes = v.block() * kv_heads * layers;
        if (int rc = allocate(c.get(), layers, kv_heads, qk_dim, v_dim, page, pages, seqs, cap)) return rc;
        *h = c.release();
        return NH_OK;
    });
}

int nh_kv8_free(nh_kv8* c) {
    if (!c) return NH_OK;
    release(c);
    delete c;
    return NH_OK;
}

int64_t nh_kv8_bytes(const nh_kv8* c) { return bytes(c); }
int nh_kv8_free_pages(const nh_kv8* c) { return free_pages(c); }
int nh_kv8_seq_new(nh_kv8* c) { return seq_new(c); }
int nh_kv8_seq_len(const nh_kv8* c, int seq) { return seq_len(c, seq); }
int nh_kv8_seq_free(nh_kv8* c, int seq) { return seq_free(c, seq); }
int nh_kv8_seq_truncate(nh_kv8* c, int seq, int len) { return seq_truncate(c, seq, len); }
int nh_kv8_seq_fork(nh_kv8* c, int seq, int n, int* branches) { return seq_fork(c, seq, n, branches); }
int nh_kv8_seq_copy(nh_kv8* c, int seq, void* stream) { return seq_copy(c, seq, (hipStream_t)stream); }

int nh_kv8_extend(nh_kv8* c, const int* seqs, const int* rows, int n, void* stream) {
    const int rc = extend(c, seqs, rows, n, (hipStream_t)stream);
    if (c) c->v.ask = c->asks;
    return rc;
}

int nh_kv8_ask(nh_kv8* c, const int* seqs, const int* rows, int n, void* stream) {
    if (int rc = check(c)) return rc;
    if (n < 0 || (n > 0 && (!seqs || !rows))) return fail(NH_EINVAL, "bad arguments");
    hipStream_t st = (hipStream_t)stream;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int {
        if (int rc = c->book.ask(seqs, rows, n)) return refused(c, rc);
        c->asks = true;
        c->v.ask = 1;
        return put_batch(c, seqs, rows, n, st);
    });
}

int nh_kv8_rows(const nh_kv8* c) { return rows(c); }

// A replayed append of a batch that is over would round the kept rows of its
// begun blocks anew: without the batch's shape it does nothing.
int nh_kv8_end_batch(nh_kv8* c, void* stream) {
    if (int rc = check(c)) return rc;
    if (!c->captured) return NH_OK;
    hipStream_t st = (hipStream_t)stream;
    if (int rc = check_eager(st)) return rc;
    return guarded([&]() -> int { return drop_batch(c, st); });
}

int nh_kv8_append(nh_kv8* c, int layer, const void* k, const void* v, int64_t ldk, int64_t ldv, int type,
                  const nh_rope* rope, const int32_t* pos, const void* q, int64_t ldq, int heads, void* q_out,
                  int64_t ldqo, void* stream) {
    if (int rc = check(c)) return rc;
    if (int rc = check_batch(c, layer)) return rc;
    if (c->asks) return fail(NH_EINVAL, "the batch's rows are queries alone: no positions to store");
    if (!known_type(type)) return fail(NH_EINVAL, "no such type");
    if (heads < 0 || heads > (1 << 20)) return fail(NH_EINVAL, "0 to 2^20 query heads");
    if (!rope && (heads || pos)) return fail(NH_EINVAL, "queries and positions go with a rope");
    if (rope && rope->device != c->device) return fail(NH_EINVAL, "the plan belongs to another device than the cache");
    if (rope && 2 * rope->v.pairs > c->v.dk) return fail(NH_EINVAL, "a head holds the plan's pairs");
    if (c->v.rows == 0) return NH_OK;
    if (!k || !v || (heads && (!q || !q_out))) return fail(NH_EINVAL, "null argument");
    const int64_t wq = (int64_t)heads * c->v.dk;
    if (ldk < (int64_t)c->v.heads * c->v.dk || ldv < (int64_t)c->v.heads * c->v.dv || (heads && (ldq < wq || ldqo < wq)))
        return fail(NH_EINVAL, "rows overlap: a row holds every head");
    if (heads && q == q_out && ldq != ldqo) return fail(NH_EINVAL, "rows turned in place stay where they are");
    nh::Kv8Append a{k, v, ldk, ldv, layer, {}, pos, {}};
    if (rope) a.r = rope->v;
    if (heads) a.q = nh::RopeRows{q, q_out, ldq, ldqo, heads};
    if (!c->captured) {
        hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing((hipStream_t)stream, &s) == hipSuccess)
            c->captured = s != hipStreamCaptureStatusNone;
        else
            (void)hipGetLastError();  // (the null stream while another captures: the launch says what it thinks of it)
    }
    NH_TRY(nh::launch_kv8_append(c->v, c->book.batch_row0.data(), a, type, (hipStream_t)stream), "kv8 append");
    return NH_OK;
}

int nh_kv8_read(nh_kv8* c, int layer, const int* seqs, const int* pos, const int* rows, int n, void* k, void* v,
                int type, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    return read(c, layer, seqs, pos, rows, n, k, v, type, st, nh::kv8_chunks,
                [&](const nh::KvSpans& p, int64_t total, int64_t row) {
                    return nh::launch_kv8_read(c->v, layer, p, total, row, k, v, type, st);
                });
}

int nh_kv8_debug_kernel(nh_kv8* c, int kernel) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (kernel < 0 || kernel > 2) return fail(NH_EINVAL, "0, 1 or 2");
    c->v.kernel = kernel;
    return NH_OK;
}

int64_t nh_kv8_attend_ws_bytes(const nh_kv8* c, int heads, int sink, int ring) {
    if (!c) return fail(NH_EINVAL, "null cache");
    if (int rc = check_attend(c, 0, heads, sink, ring)) return rc;
    return (int64_t)nh::kv8_attend_ws(c->v, c->book.batch_row0.data(), heads, sink, ring, longest(c));
}

int nh_kv8_attend(const nh_kv8* c, int layer, const void* q, int64_t ldq, int heads, float scale, int sink, int ring,
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
    const size_t need = nh::kv8_attend_ws(c->v, c->book.batch_row0.data(), heads, sink, ring, most);
    if (need && (!ws || (uintptr_t)ws % 16 != 0)) return fail(NH_EINVAL, "no 16-byte aligned workspace");
    if (ws_bytes < need) return fail(NH_ESMALL, "the workspace is too small");
    nh::Kv8AttendArgs a{q, out, lse, type, layer, heads, sink, ring, ldq, ldo, scale, ws};
    NH_TRY(nh::launch_kv8_attend(c->v, c->book.batch_row0.data(), a, most, (hipStream_t)stream), "kv8 attention");
    return NH_OK;
}

}  // extern "C"
