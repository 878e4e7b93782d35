// The cache's page book for ctypes (built by the test that loads it).
#include "../needle-rs_amd/csrc/nh_kv4_book.h"

using nh::Kv4Book;

extern "C" {
Kv4Book* book_new(int page, int pages, int seqs, int cap) {
    Kv4Book* b = new Kv4Book;
    b->init(page, pages, seqs, cap);
    return b;
}
void book_free(Kv4Book* b) { delete b; }
int book_new_seq(Kv4Book* b) { return b->new_seq(); }
int book_free_seq(Kv4Book* b, int s) { return b->free_seq(s); }
int book_fork(Kv4Book* b, int s, int n, int* out) { return b->fork(s, n, out); }
int book_truncate(Kv4Book* b, int s, int len) { return b->truncate(s, len); }
int book_free_pages(Kv4Book* b) { return (int)b->free_pages.size(); }
int book_len(Kv4Book* b, int s) { return b->live(s) ? b->seqs[s].len : -1; }
int book_table(Kv4Book* b, int s, int* out) {
    for (size_t i = 0; i < b->seqs[s].table.size(); ++i) out[i] = b->seqs[s].table[i];
    return (int)b->seqs[s].table.size();
}
int book_refs(Kv4Book* b, int p) { return b->refs[p]; }
int book_batch(Kv4Book* b, int* seqs, int* row0) {
    for (size_t i = 0; i < b->batch_seq.size(); ++i) seqs[i] = b->batch_seq[i];
    for (size_t i = 0; i < b->batch_row0.size(); ++i) row0[i] = b->batch_row0[i];
    return (int)b->batch_seq.size();
}
// The copies as (from, to) pairs; returns their number or the refusal.
int book_copy(Kv4Book* b, int s, int* to, int* pairs) {
    std::vector<std::pair<int, int>> c;
    const int rc = b->copy(s, to, &c);
    for (size_t i = 0; i < c.size(); ++i) pairs[2 * i] = c[i].first, pairs[2 * i + 1] = c[i].second;
    return rc ? rc : (int)c.size();
}
int book_extend(Kv4Book* b, const int* s, const int* rows, int n, int* pairs) {
    std::vector<std::pair<int, int>> c;
    const int rc = b->extend(s, rows, n, &c);
    for (size_t i = 0; i < c.size(); ++i) pairs[2 * i] = c[i].first, pairs[2 * i + 1] = c[i].second;
    return rc ? rc : (int)c.size();
}
// Plans, reports the moves as (seq index, src, fresh page, slot, count per position = 1) and finishes.
int book_compact(Kv4Book* b, const int* s, int n, const int* counts, const int* ranges, int* moves) {
    Kv4Book::Compaction c;
    const int rc = b->compact(s, n, counts, ranges, &c);
    if (rc) return rc;
    int m = 0;
    for (const auto& v : c.moves)
        for (int i = 0; i < v.count; ++i, ++m) {
            const int dst = v.dst + i;
            moves[4 * m] = b->seqs[s[v.seq]].table[(v.src + i) / b->page];
            moves[4 * m + 1] = (v.src + i) % b->page;
            moves[4 * m + 2] = c.fresh[v.seq][dst / b->page];
            moves[4 * m + 3] = dst % b->page;
        }
    b->compacted(s, n, c);
    return m;
}
}
