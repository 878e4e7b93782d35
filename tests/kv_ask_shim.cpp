// The paged caches' book for ctypes, as a batch of queries alone uses it (built by the test that loads it).
#include "../needle-rs_amd/csrc/nh_kv4_book.h"

using nh::Kv4Book;

extern "C" {
Kv4Book* ask_new(int page, int pages, int seqs, int cap) {
    Kv4Book* b = new Kv4Book;
    b->init(page, pages, seqs, cap);
    return b;
}
void ask_free(Kv4Book* b) { delete b; }
int ask_seq(Kv4Book* b) { return b->new_seq(); }
int ask_drop(Kv4Book* b, int s) { return b->free_seq(s); }
int ask_len(Kv4Book* b, int s) { return b->seqs[s].len; }
int ask_pages(Kv4Book* b) { return (int)b->free_pages.size(); }
int ask_extend(Kv4Book* b, const int* s, const int* rows, int n) {
    std::vector<std::pair<int, int>> copies;
    return b->extend(s, rows, n, &copies);
}
int ask_truncate(Kv4Book* b, int s, int len) { return b->truncate(s, len); }
int ask_ask(Kv4Book* b, const int* s, const int* rows, int n) { return b->ask(s, rows, n); }
// The batch: its sequences' number, and their first rows in row0[0 .. n].
int ask_batch(Kv4Book* b, int* seqs, int* row0) {
    for (size_t i = 0; i < b->batch_seq.size(); ++i) seqs[i] = b->batch_seq[i];
    for (size_t i = 0; i < b->batch_row0.size(); ++i) row0[i] = b->batch_row0[i];
    return (int)b->batch_seq.size();
}
}
