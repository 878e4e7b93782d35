// The pages of a 4-bit key/value cache, on the host: which sequence holds
// which pages, how many sequences share a page, which pages are free.  Plain
// C++ without HIP; nh_kv4.cpp mirrors the tables on the device.
//
// A sequence is a list of page ids and a length.  Branches share pages by
// count; a page is written only by its single holder, so a sequence that is
// extended inside a shared last page gets a copy of it first (the copy is in
// the plan that extend returns).  Every operation checks what it needs before
// it changes anything: a refused call leaves the book as it was.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

namespace nh {

struct Kv4Book {
    struct Seq {
        bool live = false;
        int len = 0;
        std::vector<int> table;  // page ids of positions 0 .. len - 1
        int synced = 0;          // leading entries that the device's copy holds
    };
    // One kept range of a compaction: `count` positions from `src` move to `dst`.
    struct Move {
        int seq, src, dst, count;
    };

    int page = 0;       // positions a page holds
    int cap_pages = 0;  // pages a sequence may hold
    std::vector<int> refs;
    std::vector<int> free_pages;
    std::vector<Seq> seqs;
    std::vector<int> batch_seq, batch_row0;  // the last extend: its sequences and their first rows
    std::string why;                         // the last refusal

    // 0, or NH_EINVAL / NH_ENOMEM's values (the header's codes).
    static constexpr int INVALID = -1, NO_ROOM = -4;

    void init(int page_, int pages, int n_seqs, int cap) {
        page = page_;
        cap_pages = (int)(((int64_t)cap + page - 1) / page);
        refs.assign(pages, 0);
        free_pages.resize(pages);
        for (int i = 0; i < pages; ++i) free_pages[i] = pages - 1 - i;  // page 0 is dealt first
        seqs.assign(n_seqs, Seq());
        batch_row0.assign(1, 0);
    }

    int refuse(int code, const char* text) {
        why = text;
        return code;
    }
    bool live(int s) const { return s >= 0 && s < (int)seqs.size() && seqs[s].live; }
    int pages_of(int len) const { return (int)(((int64_t)len + page - 1) / page); }

    int new_seq() {
        for (size_t i = 0; i < seqs.size(); ++i)
            if (!seqs[i].live) {
                seqs[i].live = true;
                seqs[i].len = seqs[i].synced = 0;
                seqs[i].table.clear();
                return (int)i;
            }
        return refuse(NO_ROOM, "every sequence of the cache is in use");
    }

    void release(int p) {
        if (--refs[p] == 0) free_pages.push_back(p);
    }
    int take() {
        const int p = free_pages.back();
        free_pages.pop_back();
        refs[p] = 1;
        return p;
    }
    // A sequence that changed, or whose pages another now shares, is no longer
    // the batch's, and the batch is over: a later append would write rows that
    // the book no longer places, or that a branch reads.
    void leave_batch(int s) {
        for (int b : batch_seq)
            if (b == s) {
                batch_seq.clear();
                batch_row0.assign(1, 0);
                return;
            }
    }

    int free_seq(int s) {
        if (!live(s)) return refuse(INVALID, "no such sequence");
        leave_batch(s);
        for (int p : seqs[s].table) release(p);
        seqs[s].table.clear();
        seqs[s].len = 0;
        seqs[s].live = false;
        return 0;
    }

    // n branches that share every page of s.
    int fork(int s, int n, int* out) {
        if (!live(s)) return refuse(INVALID, "no such sequence");
        int room = 0;
        for (const Seq& q : seqs) room += !q.live;
        if (n < 0) return refuse(INVALID, "a negative number of branches");
        if (n > room) return refuse(NO_ROOM, "too few unused sequences");
        if (n) leave_batch(s);
        for (int i = 0; i < n; ++i) {
            const int c = new_seq();
            seqs[c].table = seqs[s].table;
            seqs[c].len = seqs[s].len;
            for (int p : seqs[c].table) ++refs[p];
            out[i] = c;
        }
        return 0;
    }

    // A branch with pages of its own; `copies` gets (from, to).
    int copy(int s, int* out, std::vector<std::pair<int, int>>* copies) {
        if (!live(s)) return refuse(INVALID, "no such sequence");
        if (seqs[s].table.size() > free_pages.size()) return refuse(NO_ROOM, "too few free pages");
        const int c = new_seq();
        if (c < 0) return c;
        leave_batch(s);
        seqs[c].len = seqs[s].len;
        for (int p : seqs[s].table) {
            seqs[c].table.push_back(take());
            copies->push_back({p, seqs[c].table.back()});
        }
        *out = c;
        return 0;
    }

    int truncate(int s, int len) {
        if (!live(s)) return refuse(INVALID, "no such sequence");
        if (len < 0 || len > seqs[s].len) return refuse(INVALID, "the new length is not within the sequence");
        if (len == seqs[s].len) return 0;
        leave_batch(s);
        const int keep = pages_of(len);
        for (size_t i = keep; i < seqs[s].table.size(); ++i) release(seqs[s].table[i]);
        seqs[s].table.resize(keep);
        seqs[s].synced = std::min(seqs[s].synced, keep);
        seqs[s].len = len;
        return 0;
    }

    bool distinct(const int* s, int n) const {
        std::vector<char> seen(seqs.size(), 0);
        for (int i = 0; i < n; ++i) {
            if (seen[s[i]]) return false;
            seen[s[i]] = 1;
        }
        return true;
    }

    // rows[i] more positions for each sequence, which become the batch.
    // `copies` gets the pages (from, to) to copy before they are written.
    int extend(const int* s, const int* rows, int n, std::vector<std::pair<int, int>>* copies) {
        int64_t total = 0;
        for (int i = 0; i < n; ++i) {
            if (!live(s[i])) return refuse(INVALID, "no such sequence");
            if (rows[i] < 0) return refuse(INVALID, "a negative number of rows");
            if ((int64_t)seqs[s[i]].len + rows[i] > (int64_t)cap_pages * page)
                return refuse(INVALID, "the rows do not fit the sequences' capacity");
            total += rows[i];
        }
        if (!distinct(s, n)) return refuse(INVALID, "a sequence is named twice");
        if (total > INT32_MAX) return refuse(INVALID, "too many rows");
        // A shared page that several of these sequences end in: each but its
        // last holder copies it.
        int64_t need = 0;
        std::vector<std::pair<int, int>> shared;  // (page, holders left)
        for (int i = 0; i < n; ++i) {
            const Seq& q = seqs[s[i]];
            need += pages_of(q.len + rows[i]) - (int)q.table.size();
            if (rows[i] && q.len % page && refs[q.table.back()] > 1) {
                const int p = q.table.back();
                size_t j = 0;
                while (j < shared.size() && shared[j].first != p) ++j;
                if (j == shared.size()) shared.push_back({p, refs[p]});
                if (shared[j].second > 1) {
                    --shared[j].second;
                    ++need;
                }
            }
        }
        if (need > (int64_t)free_pages.size()) return refuse(NO_ROOM, "too few free pages");
        batch_seq.assign(s, s + n);
        batch_row0.assign(1, 0);
        for (int i = 0; i < n; ++i) {
            Seq& q = seqs[s[i]];
            if (rows[i] && q.len % page && refs[q.table.back()] > 1) {
                const int from = q.table.back();
                --refs[from];
                q.table.back() = take();
                q.synced = std::min(q.synced, (int)q.table.size() - 1);
                copies->push_back({from, q.table.back()});
            }
            q.len += rows[i];
            while ((int)q.table.size() < pages_of(q.len)) q.table.push_back(take());
            batch_row0.push_back(batch_row0.back() + rows[i]);
        }
        return 0;
    }

    // Sequence s[i] keeps its positions of counts[i] ascending, disjoint
    // ranges [ranges[2 j], ranges[2 j + 1]), closed up.  Leading pages that
    // stay whole stay; the others' kept positions move to fresh pages.  `moves`
    // gets the runs (seq an index into s, dst counted from the first fresh
    // page's position), `first` each sequence's first fresh page index, `fresh`
    // its fresh pages.
    struct Compaction {
        std::vector<Move> moves;
        std::vector<int> len, first;
        std::vector<std::vector<int>> fresh;
    };
    int compact(const int* s, int n, const int* counts, const int* ranges, Compaction* c) {
        int64_t need = 0;
        const int* r = ranges;
        std::vector<Move> moves;
        std::vector<int> lens, firsts;
        for (int i = 0; i < n; ++i) {
            if (!live(s[i])) return refuse(INVALID, "no such sequence");
            if (counts[i] < 0) return refuse(INVALID, "a negative number of ranges");
            const int len = seqs[s[i]].len;
            int at = 0, end = 0, prefix = 0;
            for (int j = 0; j < counts[i]; ++j, r += 2) {
                if (r[0] < end || r[1] < r[0] || r[1] > len)
                    return refuse(INVALID, "ranges are ascending, apart and within the sequence");
                if (r[0] == at) prefix = at + (r[1] - r[0]);  // (still where it was)
                at += r[1] - r[0];
                end = r[1];
            }
            lens.push_back(at);
            // All in place: the tail is cut, nothing moves.
            const int first = prefix == at ? pages_of(at) : prefix / page;
            firsts.push_back(first);
            need += pages_of(at) - first;
            const int* q = r - 2 * counts[i];
            int to = 0;
            for (int j = 0; j < counts[i]; ++j, q += 2) {
                int src = q[0], cnt = q[1] - q[0];
                const int skip = first * page - to;  // positions that stay in leading pages
                to += cnt;
                if (skip > 0) {
                    src += skip;
                    cnt -= skip;
                }
                if (cnt > 0 && prefix != at) moves.push_back({i, src, to - cnt - first * page, cnt});
            }
        }
        if (!distinct(s, n)) return refuse(INVALID, "a sequence is named twice");
        if (need > (int64_t)free_pages.size()) return refuse(NO_ROOM, "too few free pages");
        c->moves.swap(moves);
        c->len = lens;
        c->first = firsts;
        c->fresh.assign(n, {});
        for (int i = 0; i < n; ++i)
            for (int p = firsts[i]; p < pages_of(lens[i]); ++p) c->fresh[i].push_back(take());
        return 0;
    }
    // The second half of a compaction: the tables as the moves leave them.
    void compacted(const int* s, int n, const Compaction& c) {
        for (int i = 0; i < n; ++i) {
            Seq& q = seqs[s[i]];
            if (q.len != c.len[i]) leave_batch(s[i]);
            for (size_t p = c.first[i]; p < q.table.size(); ++p) release(q.table[p]);
            q.table.resize(c.first[i]);
            q.synced = std::min(q.synced, c.first[i]);
            q.table.insert(q.table.end(), c.fresh[i].begin(), c.fresh[i].end());
            q.len = c.len[i];
        }
    }
    // A compaction whose moves could not be queued.
    void give_back(const Compaction& c) {
        for (const auto& f : c.fresh)
            for (int p : f) release(p);
    }
};

}  // namespace nh
