// kv_pool.h — pages of a KV cache shared by the open sequences of a model (host side only). A sequence's pages are found through its table: page index (position / 64)
// -> pool page, or -1 in front of what its layers can still see and where a range was dropped. Pages come back in LIFO order, so a freed page is the next one handed out.
// Sequences that were forked share pages (`users` counts the tables a page stands in): a page is written by one user only, own() gives a sequence copies of its shared ones.
#pragma once
#include "../../include/prima_mi355.h"
#include <algorithm>
#include <utility>
#include <vector>

struct pm355_page_pool {
    static constexpr int PAGE = 64;
    struct Seq { bool open = false; int lo = 0, hi = 0; std::vector<int> page; };      // pages [lo, hi) are held
    int n_pages, max_seq_pages;
    std::vector<int> free_list;
    std::vector<int> users;                                // tables that hold the page, 0: free
    std::vector<Seq> seqs;
    const bool keeps_changes;                              // for an owner that takes them step by step (the C entries do not: there they would only grow)
    std::vector<std::pair<int, int>> changes;              // (seq * max_seq_pages + index, page) since the owner last took them

    pm355_page_pool(int pages, int n_seqs, int max_pages, bool keep) : n_pages(pages), max_seq_pages(max_pages), users((size_t) pages), seqs((size_t) n_seqs), keeps_changes(keep) {
        for (int i = pages - 1; i >= 0; --i) free_list.push_back(i);
    }
    bool valid(int s) const { return s >= 0 && s < (int) seqs.size() && seqs[s].open; }
    int open() {
        for (size_t s = 0; s < seqs.size(); ++s) if (!seqs[s].open) { seqs[s] = Seq(); seqs[s].open = true; return (int) s; }
        return PM355_E_NOMEM;
    }
    void room(size_t n) { if (keeps_changes && changes.capacity() < changes.size() + n) changes.reserve(std::max(2 * changes.capacity(), changes.size() + n)); }
    void changed(int s, int i) { if (keeps_changes) changes.push_back({s * max_seq_pages + i, seqs[s].page[i]}); }      // (behind room())
    void release(int page) { if (page >= 0 && --users[page] == 0) free_list.push_back(page); }
    int close(int s) {
        if (!valid(s)) return PM355_E_RANGE;
        for (int i = seqs[s].hi - 1; i >= seqs[s].lo; --i) release(seqs[s].page[i]);
        seqs[s] = Seq();
        return 0;
    }
    static int pages_of(int n_tokens) { return n_tokens / PAGE + (n_tokens % PAGE > 0); }
    int missing(int s, int n_tokens) const { const int need = pages_of(n_tokens); return need > seqs[s].hi ? need - seqs[s].hi : 0; }
    int grow(int s, int n_tokens) {
        if (!valid(s)) return PM355_E_RANGE;
        const int n = missing(s, n_tokens);
        if (n > max_seq_pages - seqs[s].hi) return PM355_E_RANGE;
        if (n > (int) free_list.size()) return PM355_E_NOMEM;
        room((size_t) n);
        seqs[s].page.reserve(seqs[s].page.size() + n);
        for (int i = 0; i < n; ++i) {
            seqs[s].page.push_back(free_list.back());
            free_list.pop_back();
            users[seqs[s].page.back()] = 1;
            changed(s, seqs[s].hi++);
        }
        return 0;
    }
    int drop_before(int s, int position) {
        if (!valid(s)) return PM355_E_RANGE;
        Seq & q = seqs[s];
        for (; q.lo < q.hi && (q.lo + 1) * PAGE <= position; ++q.lo) { release(q.page[q.lo]); q.page[q.lo] = -1; }
        return 0;
    }
    // pages that lie wholly in [from, to)
    int drop(int s, int from, int to) {
        if (!valid(s) || from < 0 || to < from) return PM355_E_RANGE;
        Seq & q = seqs[s];
        const int a = std::max(q.lo, from / PAGE + (from % PAGE != 0)), b = std::min(q.hi, to / PAGE);
        for (int i = a; i < b; ++i) { release(q.page[i]); q.page[i] = -1; }
        while (q.lo < q.hi && q.page[q.lo] < 0) ++q.lo;
        return 0;
    }
    // a sequence that shares the pages of the first n_tokens tokens of s
    int fork(int s, int n_tokens) {
        if (!valid(s) || n_tokens < 0 || missing(s, n_tokens)) return PM355_E_RANGE;
        const int hi = pages_of(n_tokens);
        std::vector<int> held(seqs[s].page.begin(), seqs[s].page.begin() + hi);
        room((size_t) hi);                                 // (what can fail for want of memory stands in front of what changes)
        const int t = open();
        if (t < 0) return t;
        Seq & q = seqs[t];
        q.hi = hi;
        q.lo = std::min(seqs[s].lo, hi);
        q.page.swap(held);
        for (int i = q.lo; i < q.hi; ++i) if (q.page[i] >= 0) { ++users[q.page[i]]; changed(t, i); }
        return t;
    }
    // pages of s from the one of position `from` on that others hold too become its own; pairs (from, to) of what has to be copied
    int own(int s, int from, int32_t * pairs, int max_pairs) {
        if (!valid(s) || from < 0 || max_pairs < 0) return PM355_E_RANGE;
        Seq & q = seqs[s];
        int n = 0;
        for (int i = std::max(q.lo, from / PAGE); i < q.hi; ++i) n += q.page[i] >= 0 && users[q.page[i]] > 1;
        if (n > max_pairs || (n && !pairs)) return PM355_E_RANGE;
        if (n > (int) free_list.size()) return PM355_E_NOMEM;
        room((size_t) n);
        for (int i = std::max(q.lo, from / PAGE); i < q.hi; ++i) {
            if (q.page[i] < 0 || users[q.page[i]] < 2) continue;
            const int to = free_list.back();
            free_list.pop_back();
            *pairs++ = q.page[i]; *pairs++ = to;
            --users[q.page[i]]; users[to] = 1; q.page[i] = to;
            changed(s, i);
        }
        return n;
    }
    // the n pages in use move to the first n; pairs (from, to): no page stands on both sides
    int compact(int32_t * pairs, int max_pairs) {
        if (max_pairs < 0) return PM355_E_RANGE;
        const int used = n_pages - (int) free_list.size();
        int n = 0;
        size_t tables = 0;
        for (int i = used; i < n_pages; ++i) { n += users[i] > 0; tables += (size_t) users[i]; }
        if (n > max_pairs || (n && !pairs)) return PM355_E_RANGE;
        room(tables);
        std::vector<int> to((size_t) n_pages, -1);
        for (int i = used, hole = 0; i < n_pages; ++i) {
            if (!users[i]) continue;
            while (users[hole]) ++hole;
            *pairs++ = i; *pairs++ = hole;
            to[i] = hole; users[hole] = users[i]; users[i] = 0;
        }
        for (size_t s = 0; s < seqs.size(); ++s)
            for (int i = seqs[s].lo; i < seqs[s].hi; ++i) {
                int & p = seqs[s].page[i];
                if (p >= 0 && to[p] >= 0) { p = to[p]; changed((int) s, i); }
            }
        free_list.clear();
        for (int i = n_pages - 1; i >= used; --i) free_list.push_back(i);
        return n;
    }
    int page(int s, int i) const { return valid(s) && i >= 0 && i < seqs[s].hi ? seqs[s].page[i] : -1; }
};
