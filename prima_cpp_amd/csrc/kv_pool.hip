// kv_pool.hip — C entry points of the page pool (kv_pool.h); no device code.
#include "kv_pool.h"
#include <new>

// (no exception leaves a C entry)
template <class F> static int guarded(F && f) { try { return f(); } catch (...) { return PM355_E_NOMEM; } }

extern "C" {
pm355_page_pool * pm355_page_pool_new(int n_pages, int n_seqs, int max_seq_pages) {
    try { return n_pages > 0 && n_seqs > 0 && max_seq_pages > 0 ? new pm355_page_pool(n_pages, n_seqs, max_seq_pages, false) : nullptr; } catch (...) { return nullptr; }
}
void pm355_page_pool_free(pm355_page_pool * p) { delete p; }
int pm355_page_pool_open(pm355_page_pool * p) { return p->open(); }
int pm355_page_pool_close(pm355_page_pool * p, int seq) { return p->close(seq); }
int pm355_page_pool_grow(pm355_page_pool * p, int seq, int n_tokens) { return guarded([&] { return p->grow(seq, n_tokens); }); }
int pm355_page_pool_drop_before(pm355_page_pool * p, int seq, int position) { return p->drop_before(seq, position); }
int pm355_page_pool_drop(pm355_page_pool * p, int seq, int from, int to) { return p ? p->drop(seq, from, to) : PM355_E_RANGE; }
int pm355_page_pool_fork(pm355_page_pool * p, int seq, int n_tokens) { return p ? guarded([&] { return p->fork(seq, n_tokens); }) : PM355_E_RANGE; }
int pm355_page_pool_own(pm355_page_pool * p, int seq, int from, int32_t * pairs, int max_pairs) { return p ? guarded([&] { return p->own(seq, from, pairs, max_pairs); }) : PM355_E_RANGE; }
int pm355_page_pool_compact(pm355_page_pool * p, int32_t * pairs, int max_pairs) { return p ? guarded([&] { return p->compact(pairs, max_pairs); }) : PM355_E_RANGE; }
int pm355_page_pool_users(const pm355_page_pool * p, int page) { return p && page >= 0 && page < p->n_pages ? p->users[page] : PM355_E_RANGE; }
int pm355_page_pool_page(const pm355_page_pool * p, int seq, int index) { return p->page(seq, index); }
int pm355_page_pool_free_pages(const pm355_page_pool * p) { return (int) p->free_list.size(); }
}
