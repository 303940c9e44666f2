// kv_pool.cpp -- which sequence holds which pages of a paged K/V cache (host only).
//
// Pages are counted by reference: a fork shares all pages of its parent, and a sequence that is
// about to write positions gets pages of its own for them.  What has to be copied first (the
// committed rows of a shared page) comes back as pairs for oasr_b200_kv_pages_copy, and page
// tables go to the kernels as they are.  Lowest free page first, so the pool stays compact.
#include <stdint.h>

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <vector>

#include "oasr_b200.h"

struct oasr_kv_pool {
    struct Seq {
        bool open = false;
        std::vector<int32_t> pages;
    };
    int32_t page, max_pages;
    std::vector<int32_t> refs;  // per page
    std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free;
    std::vector<Seq> seqs;

    bool has(int32_t seq) const { return seq >= 0 && seq < (int32_t)seqs.size() && seqs[(size_t)seq].open; }
    int32_t take() {
        const int32_t p = free.top();
        free.pop();
        refs[(size_t)p] = 1;
        return p;
    }
    void drop(int32_t p) {
        if (--refs[(size_t)p] == 0) free.push(p);
    }
    int32_t slot() {  // a closed sequence's number, or -1
        for (size_t i = 0; i < seqs.size(); ++i)
            if (!seqs[i].open) return (int32_t)i;
        return -1;
    }
};

// nothing may be thrown through the C boundary: an allocation that fails is a status
template <typename F>
static int32_t guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return OASR_STATUS_ALLOC_FAILED;
    } catch (...) {
        return OASR_STATUS_FAILED;
    }
}

extern "C" {

int oasr_b200_kv_pool_create(int32_t n_pages, int32_t page, int32_t max_pages, int32_t max_seqs, oasr_kv_pool **out) {
    if (!out) return OASR_STATUS_FAILED;
    *out = nullptr;
    if (n_pages < 1 || page < 1 || max_pages < 1 || max_seqs < 1 || (int64_t)max_pages * page > INT32_MAX) return OASR_STATUS_FAILED;
    return guarded([&]() -> int32_t {
        oasr_kv_pool *p = new oasr_kv_pool();
        try {
            p->page = page;
            p->max_pages = max_pages;
            p->refs.assign((size_t)n_pages, 0);
            p->seqs.resize((size_t)max_seqs);
            for (int32_t i = 0; i < n_pages; ++i) p->free.push(i);
        } catch (...) {
            delete p;
            throw;
        }
        *out = p;
        return OASR_STATUS_SUCCESS;
    });
}

int oasr_b200_kv_pool_free(oasr_kv_pool *pool) {
    delete pool;
    return OASR_STATUS_SUCCESS;
}

int32_t oasr_b200_kv_pool_pages_free(const oasr_kv_pool *pool) { return pool ? (int32_t)pool->free.size() : OASR_STATUS_FAILED; }

int32_t oasr_b200_kv_pool_open(oasr_kv_pool *pool) {
    if (!pool) return OASR_STATUS_FAILED;
    const int32_t s = pool->slot();
    if (s < 0) return OASR_STATUS_ALLOC_FAILED;
    pool->seqs[(size_t)s].open = true;
    return s;
}

int32_t oasr_b200_kv_pool_fork(oasr_kv_pool *pool, int32_t seq) {
    if (!pool || !pool->has(seq)) return OASR_STATUS_FAILED;
    return guarded([&]() -> int32_t {
        const int32_t s = pool->slot();
        if (s < 0) return OASR_STATUS_ALLOC_FAILED;
        pool->seqs[(size_t)s].pages = pool->seqs[(size_t)seq].pages;
        pool->seqs[(size_t)s].open = true;
        for (const int32_t p : pool->seqs[(size_t)s].pages) ++pool->refs[(size_t)p];
        return s;
    });
}

int oasr_b200_kv_pool_close(oasr_kv_pool *pool, int32_t seq) {
    if (!pool || !pool->has(seq)) return OASR_STATUS_FAILED;
    return guarded([&]() -> int32_t {
        oasr_kv_pool::Seq &q = pool->seqs[(size_t)seq];
        for (const int32_t p : q.pages) pool->drop(p);
        q.pages.clear();
        q.open = false;
        return OASR_STATUS_SUCCESS;
    });
}

int32_t oasr_b200_kv_pool_extend(oasr_kv_pool *pool, int32_t seq, int32_t from, int32_t to, int32_t *pairs, int32_t max_pairs) {
    if (!pool || !pool->has(seq) || from < 0 || to < from || max_pairs < 0 || (max_pairs && !pairs)) return OASR_STATUS_FAILED;
    if (to == from) return 0;
    return guarded([&]() -> int32_t {
        std::vector<int32_t> &own = pool->seqs[(size_t)seq].pages;
        const int32_t first = from / pool->page, last = (int32_t)(((int64_t)to + pool->page - 1) / pool->page), held = (int32_t)own.size();
        // positions before `from` have to be held, in whole pages
        if (last > pool->max_pages || from > (int64_t)held * pool->page) return OASR_STATUS_FAILED;
        // what it takes: new pages, and own ones in the place of shared pages that are written
        int32_t need = std::max(0, last - held), copies = 0;
        for (int32_t j = first; j < std::min(last, held); ++j)
            if (pool->refs[(size_t)own[(size_t)j]] > 1) {
                ++need;
                if (j == first && from % pool->page) ++copies;  // its rows before `from` stay
            }
        if (need > (int32_t)pool->free.size()) return OASR_STATUS_ALLOC_FAILED;
        if (copies > max_pairs) return OASR_STATUS_FAILED;
        own.reserve((size_t)std::max(last, held));
        int32_t n = 0;
        for (int32_t j = first; j < std::min(last, held); ++j) {
            const int32_t old = own[(size_t)j];
            if (pool->refs[(size_t)old] == 1) continue;
            own[(size_t)j] = pool->take();
            if (j == first && from % pool->page) {
                pairs[2 * n] = old;
                pairs[2 * n + 1] = own[(size_t)j];
                ++n;
            }
            pool->drop(old);
        }
        while ((int32_t)own.size() < last) own.push_back(pool->take());
        return n;
    });
}

int oasr_b200_kv_pool_truncate(oasr_kv_pool *pool, int32_t seq, int32_t n_pos) {
    if (!pool || !pool->has(seq) || n_pos < 0) return OASR_STATUS_FAILED;
    return guarded([&]() -> int32_t {
        std::vector<int32_t> &own = pool->seqs[(size_t)seq].pages;
        const size_t keep = (size_t)(((int64_t)n_pos + pool->page - 1) / pool->page);
        while (own.size() > keep) {
            pool->drop(own.back());
            own.pop_back();
        }
        return OASR_STATUS_SUCCESS;
    });
}

int32_t oasr_b200_kv_pool_table(const oasr_kv_pool *pool, int32_t seq, int32_t *row) {
    if (!pool || !pool->has(seq) || !row) return OASR_STATUS_FAILED;
    const std::vector<int32_t> &own = pool->seqs[(size_t)seq].pages;
    for (int32_t j = 0; j < pool->max_pages; ++j) row[j] = j < (int32_t)own.size() ? own[(size_t)j] : -1;
    return (int32_t)own.size();
}

}  // extern "C"
