// page_pool.cpp -- the host-side owner of a paged cache's page numbers: sequences, shared
// pages with their counts, copy-on-write, compaction.  It never touches the device: the copies
// that its calls need are queued as moves and drained by the caller (wisp_pages_copy).
//
// Free pages are handed out lowest first, so that a pool stays compact while sequences come
// and go, and the same calls give the same pages.

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <stdexcept>
#include <utility>
#include <vector>

#include "internal.h"

struct WispPagePool {
    struct Seq {
        bool open = false;
        int length = 0;
        std::vector<int> pages;
    };
    int n_pages, page_size;
    std::vector<int> refs;  // sequences that hold the page
    std::vector<int> held;  // queued moves that read it: it is not free before they are drained
    std::priority_queue<int, std::vector<int>, std::greater<int>> free_pages;
    std::vector<Seq> seqs;
    std::vector<std::pair<int, int>> moves;

    // (the free list's storage is as large as the pool: a push never allocates)
    void drop(int page) {
        if (--refs[page] == 0 && held[page] == 0) free_pages.push(page);
    }
    void release(int page) {
        if (--held[page] == 0 && refs[page] == 0) free_pages.push(page);
    }
    int take() {
        const int p = free_pages.top();
        free_pages.pop();
        refs[p] = 1;
        return p;
    }
};

namespace {

#define POOL_FAIL(code, ret, ...)            \
    do {                                     \
        WB_SET_ERR(err, code, __VA_ARGS__);  \
        return ret;                          \
    } while (0)

bool valid(const WispPagePool* p, int seq) {
    return p && seq >= 0 && seq < (int)p->seqs.size() && p->seqs[seq].open;
}

int new_seq(WispPagePool* p) {
    for (size_t i = 0; i < p->seqs.size(); ++i)
        if (!p->seqs[i].open) {
            p->seqs[i].open = true;
            return (int)i;
        }
    p->seqs.emplace_back();
    p->seqs.back().open = true;
    return (int)p->seqs.size() - 1;
}

}  // namespace

extern "C" WispPagePool* wisp_page_pool_create(int n_pages, int page_size, WispErrCtx* err) {
    if (n_pages <= 0 || page_size <= 0)
        POOL_FAIL(WISP_ERR_INVALID_ARG, nullptr, "page_pool: %d pages of %d positions", n_pages,
                  page_size);
    try {
        WispPagePool* p = new WispPagePool;
        p->n_pages = n_pages;
        p->page_size = page_size;
        try {
            p->refs.assign(n_pages, 0);
            p->held.assign(n_pages, 0);
            std::vector<int> all(n_pages);
            for (int i = 0; i < n_pages; ++i) all[i] = i;
            p->free_pages = decltype(p->free_pages)(std::greater<int>(), std::move(all));
        } catch (...) {
            delete p;
            throw;
        }
        return p;
    } catch (const std::bad_alloc&) {
        POOL_FAIL(WISP_ERR_OOM, nullptr, "page_pool: no host memory");
    }
}

extern "C" void wisp_page_pool_destroy(WispPagePool* p) { delete p; }

extern "C" int wisp_page_pool_free_pages(const WispPagePool* p) {
    return p ? (int)p->free_pages.size() : 0;
}

extern "C" int wisp_page_pool_open(WispPagePool* p, WispErrCtx* err) {
    if (!p) POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: NULL pool");
    try {
        return new_seq(p);
    } catch (const std::bad_alloc&) {
        POOL_FAIL(WISP_ERR_OOM, -1, "page_pool: no host memory");
    }
}

extern "C" WispError wisp_page_pool_extend(WispPagePool* p, int seq, int length, WispErrCtx* err) {
    if (!valid(p, seq))
        POOL_FAIL(WISP_ERR_INVALID_ARG, WISP_ERR_INVALID_ARG, "page_pool: no sequence %d", seq);
    WispPagePool::Seq& s = p->seqs[seq];
    if (length < s.length)
        POOL_FAIL(WISP_ERR_INVALID_ARG, WISP_ERR_INVALID_ARG,
                  "page_pool: extend of %d positions to %d (truncate shortens)", s.length, length);
    if (length == s.length) return WISP_OK;
    const size_t have = s.pages.size();
    const size_t want = std::max(have, ((size_t)length + p->page_size - 1) / p->page_size);
    // pages from the first new position on are written: shared ones get copies; only the page
    // that already holds positions has anything to copy
    const size_t first = s.length / p->page_size;
    size_t need = want - have;
    for (size_t i = first; i < have; ++i) need += p->refs[s.pages[i]] > 1;
    if (need > p->free_pages.size())
        POOL_FAIL(WISP_ERR_OOM, WISP_ERR_OOM, "page_pool: %zu pages needed, %zu free", need,
                  p->free_pages.size());
    try {
        s.pages.reserve(want);
        p->moves.reserve(p->moves.size() + 1);
    } catch (const std::bad_alloc&) {
        POOL_FAIL(WISP_ERR_OOM, WISP_ERR_OOM, "page_pool: no host memory");
    } catch (const std::length_error&) {
        POOL_FAIL(WISP_ERR_OOM, WISP_ERR_OOM, "page_pool: no host memory");
    }
    for (size_t i = first; i < have; ++i) {
        const int old = s.pages[i];
        if (p->refs[old] == 1) continue;
        const int fresh = p->take();
        s.pages[i] = fresh;
        if (i == first && s.length % p->page_size) {
            p->moves.emplace_back(old, fresh);
            ++p->held[old];
        }
        p->drop(old);
    }
    while (s.pages.size() < want) s.pages.push_back(p->take());
    s.length = length;
    return WISP_OK;
}

extern "C" WispError wisp_page_pool_truncate(WispPagePool* p, int seq, int length, WispErrCtx* err) {
    if (!valid(p, seq))
        POOL_FAIL(WISP_ERR_INVALID_ARG, WISP_ERR_INVALID_ARG, "page_pool: no sequence %d", seq);
    WispPagePool::Seq& s = p->seqs[seq];
    if (length < 0 || length > s.length)
        POOL_FAIL(WISP_ERR_INVALID_ARG, WISP_ERR_INVALID_ARG,
                  "page_pool: truncate of %d positions to %d", s.length, length);
    const size_t keep = ((size_t)length + p->page_size - 1) / p->page_size;
    while (s.pages.size() > keep) {
        p->drop(s.pages.back());
        s.pages.pop_back();
    }
    s.length = length;
    return WISP_OK;
}

extern "C" int wisp_page_pool_fork(WispPagePool* p, int seq, WispErrCtx* err) {
    if (!valid(p, seq)) POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: no sequence %d", seq);
    int id = -1;
    try {
        id = new_seq(p);
        p->seqs[id].pages = p->seqs[seq].pages;
    } catch (const std::bad_alloc&) {
        if (id >= 0) p->seqs[id] = WispPagePool::Seq();
        POOL_FAIL(WISP_ERR_OOM, -1, "page_pool: no host memory");
    }
    p->seqs[id].length = p->seqs[seq].length;
    for (int page : p->seqs[id].pages) ++p->refs[page];
    return id;
}

extern "C" WispError wisp_page_pool_close(WispPagePool* p, int seq, WispErrCtx* err) {
    if (!valid(p, seq))
        POOL_FAIL(WISP_ERR_INVALID_ARG, WISP_ERR_INVALID_ARG, "page_pool: no sequence %d", seq);
    for (int page : p->seqs[seq].pages) p->drop(page);
    p->seqs[seq] = WispPagePool::Seq();
    return WISP_OK;
}

extern "C" int wisp_page_pool_compact(WispPagePool* p, WispErrCtx* err) {
    if (!p) POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: NULL pool");
    if (!p->moves.empty())
        POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: compact with %zu moves queued",
                  p->moves.size());
    const int used = p->n_pages - (int)p->free_pages.size();
    try {
        std::vector<int> to(p->n_pages, -1);
        std::vector<std::pair<int, int>> moves;
        int hole = 0;
        for (int page = used; page < p->n_pages; ++page) {
            if (!p->refs[page]) continue;
            while (p->refs[hole]) ++hole;
            moves.emplace_back(page, hole);
            to[page] = hole++;
        }
        // the sources stay reserved (by their moves) until the moves are drained
        std::vector<int> left;
        left.reserve(p->n_pages);
        for (int page = 0; page < p->n_pages; ++page)
            if (!p->refs[page] && page >= used) left.push_back(page);
        decltype(p->free_pages) rest(std::greater<int>(), std::move(left));
        // nothing below allocates
        for (const auto& m : moves) {
            p->refs[m.second] = p->refs[m.first];
            p->refs[m.first] = 0;
            p->held[m.first] = 1;
        }
        for (auto& s : p->seqs)
            for (int& page : s.pages)
                if (to[page] >= 0) page = to[page];
        p->free_pages.swap(rest);
        p->moves.swap(moves);
    } catch (const std::bad_alloc&) {
        POOL_FAIL(WISP_ERR_OOM, -1, "page_pool: no host memory");
    }
    return used;
}

extern "C" int wisp_page_pool_length(const WispPagePool* p, int seq, WispErrCtx* err) {
    if (!valid(p, seq)) POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: no sequence %d", seq);
    return p->seqs[seq].length;
}

extern "C" int wisp_page_pool_pages(const WispPagePool* p, int seq, int* pages, int cap,
                                    WispErrCtx* err) {
    if (!valid(p, seq)) POOL_FAIL(WISP_ERR_INVALID_ARG, -1, "page_pool: no sequence %d", seq);
    const auto& v = p->seqs[seq].pages;
    for (size_t i = 0; pages && i < v.size() && (int)i < cap; ++i) pages[i] = v[i];
    return (int)v.size();
}

extern "C" int wisp_page_pool_queued(const WispPagePool* p, int* src, int* dst, int cap) {
    if (!p) return 0;
    for (int i = 0; src && dst && i < std::min(cap, (int)p->moves.size()); ++i) {
        src[i] = p->moves[i].first;
        dst[i] = p->moves[i].second;
    }
    return (int)p->moves.size();
}

extern "C" int wisp_page_pool_moves(WispPagePool* p, int* src, int* dst, int cap) {
    if (!p || !src || !dst || cap <= 0) return 0;
    const int n = std::min(cap, (int)p->moves.size());
    for (int i = 0; i < n; ++i) {
        src[i] = p->moves[i].first;
        dst[i] = p->moves[i].second;
    }
    for (int i = 0; i < n; ++i) p->release(src[i]);
    p->moves.erase(p->moves.begin(), p->moves.begin() + n);
    return n;
}
