// Which page of a cache belongs to which sequence (phx_pages_* of
// include/phobos_hip.h): reference counts, copies on write, compaction.  Host
// work only; phx_pages_apply launches the copies.
//
// A pending copy holds its source and its destination: neither is given out
// again before the copy has been launched, so that no destination is ever
// another's source or destination, and copies can run in any order.  A copy of
// a page that is itself the destination of a pending one is taken from that
// one's source.
#include <algorithm>
#include <exception>
#include <functional>
#include <mutex>
#include <unordered_map>
#include <vector>

#include "phx_internal.h"

using namespace phx;

namespace {
struct Sequence {
    std::vector<int32_t> pages;
    int64_t tokens = 0;
};
struct Copy {
    int32_t src, dst;
};
}  // namespace

struct phx_pages_s {
    std::mutex mu;
    int32_t page_tokens = 0;
    std::vector<int32_t> refs;   // sequences that have the page
    std::vector<int32_t> holds;  // pending copies that read or write it
    std::vector<int32_t> free;   // a heap, lowest first, with room for every page
    std::vector<Copy> pending;
    std::unordered_map<int64_t, Sequence> seqs;
    int64_t next = 0;

    int32_t take() {
        std::pop_heap(free.begin(), free.end(), std::greater<int32_t>());
        const int32_t page = free.back();
        free.pop_back();
        refs[page] = 1;
        return page;
    }
    void give(int32_t page) {
        if (refs[page] || holds[page]) return;
        free.push_back(page);
        std::push_heap(free.begin(), free.end(), std::greater<int32_t>());
    }
    void drop(int32_t page) {
        --refs[page];
        give(page);
    }
    void done() {  // the pending copies are on their way
        for (const Copy &c : pending) {
            --holds[c.src];
            give(c.src);
            --holds[c.dst];
            give(c.dst);
        }
        pending.clear();
    }
};

namespace {

// Runs body(pages) under the pool's lock; no exception leaves it.
template <typename F>
int with_pool(phx_pages p, const char *who, F body) {
    if (!p) return set_error(PHX_E_INVALID, "%s: null pool", who);
    try {
        std::lock_guard<std::mutex> lock(p->mu);
        return body(*p);
    } catch (const std::exception &e) {
        return set_error(PHX_E_EXHAUSTED, "%s: %s", who, e.what());
    }
}

Sequence *find(phx_pages_s &p, int64_t seq, const char *who, int *rc) {
    auto it = p.seqs.find(seq);
    *rc = it == p.seqs.end()
              ? set_error(PHX_E_INVALID, "%s: no sequence %lld", who, (long long)seq)
              : PHX_OK;
    return it == p.seqs.end() ? nullptr : &it->second;
}

}  // namespace

extern "C" {

int phx_pages_create(phx_pages *out, int32_t pages, int32_t page_tokens) {
    if (!out || pages < 1 || page_tokens < 1)
        return set_error(PHX_E_INVALID, "pages_create: %d pages of %d tokens", pages, page_tokens);
    phx_pages_s *p = nullptr;
    try {
        p = new phx_pages_s;
        p->page_tokens = page_tokens;
        p->refs.assign((size_t)pages, 0);
        p->holds.assign((size_t)pages, 0);
        p->free.resize((size_t)pages);
        for (int32_t i = 0; i < pages; ++i) p->free[i] = i;  // ascending: a heap
    } catch (const std::exception &e) {
        delete p;
        return set_error(PHX_E_EXHAUSTED, "pages_create: %s", e.what());
    }
    *out = p;
    return PHX_OK;
}

int phx_pages_destroy(phx_pages p) {
    delete p;
    return PHX_OK;
}

int phx_pages_new(phx_pages p, int64_t *seq) {
    return with_pool(p, "pages_new", [&](phx_pages_s &p) {
        if (!seq) return set_error(PHX_E_INVALID, "pages_new: null result");
        p.seqs.emplace(p.next, Sequence{});
        *seq = p.next++;
        return PHX_OK;
    });
}

int phx_pages_resize(phx_pages p, int64_t seq, int64_t tokens) {
    return with_pool(p, "pages_resize", [&](phx_pages_s &p) {
        int rc;
        Sequence *s = find(p, seq, "pages_resize", &rc);
        if (!s) return rc;
        const int64_t P = p.page_tokens, total = (int64_t)p.refs.size();
        if (tokens < 0)
            return set_error(PHX_E_INVALID, "pages_resize: %lld tokens", (long long)tokens);
        const int64_t need = tokens / P + (tokens % P != 0), have = (int64_t)s->pages.size();
        if (tokens <= s->tokens) {
            for (int64_t i = need; i < have; ++i) p.drop(s->pages[i]);
            s->pages.resize((size_t)need);
            s->tokens = tokens;
            return PHX_OK;
        }
        // the last page is written next: it has to be the sequence's own
        const bool copy = s->tokens % P && p.refs[s->pages.back()] > 1;
        const int64_t take = need - have + copy;
        if (need > total || take > (int64_t)p.free.size())
            return set_error(PHX_E_EXHAUSTED, "pages exhausted: %lld more needed, %zu of %lld free",
                             (long long)take, p.free.size(), (long long)total);
        s->pages.reserve((size_t)need);  // nothing throws from here on
        if (copy) {
            p.pending.reserve(p.pending.size() + 1);
            const int32_t old = s->pages.back(), own = p.take();
            int32_t src = old;
            for (const Copy &c : p.pending)
                if (c.dst == old) src = c.src;
            p.pending.push_back({src, own});
            ++p.holds[src];
            ++p.holds[own];
            s->pages.back() = own;
            p.drop(old);
        }
        for (int64_t i = have; i < need; ++i) s->pages.push_back(p.take());
        s->tokens = tokens;
        return PHX_OK;
    });
}

int phx_pages_fork(phx_pages p, int64_t seq, int64_t *child) {
    return with_pool(p, "pages_fork", [&](phx_pages_s &p) {
        int rc;
        Sequence *s = find(p, seq, "pages_fork", &rc);
        if (!s) return rc;
        if (!child) return set_error(PHX_E_INVALID, "pages_fork: null result");
        Sequence copy = *s;
        for (int32_t page : copy.pages)
            if (p.refs[page] == INT32_MAX)
                return set_error(PHX_E_EXHAUSTED, "pages_fork: page %d has too many owners", page);
        auto it = p.seqs.emplace(p.next, std::move(copy)).first;
        for (int32_t page : it->second.pages) ++p.refs[page];
        *child = p.next++;
        return PHX_OK;
    });
}

int phx_pages_free(phx_pages p, int64_t seq) {
    return with_pool(p, "pages_free", [&](phx_pages_s &p) {
        int rc;
        Sequence *s = find(p, seq, "pages_free", &rc);
        if (!s) return rc;
        for (int32_t page : s->pages) p.drop(page);
        p.seqs.erase(seq);
        return PHX_OK;
    });
}

int phx_pages_compact(phx_pages p) {
    return with_pool(p, "pages_compact", [&](phx_pages_s &p) {
        if (!p.pending.empty())
            return set_error(PHX_E_INVALID, "pages_compact: %zu copies are pending",
                             p.pending.size());
        const int32_t total = (int32_t)p.refs.size();
        int32_t used = 0;
        for (int32_t r : p.refs) used += r > 0;
        std::vector<int32_t> to((size_t)total, -1);
        std::vector<Copy> moves;
        for (int32_t hole = 0, page = used; page < total; ++page) {
            if (!p.refs[page]) continue;
            while (p.refs[hole]) ++hole;
            to[page] = hole;
            moves.push_back({page, hole++});
        }
        for (const Copy &m : moves) {  // nothing throws from here on
            p.refs[m.dst] = p.refs[m.src];
            p.refs[m.src] = 0;
            p.holds[m.src] = p.holds[m.dst] = 1;
        }
        for (auto &kv : p.seqs)
            for (int32_t &page : kv.second.pages)
                if (to[page] >= 0) page = to[page];
        p.free.clear();
        for (int32_t page = used; page < total; ++page)
            if (!p.holds[page]) p.free.push_back(page);
        p.pending.swap(moves);
        return PHX_OK;
    });
}

int phx_pages_table(phx_pages p, int64_t seq, int32_t *out, int64_t cap, int64_t *count) {
    return with_pool(p, "pages_table", [&](phx_pages_s &p) {
        int rc;
        Sequence *s = find(p, seq, "pages_table", &rc);
        if (!s) return rc;
        if (cap < 0 || (cap && !out))
            return set_error(PHX_E_INVALID, "pages_table: room for %lld", (long long)cap);
        const size_t n = s->pages.size();
        std::copy_n(s->pages.begin(), std::min(n, (size_t)cap), out);
        if (count) *count = (int64_t)n;
        return PHX_OK;
    });
}

int phx_pages_stats(phx_pages p, int64_t *used, int64_t *top, int64_t *pending) {
    return with_pool(p, "pages_stats", [&](phx_pages_s &p) {
        int64_t high = 0;
        for (size_t i = 0; i < p.refs.size(); ++i)
            if (p.refs[i] || p.holds[i]) high = (int64_t)i + 1;
        if (used) *used = (int64_t)(p.refs.size() - p.free.size());
        if (top) *top = high;
        if (pending) *pending = (int64_t)p.pending.size();
        return PHX_OK;
    });
}

int phx_pages_pending(phx_pages p, int32_t *src, int32_t *dst, int64_t cap, int64_t *count,
                      int clear) {
    return with_pool(p, "pages_pending", [&](phx_pages_s &p) {
        if (cap < 0 || (cap && (!src || !dst)))
            return set_error(PHX_E_INVALID, "pages_pending: room for %lld", (long long)cap);
        for (size_t i = 0; i < std::min(p.pending.size(), (size_t)cap); ++i) {
            src[i] = p.pending[i].src;
            dst[i] = p.pending[i].dst;
        }
        if (count) *count = (int64_t)p.pending.size();
        if (clear && p.pending.size() > (size_t)cap)
            return set_error(PHX_E_INVALID, "pages_pending: %zu copies, room for %lld",
                             p.pending.size(), (long long)cap);
        if (clear) p.done();
        return PHX_OK;
    });
}

int phx_pages_apply(phx_pages p, phx_stream s, uint64_t pool, size_t page_bytes, int64_t layers,
                    uint64_t layer_stride) {
    return with_pool(p, "pages_apply", [&](phx_pages_s &p) {
        if (layers < 1 && !p.pending.empty())
            return set_error(PHX_E_INVALID, "pages_apply: %zu copies are pending in %lld layers",
                             p.pending.size(), (long long)layers);
        // captured, they would not have run, and every replay would run them again
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (s && !p.pending.empty()) {
            hipError_t e = hipStreamIsCapturing((hipStream_t)s, &capture);
            if (e != hipSuccess) return hip_error(e, "hipStreamIsCapturing");
        }
        if (capture != hipStreamCaptureStatusNone)
            return set_error(PHX_E_INVALID, "pages_apply: %zu copies are pending on a stream that is "
                             "being captured", p.pending.size());
        std::vector<int32_t> src, dst;
        for (const Copy &c : p.pending) {
            src.push_back(c.src);
            dst.push_back(c.dst);
        }
        if (int rc = phx_pages_copy(s, pool, (int64_t)p.refs.size(), page_bytes, src.data(),
                                    dst.data(), (int64_t)src.size(), layers, layer_stride))
            return rc;
        p.done();
        return PHX_OK;
    });
}

}  // extern "C"
