// Plans of page copies: a request that goes on twice, and private pages moved to the front of a pool.  The copies themselves are
// warp34_kv_cache_copy_pages; nothing here touches the GPU.  The reference shares pages only through its radix tree
// (crates/warp34-host/src/radix.rs:1129-1157) and has no counterpart of either.
#include <algorithm>
#include <stdexcept>

#include "kv_host.h"

namespace warp34_host {

namespace {
// Rows of page `index` of a request that hold its first `tokens`.
size_t filled_rows(size_t tokens, size_t index, size_t page_size) {
    const size_t first = index * page_size;
    return tokens <= first ? 0 : std::min(page_size, tokens - first);
}
void add_copies(const RequestPages& parent, const std::vector<int32_t>& from, const std::vector<int32_t>& to, size_t page_size, PageCopies* out) {
    for (size_t i = parent.protected_pages; i < to.size(); ++i) out->add(from[i], to[i], (int32_t)filled_rows(parent.token_ids.size(), i, page_size));
}
}  // namespace

bool fork_request_pages(KvPool& pool, PrefixPageCache& cache, const RequestPages& parent, RequestPages* child, PageCopies* copies, KvPool* draft_pool,
                        PageCopies* draft_copies) {
    const size_t page_size = parent.page_size ? parent.page_size : cache.page_size();
    const size_t needed = std::max((parent.token_ids.size() + page_size - 1) / page_size, parent.protected_pages);
    // the draft model may have no pages, or the prefix's alone
    const size_t drafts = std::min(parent.draft_pages.size(), needed), shared_drafts = std::min(drafts, parent.protected_pages);
    if (parent.kv_pages.size() < needed) throw std::invalid_argument("fork_request_pages: fewer pages than committed tokens");
    if (drafts > shared_drafts && (!draft_pool || !draft_copies))
        throw std::invalid_argument("fork_request_pages: private draft pages and no draft pool");
    RequestPages r;
    r.token_ids = parent.token_ids;
    r.protected_pages = parent.protected_pages;
    r.last_locked_node = parent.last_locked_node;
    r.page_size = page_size;
    r.kv_pages.assign(parent.kv_pages.begin(), parent.kv_pages.begin() + (long)parent.protected_pages);
    r.draft_pages.assign(parent.draft_pages.begin(), parent.draft_pages.begin() + (long)shared_drafts);
    const auto give_back = [&]() {
        for (size_t i = shared_drafts; i < r.draft_pages.size(); ++i) draft_pool->free_page(r.draft_pages[i]);
        return false;
    };
    while (r.draft_pages.size() < drafts) {
        const auto page = draft_pool->alloc_page();
        if (!page) return give_back();
        r.draft_pages.push_back(*page);
    }
    // the parent's lock keeps the shared prefix where it is while others make room
    if (!reserve_kv_pages_from(pool, cache, &r.kv_pages, needed)) return give_back();
    if (r.last_locked_node != 0) cache.inc_lock_ref(r.last_locked_node);
    add_copies(parent, parent.kv_pages, r.kv_pages, page_size, copies);
    if (drafts > shared_drafts) add_copies(parent, parent.draft_pages, r.draft_pages, page_size, draft_copies);
    *child = std::move(r);
    return true;
}

size_t pack_request_pages(KvPool& pool, const std::vector<RequestPages*>& requests, size_t below, PageCopies* copies,
                          const std::vector<size_t>* written_tokens) {
    if (written_tokens && written_tokens->size() != requests.size())
        throw std::invalid_argument("pack_request_pages: written tokens of other requests");
    std::vector<int32_t> left;  // freed behind the last move, so that no page is taken and given in one batch of copies
    size_t without = 0;
    for (size_t n = 0; n < requests.size(); ++n) {
        RequestPages* const r = requests[n];
        const size_t page_size = r->page_size ? r->page_size : pool.block_size;
        const size_t tokens = std::max(r->token_ids.size(), written_tokens ? (*written_tokens)[n] : 0);
        for (size_t i = r->protected_pages; i < r->kv_pages.size(); ++i) {
            int32_t& page = r->kv_pages[i];
            if (page < 0 || (size_t)page < below) continue;
            const auto to = without ? std::optional<int32_t>() : pool.alloc_page();
            if (!to || (size_t)*to >= below) {  // the lowest free page: there is none further down
                if (to) pool.free_page(*to);
                ++without;
                continue;
            }
            copies->add(page, *to, (int32_t)filled_rows(tokens, i, page_size));
            left.push_back(page);
            page = *to;
        }
    }
    for (int32_t page : left) pool.free_page(page);
    return without;
}

}  // namespace warp34_host
