// Forked requests and packed pools: which pages are shared, taken, copied and freed.
// Prints one "ok <name>" line per passing test; exits non-zero at the first failure.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <stdexcept>
#include <string>

#include "../../warp34_amd/host/kv_host.h"

using namespace warp34_host;
typedef std::vector<int32_t> Pages;

#define CHECK(cond)                                                       \
    do {                                                                  \
        if (!(cond)) {                                                    \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            std::exit(1);                                                 \
        }                                                                 \
    } while (0)

struct HostAllocator final : DeviceAllocator {
    int alloc(int, size_t, uint64_t* addr) override {
        *addr = next += 1 << 20;
        return 0;
    }
    void release(int, uint64_t) override {}
    uint64_t next = 1 << 20;
};
static KvPool make_pool(HostAllocator& ha, size_t pages) {
    KvPool pool;
    CHECK(!KvPool::new_target_full_attn(&pool, ha, 0, {0}, 2, 256, 16, pages, KvFormatPolicy::Tq4All, false));
    return pool;
}
static std::vector<int32_t> tokens(size_t n, int32_t from) {
    std::vector<int32_t> t(n);
    for (size_t i = 0; i < n; ++i) t[i] = from + (int32_t)i;
    return t;
}
static void check_disjoint(const PageCopies& c) {
    CHECK(c.src.size() == c.dst.size() && c.src.size() == c.rows.size());
    std::set<int32_t> src(c.src.begin(), c.src.end()), dst(c.dst.begin(), c.dst.end());
    CHECK(dst.size() == c.dst.size());
    for (int32_t d : dst) CHECK(!src.count(d));
    for (int32_t n : c.rows) CHECK(n >= 1 && n <= 16);
}

static void test_fork_of_a_private_request() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 12);
    PrefixPageCache cache(16, 16);
    RequestPages a, b;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 5));  // one page more than the 50 tokens fill
    a.token_ids = tokens(50, 1);
    PageCopies c;
    CHECK(fork_request_pages(pool, cache, a, &b, &c));
    CHECK((b.kv_pages == Pages{5, 6, 7, 8}) && b.token_ids == a.token_ids && b.protected_pages == 0 && b.page_size == 16);
    CHECK((c.src == Pages{0, 1, 2, 3}) && c.dst == b.kv_pages && (c.rows == Pages{16, 16, 16, 2}));
    CHECK(pool.free_count() == 3);
    check_disjoint(c);
    // a third one does not fit: nothing is taken, the child is left alone
    RequestPages d;
    d.token_ids = {7};
    CHECK(!fork_request_pages(pool, cache, a, &d, &c));
    CHECK(pool.free_count() == 3 && c.src.size() == 4 && d.token_ids == std::vector<int32_t>{7});
    std::puts("ok fork_of_a_private_request");
}

static void test_fork_behind_a_shared_prefix() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 12), drafts = make_pool(ha, 12);
    PrefixPageCache cache(16, 16);
    RequestPages a;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 3));
    CHECK(reserve_kv_pages_from(drafts, cache, &a.draft_pages, 3));
    a.token_ids = tokens(40, 1);
    a.donate_pages(cache, 32, 500, false);  // two whole pages are the tree's, the request goes on
    CHECK(a.protected_pages == 2 && cache.full_protected_pages() == 2);
    RequestPages b;
    PageCopies c, dc;
    bool threw = false;
    try {
        fork_request_pages(pool, cache, a, &b, &c);  // private draft pages and nowhere to copy them
    } catch (const std::invalid_argument&) {
        threw = true;
    }
    CHECK(threw && pool.free_count() == 9 && c.src.empty());
    CHECK(fork_request_pages(pool, cache, a, &b, &c, &drafts, &dc));
    CHECK((b.kv_pages == Pages{0, 1, 3}) && (c.src == Pages{2}) && (c.dst == Pages{3}) && (c.rows == Pages{8}));
    CHECK((b.draft_pages == Pages{0, 1, 3}) && (dc.src == Pages{2}) && (dc.dst == Pages{3}) && (dc.rows == Pages{8}));
    CHECK(b.protected_pages == 2 && b.last_locked_node == a.last_locked_node && cache.full_protected_pages() == 2);
    // each lets go of the prefix for itself: it stays locked until both have
    std::string why;
    free_kv_pages(pool, a.donate_pages(cache, 0, -1, true).freed_kv_pages);
    CHECK(cache.full_protected_pages() == 2 && cache.sanity_check(&why));
    free_kv_pages(pool, b.donate_pages(cache, 0, -1, true).freed_kv_pages);
    CHECK(cache.full_protected_pages() == 0 && cache.full_evictable_pages() == 2 && pool.free_count() == 10 && cache.sanity_check(&why));
    std::puts("ok fork_behind_a_shared_prefix");
}

static void test_fork_at_a_page_border_and_of_nothing() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 8);
    PrefixPageCache cache(16, 16);
    RequestPages a, b;
    PageCopies c;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 2));
    a.token_ids = tokens(32, 1);
    a.donate_pages(cache, 32, 1, false);
    CHECK(fork_request_pages(pool, cache, a, &b, &c));  // all of it is the tree's: nothing to copy
    CHECK(c.src.empty() && b.kv_pages == a.kv_pages && pool.free_count() == 6);
    RequestPages empty, child;
    CHECK(fork_request_pages(pool, cache, empty, &child, &c) && child.kv_pages.empty() && c.src.empty());
    RequestPages short_of_pages;
    short_of_pages.token_ids = tokens(17, 1);
    short_of_pages.kv_pages = {3};
    bool threw = false;
    try {
        fork_request_pages(pool, cache, short_of_pages, &child, &c);
    } catch (const std::invalid_argument&) {
        threw = true;
    }
    CHECK(threw);
    std::puts("ok fork_at_a_page_border_and_of_nothing");
}

static void test_fork_makes_room() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 6);
    PrefixPageCache cache(16, 16);
    RequestPages old;  // a finished request's two pages can be evicted
    CHECK(reserve_kv_pages_from(pool, cache, &old.kv_pages, 2));
    old.token_ids = tokens(32, 5000);
    old.donate_pages(cache, 32, 7, true);
    RequestPages a, b;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 3));
    a.token_ids = tokens(35, 1);
    PageCopies c;
    CHECK(fork_request_pages(pool, cache, a, &b, &c));  // one page was free, two come from the cache
    CHECK(b.kv_pages.size() == 3 && pool.free_count() == 0 && cache.cached_pages() == 0);
    check_disjoint(c);
    std::puts("ok fork_makes_room");
}

static void test_packing() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 200);
    PrefixPageCache cache(16, 16);
    std::vector<RequestPages> r(6);
    for (auto& x : r) {
        CHECK(reserve_kv_pages_from(pool, cache, &x.kv_pages, 30));
        x.token_ids = tokens(29 * 16 + 5, 1);
        x.page_size = 16;
    }
    for (int i : {0, 2, 3}) free_kv_pages(pool, r[i].kv_pages), r[i] = RequestPages();
    r[4].protected_pages = 4;  // pages 120 .. 123 are not the request's own
    const std::vector<RequestPages*> live = {&r[1], &r[4], &r[5]};
    PageCopies c;
    CHECK(pack_request_pages(pool, live, 90, &c) == 0);
    check_disjoint(c);
    CHECK(c.src.size() == 26 + 30 && c.dst[0] == 0 && c.rows[25] == 5);
    for (size_t i = 0; i < c.src.size(); ++i) CHECK(c.src[i] >= 90 && c.dst[i] < 90);
    CHECK((Pages(r[4].kv_pages.begin(), r[4].kv_pages.begin() + 4) == Pages{120, 121, 122, 123}) && r[1].kv_pages[0] == 30);
    std::set<int32_t> used;
    for (auto* x : live)
        for (int32_t p : x->kv_pages) CHECK(used.insert(p).second);
    CHECK(pool.free_count() == 200 - 90);
    for (size_t i = 0; i < c.src.size(); ++i) CHECK(used.count(c.dst[i]) && !used.count(c.src[i]));
    // again: nothing is left to move
    PageCopies again;
    CHECK(pack_request_pages(pool, live, 90, &again) == 0 && again.src.empty());
    // too little room: as many as there are places, the rest stay where they are
    PageCopies few;
    CHECK(pack_request_pages(pool, live, 40, &few) > 0);
    check_disjoint(few);
    CHECK(pool.free_count() == 200 - 90);
    std::puts("ok packing");
}

static void test_packing_moves_empty_pages_without_a_copy() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 20);
    PrefixPageCache cache(16, 16);
    RequestPages a, b;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 4));
    CHECK(reserve_kv_pages_from(pool, cache, &b.kv_pages, 3));
    b.token_ids = tokens(20, 1);  // two pages of tokens, one reserved
    b.page_size = 16;
    free_kv_pages(pool, a.kv_pages);
    PageCopies c;
    CHECK(pack_request_pages(pool, {&b}, 3, &c) == 0);
    CHECK((b.kv_pages == Pages{0, 1, 2}) && (c.src == Pages{4, 5}) && (c.dst == Pages{0, 1}) && (c.rows == Pages{16, 4}));
    CHECK(pool.free_count() == 17);
    std::puts("ok packing_moves_empty_pages_without_a_copy");
}

int main() {
    test_fork_of_a_private_request();
    test_fork_behind_a_shared_prefix();
    test_fork_at_a_page_border_and_of_nothing();
    test_fork_makes_room();
    test_packing();
    test_packing_moves_empty_pages_without_a_copy();
    std::puts("all page move tests passed");
    return 0;
}
