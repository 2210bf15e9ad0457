// Packed pools in the middle of a step, and forks for which the draft model's pool runs out.
// Prints one "ok <name>" line per passing test; exits non-zero at the first failure.
#include <cstdio>
#include <cstdlib>
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

// 30 committed tokens and five drafted ones whose rows are written: the drafted rows go with their pages, the last page's only rows are drafts.
static void test_rows_of_drafts_travel() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 20);
    PrefixPageCache cache(16, 16);
    RequestPages gone, a, b;
    CHECK(reserve_kv_pages_from(pool, cache, &gone.kv_pages, 5));
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 3));
    CHECK(reserve_kv_pages_from(pool, cache, &b.kv_pages, 2));
    a.token_ids.assign(30, 1), b.token_ids.assign(17, 2);
    a.page_size = b.page_size = 16;
    free_kv_pages(pool, gone.kv_pages);
    PageCopies c;
    const std::vector<size_t> written = {35, 0};  // never less than what is committed
    CHECK(pack_request_pages(pool, {&a, &b}, 5, &c, &written) == 0);
    CHECK((a.kv_pages == Pages{0, 1, 2}) && (b.kv_pages == Pages{3, 4}));
    CHECK((c.src == Pages{5, 6, 7, 8, 9}) && (c.dst == Pages{0, 1, 2, 3, 4}) && (c.rows == Pages{16, 16, 3, 16, 1}));
    std::puts("ok rows_of_drafts_travel");
}

static void test_written_tokens_of_other_requests() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 8);
    PrefixPageCache cache(16, 16);
    RequestPages a;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 3));
    a.page_size = 16;
    pool.free_page(0), a.kv_pages.erase(a.kv_pages.begin());
    PageCopies c;
    bool threw = false;
    const std::vector<size_t> written = {1, 2};
    try {
        pack_request_pages(pool, {&a}, 1, &c, &written);
    } catch (const std::invalid_argument&) {
        threw = true;
    }
    CHECK(threw && c.src.empty() && (a.kv_pages == Pages{1, 2}) && pool.free_count() == 6);
    std::puts("ok written_tokens_of_other_requests");
}

// The draft pool has one page where two are wanted: it is given back, and the target's pool and the child are left alone.
static void test_fork_gives_draft_pages_back() {
    HostAllocator ha;
    KvPool pool = make_pool(ha, 12), drafts = make_pool(ha, 3);
    PrefixPageCache cache(16, 16);
    RequestPages a, b;
    CHECK(reserve_kv_pages_from(pool, cache, &a.kv_pages, 2));
    CHECK(reserve_kv_pages_from(drafts, cache, &a.draft_pages, 2));
    a.token_ids.assign(20, 1);
    PageCopies c, dc;
    CHECK(!fork_request_pages(pool, cache, a, &b, &c, &drafts, &dc));
    CHECK(drafts.free_count() == 1 && pool.free_count() == 10 && c.src.empty() && dc.src.empty() && b.kv_pages.empty() && b.draft_pages.empty());
    // and where the target's pool is the one that has too few
    KvPool small = make_pool(ha, 3), enough = make_pool(ha, 8);
    RequestPages p;
    CHECK(reserve_kv_pages_from(small, cache, &p.kv_pages, 2));
    CHECK(reserve_kv_pages_from(enough, cache, &p.draft_pages, 2));
    p.token_ids.assign(20, 1);
    CHECK(!fork_request_pages(small, cache, p, &b, &c, &enough, &dc));
    CHECK(small.free_count() == 1 && enough.free_count() == 6 && c.src.empty() && dc.src.empty() && b.kv_pages.empty());
    std::puts("ok fork_gives_draft_pages_back");
}

int main() {
    test_rows_of_drafts_travel();
    test_written_tokens_of_other_requests();
    test_fork_gives_draft_pages_back();
    std::puts("all page row tests passed");
    return 0;
}
