// The walk of the scored decode kernels over a request's block table, on the CPU: PageWalk, page_slot, the TQ4 kernel's `locate` and the line of
// its loop that moves to the next unit are the kernels' own text (page_walk.inc and the others, cut out of the sources by the test).  Every lane
// that the walk reads an entry from is checked: one of 64, and its entry one of the pages that the chunk's keys lie in.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <utility>

using std::max;

struct Layout {
    uint64_t k_base = 0, v_base = 0, k_head_stride_bytes = 0, v_head_stride_bytes = 0, k_page_stride_bytes = 1 << 20, v_page_stride_bytes = 1 << 20;
    int block_size = 0;
};
struct Batch {
    const int32_t* block_tables = nullptr;
    int max_blocks_per_req = 1 << 20;
};
struct ScoredParams {
    Layout L;
    Batch B;
    uint32_t block_magic = 0;
};
struct ScoredTile {
    int req = 0;
};
typedef const uint8_t slab_byte;
static const slab_byte* slab_at(uint64_t a) { return reinterpret_cast<const uint8_t*>((uintptr_t)a); }
static uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }

// The block table is its own index: entry i is i, so that an address tells the page.  first, last: the pages of the chunk's keys.
static int g_first, g_last, g_block, g_begin, g_end, g_wave;
static int entry(int base, int lane) {
    if (lane < 0 || lane >= 64 || base + lane < g_first || base + lane > g_last) {
        std::printf("block %d, half units [%d, %d), wave %d: lane %d of the entries from %d on, pages in use %d to %d\n", g_block, g_begin, g_end,
                    g_wave, lane, base, g_first, g_last);
        std::exit(1);
    }
    return base + lane;
}
#define __device__
#define __forceinline__ inline
#define __builtin_amdgcn_readlane(value, lane) entry(slot_base, (lane))
#include "page_slot.inc"
#include "page_walk.inc"

static uint64_t address(const ScoredParams& P, int half, int row_bytes) {
    const int pos = half * 16, page = pos / P.L.block_size;
    return (uint64_t)page * P.L.k_page_stride_bytes + (uint64_t)(pos - page * P.L.block_size) * row_bytes;
}
static void same(const slab_byte* got, uint64_t want, int half) {
    if ((uint64_t)(uintptr_t)got != want) {
        std::printf("block %d, half units [%d, %d), wave %d: not the rows of half unit %d\n", g_block, g_begin, g_end, g_wave, half);
        std::exit(1);
    }
}

// A wave of the TQ4 kernel: units of two half units, every eighth
static void tq4_wave(const ScoredParams& P, int begin, int end, int wave) {
    constexpr int lane = 0, kScoredWaves = 8;
    PageWalk walk;
    walk.start(P, ScoredTile{}, 0, begin, lane);
    const slab_byte* k_rows[2] = {nullptr, nullptr};
    const slab_byte* v_rows[2] = {nullptr, nullptr};
#include "tq4_locate.inc"
    int half = begin + 2 * wave;
    if (half < end) locate(half);
    while (half < end) {
        const int next = half + 2 * kScoredWaves;
        const bool more = next < end;
        for (int h = 0; h < 2; ++h) {
            const int of = h == 1 && half + 1 < end ? half + 1 : half;
            same(k_rows[h], address(P, of, 132), of);
            same(v_rows[h], address(P, of, 132), of);
        }
#include "tq4_next.inc"
        half = next;
    }
}
// A wave of the other one: every eighth half unit
static void rows_wave(const ScoredParams& P, int begin, int end, int wave) {
    PageWalk walk;
    walk.start(P, ScoredTile{}, 0, begin, 0);
    for (int half = begin + wave; half < end; half += 8) {
        const slab_byte *k_rows, *v_rows;
        walk.locate(P, half, 512, 0, k_rows, v_rows);
        same(k_rows, address(P, half, 512), half);
        same(v_rows, address(P, half, 512), half);
    }
}

int main() {
    long walks = 0;
    for (const int block : {16, 32, 48, 64, 80, 96, 112, 128, 192, 256}) {
        ScoredParams P;
        P.L.block_size = block;
        P.block_magic = (uint32_t)((1ull << 32) / (uint32_t)block);
        const int page_halves = block / 16;
        for (int begin = 0; begin < std::min(3 * page_halves, 24); ++begin)
            for (int halves = 0; halves <= 2200; halves += halves < 40 || block < 96 ? 1 : 1 + halves % 3) {
                g_block = block, g_begin = begin, g_end = begin + halves;
                g_first = begin / page_halves, g_last = (begin + std::max(halves, 1) - 1) / page_halves;
                for (g_wave = 0; g_wave < 8; ++g_wave) {
                    tq4_wave(P, begin, begin + halves, g_wave);
                    rows_wave(P, begin, begin + halves, g_wave);
                    ++walks;
                }
            }
    }
    std::printf("%ld walks\n", walks);
}
