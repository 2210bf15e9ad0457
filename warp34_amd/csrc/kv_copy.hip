// Pages of a cache copied in all layers: rows 0 .. rows[i] - 1 of every head of page src_pages[i] to page dst_pages[i], K and V.
//
// Bound: HBM, each byte read once and written once: 128 pages of 64 rows and eight heads in 24 layers of BF16, 805 MB, 155 us (5.2 TB/s, the
// rate of a large copy); 24 pages, most of them partly filled, of 40 TQ4 layers, 30 MB, 7.4 us, of which a launch and a round trip are 4.
#include "attn_launch.h"
#include "kv_common.h"

namespace w34 {

// One slab.  The descriptors of 48 layers (96 slabs) fit the 4 096 bytes of a kernel's arguments, so that they need no memory of their own
// and are recorded with a captured launch.
struct CopySlab {
    uint64_t base, page_stride, head_stride;
    uint32_t token_stride, row_bytes;
};
constexpr int kCopySlabs = 96;
constexpr int kCopyMostPairs = 1 << 24;
struct CopyArgs {
    const int32_t *src_pages, *dst_pages, *rows;
    int num_pairs, heads, block_size, reserved;
    CopySlab slabs[kCopySlabs];
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

// A workgroup copies the rows of one head of one page of one slab, GRAIN bytes a thread at a time.  Rows that lie one behind the other are one
// run, whose last bytes (rows of 132 bytes end anywhere) go by in twos.
template <int GRAIN>
struct CopyWord;
template <>
struct CopyWord<16> {
    typedef uint4 type;
};
template <>
struct CopyWord<4> {
    typedef uint32_t type;
};
template <>
struct CopyWord<2> {
    typedef uint16_t type;
};

template <int GRAIN>
__global__ __launch_bounds__(256) void kv_copy_kernel(const CopyArgs a) {
    typedef typename CopyWord<GRAIN>::type W;
    uint32_t at = blockIdx.x;
    const int head = (int)(at % (uint32_t)a.heads);
    at /= (uint32_t)a.heads;
    const int pair = (int)(at % (uint32_t)a.num_pairs);
    const CopySlab& s = a.slabs[at / (uint32_t)a.num_pairs];
    const int src = a.src_pages[pair], dst = a.dst_pages[pair];
    const int rows = a.rows == nullptr ? a.block_size : min(a.rows[pair], a.block_size);
    if (src < 0 || dst < 0 || src == dst || rows <= 0) return;
    const uint8_t* from = reinterpret_cast<const uint8_t*>((uintptr_t)(s.base + (uint64_t)src * s.page_stride + (uint64_t)head * s.head_stride));
    uint8_t* to = reinterpret_cast<uint8_t*>((uintptr_t)(s.base + (uint64_t)dst * s.page_stride + (uint64_t)head * s.head_stride));
    const bool one_run = s.token_stride == s.row_bytes;
    const uint64_t run = one_run ? (uint64_t)rows * s.row_bytes : s.row_bytes;
    const uint64_t words = run / GRAIN, tail = (run - words * GRAIN) / 2;
    for (int r = 0; r < (one_run ? 1 : rows); ++r) {
        const W* f = reinterpret_cast<const W*>(from + (uint64_t)r * s.token_stride);
        W* t = reinterpret_cast<W*>(to + (uint64_t)r * s.token_stride);
        for (uint64_t i = threadIdx.x; i < words; i += 256) t[i] = f[i];
        if (threadIdx.x < tail)
            reinterpret_cast<uint16_t*>(t + words)[threadIdx.x] = reinterpret_cast<const uint16_t*>(f + words)[threadIdx.x];
    }
}

// bytes of a row as the append lays it out; 0: there is no such row
static uint32_t copy_row_bytes(int format, int head_dim) {
    switch (format) {
        case WARP34_KV_FORMAT_FP16:
        case WARP34_KV_FORMAT_BF16: return 2u * (uint32_t)head_dim;
        case WARP34_KV_FORMAT_TQ4: return head_dim % 128 ? 0 : 66u * (uint32_t)(head_dim / 128);
        case WARP34_KV_FORMAT_Q8_0: return head_dim % 64 ? 0 : 68u * (uint32_t)(head_dim / 64);
        case WARP34_KV_FORMAT_FP8_E4M3: return head_dim % 256 ? 0 : 264u * (uint32_t)(head_dim / 256);
        default: return 0;
    }
}

static int kv_copy_entry(const warp34_exec* ex, const warp34_kv_layer_layout* layouts, int num_layers, const int32_t* src_pages, const int32_t* dst_pages,
                         const int32_t* rows, int num_pairs) {
    if (!ex || num_layers < 0 || (num_layers > 0 && !layouts) || (num_pairs > 0 && (!src_pages || !dst_pages)) || num_pairs > kCopyMostPairs)
        return (int)hipErrorInvalidValue;
    for (int l = 0; l < num_layers; ++l) {  // everything is looked at before anything is launched
        const warp34_kv_layer_layout& y = layouts[l];
        if (!y.k_base || !y.v_base || y.local_kv_heads <= 0 || y.block_size <= 0 || y.head_dim <= 0 || y.head_dim > 4096) return (int)hipErrorInvalidValue;
        if (!grid_fits((long long)kCopySlabs * y.local_kv_heads, 256)) return (int)hipErrorInvalidValue;
        const uint32_t kr = copy_row_bytes(y.k_format, y.head_dim), vr = copy_row_bytes(y.v_format, y.head_dim);
        if (!kr || !vr || y.k_token_stride_bytes < kr || y.v_token_stride_bytes < vr || (y.k_token_stride_bytes | y.v_token_stride_bytes) >> 31)
            return (int)hipErrorNotSupported;
        if ((y.k_base | y.v_base | y.k_page_stride_bytes | y.v_page_stride_bytes | y.k_head_stride_bytes | y.v_head_stride_bytes | y.k_token_stride_bytes |
             y.v_token_stride_bytes) & 1u)
            return (int)hipErrorNotSupported;
    }
    if (num_pairs <= 0) return 0;
    for (int l = 0; l < num_layers;) {
        CopyArgs a{src_pages, dst_pages, rows, num_pairs, layouts[l].local_kv_heads, layouts[l].block_size, 0, {}};
        int n = 0;
        uint64_t bits = 0;  // what addresses and runs are made of
        for (; l < num_layers && n < kCopySlabs && layouts[l].local_kv_heads == a.heads && layouts[l].block_size == a.block_size; ++l) {
            const warp34_kv_layer_layout& y = layouts[l];
            a.slabs[n++] = {y.k_base, y.k_page_stride_bytes, y.k_head_stride_bytes, (uint32_t)y.k_token_stride_bytes, copy_row_bytes(y.k_format, y.head_dim)};
            a.slabs[n++] = {y.v_base, y.v_page_stride_bytes, y.v_head_stride_bytes, (uint32_t)y.v_token_stride_bytes, copy_row_bytes(y.v_format, y.head_dim)};
            for (int s = n - 2; s < n; ++s) {
                bits |= a.slabs[s].base | a.slabs[s].page_stride | a.slabs[s].head_stride;
                if (a.slabs[s].token_stride != a.slabs[s].row_bytes) bits |= a.slabs[s].token_stride;
            }
        }
        const int most = (int)(((1ll << 32) / 256 - 1) / ((long long)n * a.heads));  // pairs that a launch has room for
        for (int first = 0; first < num_pairs; first += most) {
            a.src_pages = src_pages + first, a.dst_pages = dst_pages + first, a.rows = rows ? rows + first : nullptr;
            a.num_pairs = min(most, num_pairs - first);
            const dim3 grid((unsigned)((long long)n * a.num_pairs * a.heads));
            if ((bits & 15u) == 0) hipLaunchKernelGGL(kv_copy_kernel<16>, grid, dim3(256), 0, (hipStream_t)ex->stream, a);
            else if ((bits & 3u) == 0) hipLaunchKernelGGL(kv_copy_kernel<4>, grid, dim3(256), 0, (hipStream_t)ex->stream, a);
            else hipLaunchKernelGGL(kv_copy_kernel<2>, grid, dim3(256), 0, (hipStream_t)ex->stream, a);
            const int rc = (int)hipGetLastError();
            if (rc) return rc;
        }
    }
    return 0;
}

}  // namespace w34

extern "C" int warp34_kv_cache_copy_pages(const warp34_exec* ex, const warp34_kv_layer_layout* layouts, int num_layers, const int32_t* src_pages,
                                          const int32_t* dst_pages, const int32_t* rows, int num_pairs) {
    return w34::kv_copy_entry(ex, layouts, num_layers, src_pages, dst_pages, rows, num_pairs);
}
