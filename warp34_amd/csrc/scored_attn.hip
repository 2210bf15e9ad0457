// Scored paged attention: checks, dispatch and entry points.
#include <algorithm>
#include <cmath>

#include "attn_launch.h"
#include "scored_chunk.h"
#include "scored_decode_tq4.h"

namespace w34 {

constexpr int kDecodeCols = 16;  // query columns of a workgroup of the decode kernel (TQ4: kTq4Cols)

// Shortest chunks, in half units of 16 keys.  Decode, us a call at 8 / 4 / 3 / 2: 700 FP16 keys 12.5 / 10.7 / 10.3 / 9.9, 3 000 TQ4 keys
// 13.7 / 13.2 / 13.6 / 14.8, 4 requests of 300 to 900 BF16 keys 10.0 / 9.2 / 9.8 / 9.7.  Chunk kernel at 64 / 32 / 16 / 8, 32 tokens of
// BF16: on 16 000 keys 99 / 56 / 46 / 53, 8 requests on 4 000 92 / 69 / 61 / 66, 2 on 1 000 72 / 53 / 39 / 32.
constexpr int kDecodeMinHalves = 4, kChunkMinHalves = 16;
// Up to so many half units, two for each wave, the keys of a decode call are not cut: the join's launch takes longer.  us a call, whole /
// cut: 100 FP16 keys 7.6 / 10.3, 250 10.2 / 10.4, 330 12.5 / 10.7; TQ4 8.7 / 12.4, 11.6 / 12.5, 13.2 / 12.7.
constexpr int kDecodeWhole = 16;

// Batches of up to so many tiles have a workgroup a column to join their chunks, others a wave a column: a few tiles have many chunks each.
// us a call, workgroups / waves: decode, 1 tile of 131 072 TQ4 keys 28.4 / 41.6, 10 tiles 34.3 / 37.8, 16 tiles 26.6 / 25.7, 32 tiles 55.7 /
// 51.1; chunks, 1 tile of 16 000 keys 47 / 102, 8 tiles 51 / 45 and 60 / 62, 16 tiles 94 / 77.
constexpr int kSpreadTiles = 12, kSpreadChunkTiles = 8;

// Requests with at least this many query columns (tokens x q heads of a kv head), a full tile, go through the chunk kernel.  us a call,
// decode / chunk kernel, for 1 request on 16 000 keys, 8 on 4 000, 2 on 1 000, 1 on 64 000.  256 columns: BF16 49 / 46, 95 / 61, 19 / 39,
// 168 / 87; TQ4 62 / 64, 129 / 75, 23 / 56, 193 / 103; Q8_0 46 / 58, 85 / 72, 19 / 48, 140 / 103.  128 columns: BF16 31 / 34, 57 / 47,
// 16 / 29, 93 / 61; TQ4 39 / 51, 69 / 64, 17 / 45, 106 / 85; Q8_0 29 / 46, 53 / 62, 16 / 40, 77 / 84.
constexpr int kChunkFrom = 256;

constexpr int kLeastRound = 16;  // slots for each kv head, whatever their number

static int decode_cols(int format) { return format == WARP34_KV_FORMAT_TQ4 ? kTq4Cols : kDecodeCols; }

// The tiles of a batch: the kernel, a tile's tokens, tiles of a request, slots for each kv head (0: no split).
struct ScoredShape {
    bool chunk;
    int cols, tok_tile;
    long long tiles, entries;
    int slots, round;
    bool full_rounds;
};
static ScoredShape scored_shape(int format, int head_dim, int kv_subs, int num_reqs, int total_tokens, int max_q_len, int q_group) {
    ScoredShape s;
    const int q_len = max_q_len > 0 ? std::min(max_q_len, total_tokens) : total_tokens;
    s.chunk = (long long)q_len * q_group >= kChunkFrom;
    s.cols = s.chunk ? kChunkCols : decode_cols(format);
    s.tok_tile = s.cols / q_group;
    s.tiles = ((long long)q_len + s.tok_tile - 1) / s.tok_tile;
    s.entries = s.tiles * num_reqs;
    // A round of workgroups: 256, or twice as many of the decode kernel at head_dim 128 (two to a CU).  us a call, 128 slots whatever the kv
    // heads / so.  One kv head: Q8_0 verify 31.0 / 23.7, 12 requests over TQ4 49.6 / 33.1; four: 8 000 TQ4 keys 22.9 / 14.6, 50 000 36.2 / 24.8,
    // verify 64 / 59; eight: 8 000 TQ4 keys 38 / 17, prefixes over FP8 1 083 / 982.
    s.round = std::max(kLeastRound, (!s.chunk && head_dim == 128 ? 512 : 256) / kv_subs);
    // Decode batches of few tiles: chunks for one round at most.  Others: up to two rounds, or a chunk for each tile and some more.
    s.full_rounds = s.chunk || s.entries > std::min(64, s.round / 2);
    s.slots = s.entries > kMaxSplitEntries ? 0 : (int)(s.full_rounds ? 2 * s.round + s.entries : s.round);
    return s;
}
// Bytes of the partial records of a slot, and of the tiles' table.
static size_t scored_slot_bytes(const ScoredShape& s, int kv_subs, int head_dim) { return (size_t)kv_subs * s.cols * (size_t)(head_dim + 2) * 4; }
static size_t scored_table_bytes(long long entries) { return ((size_t)entries * 8 + 15) / 16 * 16; }

// Largest divisor of the q heads of a kv head that fits a column tile
static int scored_q_group(int format, int gqa) {
    int d = std::min(gqa, decode_cols(format));
    while (gqa % d != 0) --d;
    return d;
}

static bool scored_format_ok(const warp34_kv_layer_layout* l, int storage_format) {
    if (l->k_format != l->v_format) return false;
    const auto xf_ok = [](int t) { return t == WARP34_KV_TRANSFORM_IDENTITY || t == WARP34_KV_TRANSFORM_RADEMACHER_WHT256; };
    if (!xf_ok(l->k_transform) || !xf_ok(l->v_transform)) return false;
    if (l->k_format == storage_format) {
        return (l->head_dim == 256 || l->head_dim == 128) && l->k_transform == WARP34_KV_TRANSFORM_IDENTITY &&
               l->v_transform == WARP34_KV_TRANSFORM_IDENTITY;
    }
    return l->head_dim == 256 &&
           (l->k_format == WARP34_KV_FORMAT_TQ4 || l->k_format == WARP34_KV_FORMAT_FP8_E4M3 || l->k_format == WARP34_KV_FORMAT_Q8_0);
}
static unsigned scored_row_bytes(const warp34_kv_layer_layout* l) {
    return l->k_format == WARP34_KV_FORMAT_TQ4        ? 132u
           : l->k_format == WARP34_KV_FORMAT_FP8_E4M3 ? 264u
           : l->k_format == WARP34_KV_FORMAT_Q8_0     ? 272u
                                                      : 2u * (unsigned)l->head_dim;
}
// rows of a page contiguous, runs of 16 rows 16-byte aligned, as the other attention calls want them
static bool scored_geometry_ok(const warp34_kv_layer_layout* l, const void* q, const void* out, const float* lse) {
    const uint64_t all = l->k_base | l->v_base | l->k_page_stride_bytes | l->k_head_stride_bytes | l->v_page_stride_bytes | l->v_head_stride_bytes;
    const unsigned row = scored_row_bytes(l);
    return l->block_size > 0 && (l->block_size % 16) == 0 && l->k_token_stride_bytes == row && l->v_token_stride_bytes == row && (all & 15u) == 0 &&
           (((uintptr_t)q) & 15u) == 0 && (((uintptr_t)out) & 7u) == 0 && (((uintptr_t)lse) & 3u) == 0;
}

template <typename TQ, int KVF, int HD>
static int launch_scored(const warp34_exec* ex, ScoredParams P) {
    const warp34_attention_batch& B = P.B;
    const int kv_subs = P.L.local_kv_heads * P.q_subgroups;
    const ScoredShape s = scored_shape(KVF, HD, kv_subs, B.num_reqs, B.total_tokens, B.max_q_len, P.q_group);
    if (kv_subs > 65535 || s.entries * kv_subs > 0x7FFFFFFF || !grid_fits(s.entries, kScoredWaves * 64)) return (int)hipErrorInvalidValue;
    P.tok_tile = s.tok_tile;
    P.tiles = (int)s.tiles;
    P.entries = (int)s.entries;
    P.min_halves = s.chunk ? kChunkMinHalves : kDecodeMinHalves;
    // records: as many as the scratch holds; no split where a tile has too few keys for two chunks
    long long slots = s.slots, records = 0;
    const size_t table = scored_table_bytes(s.entries);
    if (ex->scratch_ptr != 0 && (ex->scratch_ptr & 15u) == 0 && ex->scratch_size > table)
        records = std::min<long long>(slots, (long long)((ex->scratch_size - table) / scored_slot_bytes(s, kv_subs, HD)));
    if (records < 2 || (B.max_seq_len > 0 && B.max_seq_len <= 16 * (s.chunk ? kChunkMinHalves : kDecodeWhole))) slots = 0;
    if (slots > 0 && B.max_seq_len > 0) {
        const long long most = (((long long)B.max_seq_len + 30) / 16 + P.min_halves - 1) / P.min_halves;  // chunks of a tile
        slots = std::min(slots, std::max<long long>(s.entries * most, 2));
    }
    P.target = (int)slots;
    P.full_rounds = s.full_rounds ? 1 : 0;
    P.round = s.round;
    P.records = (int)records;
    if (slots > 0) {
        uint8_t* at = reinterpret_cast<uint8_t*>((uintptr_t)ex->scratch_ptr);
        P.table = reinterpret_cast<int32_t*>(at);
        P.part_acc = reinterpret_cast<float*>(at + table);
        P.part_ml = P.part_acc + (size_t)records * kv_subs * s.cols * HD;
    }
    hipStream_t stream = (hipStream_t)ex->stream;
    const dim3 grid((unsigned)(slots > 0 ? slots : s.entries), (unsigned)kv_subs);
    const auto launch = [&](auto kernel, int threads, int lds) {
        const int rc = ensure_dynamic_lds(kernel, lds, true);
        if (rc) return rc;
        hipLaunchKernelGGL(kernel, grid, dim3((unsigned)threads), (unsigned)lds, stream, P);
        return (int)hipGetLastError();
    };
    const bool cap = P.cap2 > 0.f;
    int rc;
    if (!s.chunk) {
        if constexpr (KVF == WARP34_KV_FORMAT_TQ4)
            rc = cap ? launch(scored_decode_tq4_kernel<TQ, true>, kScoredWaves * 64, Tq4Lds::kBytes)
                     : launch(scored_decode_tq4_kernel<TQ, false>, kScoredWaves * 64, Tq4Lds::kBytes);
        else
            rc = cap ? launch(scored_decode_kernel<TQ, KVF, HD, true>, kScoredWaves * 64, ScoredLds<KVF, HD>::kBytes)
                     : launch(scored_decode_kernel<TQ, KVF, HD, false>, kScoredWaves * 64, ScoredLds<KVF, HD>::kBytes);
    } else {
        constexpr int lds = ChunkLds<KVF, HD>::kBytes;
        rc = cap ? launch(scored_chunk_kernel<TQ, KVF, HD, true>, kChunkWaves * 64, lds)
                 : launch(scored_chunk_kernel<TQ, KVF, HD, false>, kChunkWaves * 64, lds);
    }
    if (rc || slots == 0) return rc;
    const float value_scale = KVF == WARP34_KV_FORMAT_TQ4 && !s.chunk ? kTableInvGain : ScoredRows<KVF, HD>::kOutScale;
    if (s.entries > (s.chunk ? kSpreadChunkTiles : kSpreadTiles)) {
        hipLaunchKernelGGL((scored_join_kernel<TQ, HD, false>), dim3((unsigned)s.entries, (unsigned)kv_subs, (unsigned)((s.cols + kJoinCols - 1) / kJoinCols)), dim3(512), 0, stream, P,
                           s.cols, value_scale);
    } else {
        hipLaunchKernelGGL((scored_join_kernel<TQ, HD, true>), dim3((unsigned)s.entries, (unsigned)kv_subs, (unsigned)s.cols), dim3(512), 0, stream, P,
                           s.cols, value_scale);
    }
    return (int)hipGetLastError();
}

template <typename TQ>
static int scored_entry(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch,
                        const warp34_attention_scores* scores, const void* q, void* out, int num_q_heads) {
    if (!ex || !layout || !batch || !scores || !q || !out) return (int)hipErrorInvalidValue;
    if (num_q_heads <= 0 || batch->total_tokens < 0) return (int)hipErrorInvalidValue;
    if (batch->total_tokens == 0) return 0;
    if (layout->local_kv_heads <= 0 || num_q_heads % layout->local_kv_heads != 0 || batch->num_reqs <= 0 || !batch->query_start_loc ||
        !batch->seq_lens_after || !batch->block_tables || batch->max_blocks_per_req <= 0 || batch->sliding_window < 0 ||
        (batch->mask_mode != WARP34_ATTN_MASK_CAUSAL && batch->mask_mode != WARP34_ATTN_MASK_NONCAUSAL_WINDOW) || !(scores->softcap >= 0.f) ||
        !(scores->softcap < INFINITY)) {
        return (int)hipErrorInvalidValue;
    }
    if (!scored_format_ok(layout, TQ::kStorageFormat) || !scored_geometry_ok(layout, q, out, scores->lse_out)) return (int)hipErrorNotSupported;
    ScoredParams P{};
    P.L = *layout;
    P.B = *batch;
    P.q = (const uint16_t*)q;
    P.out = (uint16_t*)out;
    P.slopes = scores->distance_slopes;
    P.document_starts = scores->document_starts;
    P.prefix_ends = scores->prefix_ends;
    P.lse = scores->lse_out;
    P.scale2 = std::fabs(batch->sm_scale) * kLog2e;
    P.q_flip = batch->sm_scale < 0.f ? 0x80008000u : 0u;
    const float cap = std::min(scores->softcap, kLargestCap);
    P.cap2 = cap * kLog2e;
    // (finite under the smallest of caps; cap_factor)
    P.cap_arg = cap > 0.f ? std::min(2.0f * std::fabs(batch->sm_scale) * kLog2e / cap, 1.0e30f) : 0.f;
    P.wide_cap = cap > kWideCap ? 1 : 0;
    P.num_q_heads = num_q_heads;
    P.gqa = num_q_heads / layout->local_kv_heads;
    P.q_group = scored_q_group(layout->k_format, P.gqa);
    P.q_subgroups = P.gqa / P.q_group;
    P.block_magic = block_magic_for(layout->block_size);
    P.q_group_magic = q_group_magic_for(P.q_group);
    P.rot_q = layout->k_transform == WARP34_KV_TRANSFORM_RADEMACHER_WHT256 ? 1 : 0;
    P.rot_out = layout->v_transform == WARP34_KV_TRANSFORM_RADEMACHER_WHT256 ? 1 : 0;
    if (layout->k_format == WARP34_KV_FORMAT_TQ4) return launch_scored<TQ, WARP34_KV_FORMAT_TQ4, 256>(ex, P);
    if (layout->k_format == WARP34_KV_FORMAT_FP8_E4M3) return launch_scored<TQ, WARP34_KV_FORMAT_FP8_E4M3, 256>(ex, P);
    if (layout->k_format == WARP34_KV_FORMAT_Q8_0) return launch_scored<TQ, WARP34_KV_FORMAT_Q8_0, 256>(ex, P);
    if (layout->head_dim == 128) return launch_scored<TQ, TQ::kStorageFormat, 128>(ex, P);
    return launch_scored<TQ, TQ::kStorageFormat, 256>(ex, P);
}

}  // namespace w34

using namespace w34;

extern "C" int warp34_paged_attention_scored_f16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch,
                                                 const warp34_attention_scores* scores, const void* q_in, void* attn_out, int num_q_heads) {
    return scored_entry<F16>(ex, layout, batch, scores, q_in, attn_out, num_q_heads);
}
extern "C" int warp34_paged_attention_scored_bf16(const warp34_exec* ex, const warp34_kv_layer_layout* layout, const warp34_attention_batch* batch,
                                                  const warp34_attention_scores* scores, const void* q_in, void* attn_out, int num_q_heads) {
    return scored_entry<BF16>(ex, layout, batch, scores, q_in, attn_out, num_q_heads);
}

extern "C" size_t warp34_paged_attention_scored_scratch_bytes(const warp34_kv_layer_layout* layout, int num_reqs, int total_tokens, int max_q_len,
                                                              int num_q_heads) {
    if (!layout || layout->local_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % layout->local_kv_heads != 0 || num_reqs <= 0 || total_tokens <= 0)
        return 0;
    const int gqa = num_q_heads / layout->local_kv_heads, group = scored_q_group(layout->k_format, gqa);
    const int kv_subs = layout->local_kv_heads * (gqa / group);
    const ScoredShape s = scored_shape(layout->k_format, layout->head_dim, kv_subs, num_reqs, total_tokens, max_q_len, group);
    return s.slots == 0 ? 0 : scored_table_bytes(s.entries) + (size_t)s.slots * scored_slot_bytes(s, kv_subs, layout->head_dim);
}
