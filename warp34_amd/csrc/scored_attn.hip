// Scored paged attention: checks, dispatch and entry points.
#include <algorithm>

#include "attn_launch.h"
#include "scored_decode.h"

namespace w34 {

constexpr int kScoredSlots = 128;       // chunks for each kv head of a batch of up to 64 tiles: with two kv heads one for every CU
constexpr int kScoredSplitTiles = 512;  // from here on a kv head's tiles fill the chip by themselves

// Bytes of the partial records of `slots` chunks and of the tiles' table.
static size_t scored_slot_bytes(int kv_subs, int head_dim) { return (size_t)kv_subs * 16 * (size_t)(head_dim + 2) * 4; }
static size_t scored_table_bytes(long long entries) { return ((size_t)entries * 8 + 15) / 16 * 16; }
static int scored_slots(long long entries) {
    if (entries >= kScoredSplitTiles) return 0;
    return kScoredSlots * (int)((std::max<long long>(2 * entries, kScoredSlots) + kScoredSlots - 1) / kScoredSlots);
}
static_assert(kScoredSplitTiles <= kMaxSplitEntries, "tile counts in LDS");

// Largest divisor of the q heads of a kv head that fits a column tile
static int scored_q_group(int gqa) {
    int d = std::min(gqa, 16);
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
    if (kv_subs > 65535) return (int)hipErrorInvalidValue;
    P.tok_tile = std::max(1, 16 / P.q_group);
    const long long tiles = ((long long)(B.max_q_len > 0 ? std::min(B.max_q_len, B.total_tokens) : B.total_tokens) + P.tok_tile - 1) / P.tok_tile;
    const long long entries = tiles * B.num_reqs;
    if (entries > 0x7FFFFFFF) return (int)hipErrorInvalidValue;
    P.tiles = (int)tiles;
    P.entries = (int)entries;
    // chunks: as many as the scratch holds, none where a tile has too few keys for two
    long long slots = scored_slots(entries);
    const size_t table = scored_table_bytes(entries), per_slot = scored_slot_bytes(kv_subs, HD);
    if (ex->scratch_ptr == 0 || (ex->scratch_ptr & 15u) != 0 || ex->scratch_size <= table) slots = 0;
    else slots = std::min<long long>(slots, (long long)((ex->scratch_size - table) / per_slot));
    if (B.max_seq_len > 0) {
        const long long most = (((long long)B.max_seq_len + 30) / 16 + kMinHalvesPerChunk - 1) / kMinHalvesPerChunk;  // chunks of a tile
        slots = B.max_seq_len <= 16 * kMinHalvesPerChunk ? 0 : std::min(slots, entries * (most + 1));
    }
    if (slots < entries + std::max<long long>(2, entries / 2)) slots = 0;
    P.target = (int)slots;
    if (slots > 0) {
        uint8_t* at = reinterpret_cast<uint8_t*>((uintptr_t)ex->scratch_ptr);
        P.table = reinterpret_cast<int32_t*>(at);
        P.part_acc = reinterpret_cast<float*>(at + table);
        P.part_ml = P.part_acc + (size_t)slots * kv_subs * 16 * HD;
    }
    hipStream_t stream = (hipStream_t)ex->stream;
    using M = ScoredLds<KVF, HD>;
    const dim3 grid((unsigned)(slots > 0 ? slots : entries), (unsigned)kv_subs);
    const auto launch = [&](auto kernel) {
        const int rc = ensure_dynamic_lds(kernel, M::kBytes, true);
        if (rc) return rc;
        hipLaunchKernelGGL(kernel, grid, dim3(kScoredWaves * 64), M::kBytes, stream, P);
        return (int)hipGetLastError();
    };
    const int rc = P.cap2 > 0.f ? launch(scored_decode_kernel<TQ, KVF, HD, true>) : launch(scored_decode_kernel<TQ, KVF, HD, false>);
    if (rc || slots == 0) return rc;
    hipLaunchKernelGGL((scored_join_kernel<TQ, HD>), dim3((unsigned)entries, (unsigned)kv_subs, 16u), dim3(512), 0, stream, P, 16,
                       ScoredRows<KVF, HD>::kOutScale);
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
    P.scale2 = batch->sm_scale * kLog2e;
    P.cap2 = scores->softcap * kLog2e;
    P.cap_arg = scores->softcap > 0.f ? 2.0f * batch->sm_scale * kLog2e / scores->softcap : 0.f;
    P.wide_cap = scores->softcap > kWideCap ? 1 : 0;
    P.num_q_heads = num_q_heads;
    P.gqa = num_q_heads / layout->local_kv_heads;
    P.q_group = scored_q_group(P.gqa);
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
    const int gqa = num_q_heads / layout->local_kv_heads, group = scored_q_group(gqa), tok_tile = std::max(1, 16 / group);
    const long long tiles = ((long long)(max_q_len > 0 ? std::min(max_q_len, total_tokens) : total_tokens) + tok_tile - 1) / tok_tile;
    const long long entries = tiles * num_reqs;
    const int slots = scored_slots(entries);
    return slots == 0 ? 0 : scored_table_bytes(entries) + (size_t)slots * scored_slot_bytes(layout->local_kv_heads * (gqa / group), layout->head_dim);
}
