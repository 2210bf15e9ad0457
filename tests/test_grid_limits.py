"""Calls whose launch would have 2^32 threads or more, which no grid has: refused before anything is launched."""
import ctypes as C

import pytest

from oracle import FMT_BF16, FMT_TQ4, XF_IDENTITY, XF_WHT256

MANY = 1 << 24  # workgroups of 256 threads


@pytest.mark.parametrize("head_dim,rows", [(256, 8 * MANY), (8, 256 * MANY), (2048, MANY), (2048, (1 << 31) - 1)])
@pytest.mark.parametrize("name", ["warp34_attention_merge_f16", "warp34_attention_merge_bf16"])
def test_merges_of_too_many_rows(name, head_dim, rows):
    from warp34_amd import ffi

    ex = ffi.Warp34Exec(0, 0, 0, 0)
    assert getattr(ffi.load(), name)(C.byref(ex), 1 << 20, 1 << 21, 2, rows * head_dim, rows, 1 << 22, None, rows, head_dim) == 1


@pytest.mark.parametrize("fmt,xf,head_dim,rows", [(FMT_BF16, XF_IDENTITY, 256, 8 * MANY), (FMT_BF16, XF_IDENTITY, 128, 16 * MANY),
                                                  (FMT_TQ4, XF_WHT256, 256, 16 * MANY), (FMT_TQ4, XF_IDENTITY, 256, 8 * MANY),
                                                  (FMT_TQ4, XF_WHT256, 256, (1 << 31) - 1)])
@pytest.mark.parametrize("want_k,want_v", [(True, True), (True, False), (False, True)])
def test_reads_of_too_many_rows(fmt, xf, head_dim, rows, want_k, want_v):
    from warp34_amd import ffi

    tok = 2 * head_dim if fmt == FMT_BF16 else 132
    layout = ffi.Warp34KvLayerLayout(1 << 20, 1 << 30, 16 * tok, 16 * tok, tok, 16 * tok, 16 * tok, tok, 0, 0, 1, head_dim, 16, fmt, fmt, xf, xf, 0)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    assert ffi.load().warp34_kv_cache_read_bf16(C.byref(ex), C.byref(layout), 1 << 24, rows, 1 << 25 if want_k else None,
                                                1 << 26 if want_v else None, head_dim, head_dim) == 1


@pytest.mark.parametrize("reqs,tokens,max_q_len", [(1 << 23, 1 << 23, 1), (1 << 14, 1 << 19, 0), (1 << 18, 1 << 18, 2048)])
def test_scored_batches_of_too_many_tiles(reqs, tokens, max_q_len):
    """Tiles are counted by the bounds: requests times the tiles of max_q_len (of all tokens where it is not known)."""
    from warp34_amd import ffi

    strides = (512 * 16, 512 * 16, 512)
    layout = ffi.Warp34KvLayerLayout(1 << 20, 1 << 30, *strides, *strides, 0, 0, 1, 256, 16, FMT_BF16, FMT_BF16, XF_IDENTITY, XF_IDENTITY, 0)
    batch = ffi.Warp34AttentionBatch(1 << 16, None, 1 << 17, 1 << 18, None, None, None, reqs, tokens, 4, max_q_len, 64, 0, 0, 0.0625, 0)
    scores = ffi.Warp34AttentionScores(None, None, None, None, 0.0, 0)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    assert ffi.load().warp34_paged_attention_scored_bf16(C.byref(ex), C.byref(layout), C.byref(batch), C.byref(scores), 1 << 24, 1 << 25, 8) == 1
