"""Scored attention over pages in which every row that no live token sees holds bytes of 0xFF (NaN elements, codes and scales): rows of masked
tokens, which the append leaves unwritten, and rows between the keys of two tokens."""
import numpy as np
import pytest

import oracle
from cases import make_case
from oracle import DT_BF16, DT_F16, FMT_BF16, FMT_FP16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_IDENTITY, XF_WHT256
from plain_kv import scored_attention
from scored_harness import CHUNK_FROM, SENTINEL, run_scored

FORMS = [(FMT_TQ4, XF_WHT256, DT_BF16, 256), (FMT_FP8, XF_IDENTITY, DT_F16, 256), (FMT_FP8, XF_WHT256, DT_BF16, 256),
         (FMT_Q8_0, XF_IDENTITY, DT_F16, 256), (FMT_FP16, XF_IDENTITY, DT_F16, 256), (FMT_BF16, XF_IDENTITY, DT_BF16, 256),
         (FMT_BF16, XF_IDENTITY, DT_BF16, 128)]
NOWHERE = 1 << 20  # a document that starts behind everything


def check(fmt, xf, dt, hd, seq, tokens, live, *, ctx=None, kv_heads=2, heads=8, scratch=8 << 20, window=0, documents=None, prefixes=None, block=16):
    """live: which of the request's tokens count."""
    pool, bt, k, v, q, aq, before = make_case(fmt, block, [seq], [tokens], 1400, dt, xf=xf, head_dim=hd, kv_heads=kv_heads, q_heads=heads)
    before = before if ctx is None else [ctx]
    seen = np.zeros(bt.shape[1] * block, dtype=bool)
    for t in np.nonzero(live)[0]:
        pos = before[0] + t
        hi = min(max(pos, -1 if prefixes is None else prefixes[t] - 1), seq - 1)
        lo = max(0, pos - window + 1 if window else 0, 0 if documents is None else documents[t])
        seen[lo:max(lo, hi + 1)] = True
    rows = np.ones(pool.k.size // pool.page * block, dtype=bool)
    rows[oracle.slot_mapping(bt[0], 0, seen.size, block)[seen]] = False
    views = [s.reshape(-1, kv_heads, block, pool.tok) for s in (pool.k, pool.v)]
    for s in views:
        for h in range(kv_heads):
            s[:, h][rows.reshape(-1, block)] = 0xFF
    hb = oracle.HostBatch(aq, [seq], bt, context_lens_before=before, valid_token_mask=np.asarray(live, dtype=np.uint8))
    hb.sliding_window = window
    terms = dict(cap=30.0, documents=documents, prefixes=prefixes)
    bits, lse = run_scored(pool, hb, q, dt, heads, scratch=scratch, **terms)
    for s in views:
        for h in range(kv_heads):
            s[:, h][rows.reshape(-1, block)] = 0
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [seq], oracle.bits_to_f32(q, dt).astype(np.float64), aq, before, window=window,
                                                        scale=hb.sm_scale, dt=dt, chunk=tokens * (heads // kv_heads) >= CHUNK_FROM, **terms)
    live = np.asarray(live, dtype=bool)
    assert (bits[~live] == SENTINEL).all() and (lse[~live] == 77.0).all()
    got = oracle.bits_to_f32(bits, dt).astype(np.float64)[live]
    assert np.isfinite(got).all() and (np.abs(got - want[live]) <= bound[live]).all()
    empty = np.isneginf(want_lse[live])
    assert np.isneginf(lse[live][empty]).all() and (got[empty] == 0).all()
    assert (np.abs(lse[live][~empty] - want_lse[live][~empty]) <= lse_bound[live][~empty]).all()


def all_but(tokens, a, b):
    live = np.ones(tokens, dtype=bool)
    live[a:b] = False
    return live


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf,dt,hd", FORMS)
@pytest.mark.parametrize("tokens,seq", [(6, 309), (100, 409)])
def test_masked_tokens_at_the_end_and_at_the_start(fmt, xf, dt, hd, tokens, seq):
    """Padding behind a request's tokens, and masked first tokens before whose keys nobody else's window reaches."""
    n = tokens // 2
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, n, tokens))
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, 0, n), window=4)


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", [0, 8 << 20])
@pytest.mark.parametrize("fmt,xf,dt,hd", FORMS)
@pytest.mark.parametrize("tokens,seq", [(20, 309), (100, 409)])
def test_rows_between_the_keys_of_two_tokens(fmt, xf, dt, hd, tokens, seq, scratch):
    a, b = tokens // 4, 3 * tokens // 4
    # masked tokens in the middle of a window's slide
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, a, b), window=3, scratch=scratch)
    # tokens whose document starts nowhere, in the same place
    documents = np.zeros(tokens, dtype=np.int32)
    documents[a:b] = NOWHERE
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, 0, 0), window=2, documents=documents, scratch=scratch)
    # a packed document that is masked as a whole
    documents = seq - tokens + np.where(np.arange(tokens) < a, 0, np.where(np.arange(tokens) < b, a, b)).astype(np.int32)
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, a, b), documents=documents, scratch=scratch)
    # tokens that see a part of a prefix far behind them only
    documents, prefixes = np.zeros(tokens, dtype=np.int32), np.zeros(tokens, dtype=np.int32)
    documents[::3], prefixes[::3] = seq - 50, seq - 20
    check(fmt, xf, dt, hd, seq, tokens, all_but(tokens, 0, 0), ctx=100, documents=documents, prefixes=prefixes, scratch=scratch)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf,dt,hd", [FORMS[0], FORMS[2], FORMS[5], FORMS[6]])
def test_gaps_in_tiles_of_many_tokens(fmt, xf, dt, hd):
    """One query head for each kv head: 256 tokens in a tile, gaps of many sizes."""
    live = np.random.default_rng(8).random(300) < 0.05
    check(fmt, xf, dt, hd, 700, 300, live, window=7, heads=2)
    check(fmt, xf, dt, hd, 700, 300, live, window=2, heads=2, block=48)
