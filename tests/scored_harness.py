"""Calls of warp34_paged_attention_scored_* for the tests."""
import ctypes as C

import numpy as np

import oracle
from oracle import DT_BF16
from plain_kv import scored_attention

SENTINEL = 0x5500
CHUNK_FROM = 256  # query columns of a request from which the call takes its chunk kernel


def scores_struct(G, cap=0.0, slopes=None, documents=None, prefixes=None, lse=None):
    from warp34_amd import ffi

    keep = [None if a is None else G.to_dev(np.asarray(a, dtype=t))
            for a, t in ((slopes, np.float32), (documents, np.int32), (prefixes, np.int32))]
    at = [None if k is None else k.data_ptr() for k in keep]
    return ffi.Warp34AttentionScores(at[0], at[1], at[2], None if lse is None else lse.data_ptr(), cap, 0), keep


def run_scored(pool, hb, q, dt, heads, *, scratch=8 << 20, with_lse=True, max_q_len=None, max_seq_len=None, dpool=None, layout=None, **terms):
    """(out bits, lse) of one call; rows of the outputs start as SENTINEL / 77."""
    import torch

    import gpu_harness as G

    if dpool is None:
        dpool = G.DevPool(pool)
        dpool.upload()
    layout = dpool.layout() if layout is None else layout
    db = G.DevBatch(hb, max_q_len=max_q_len, max_seq_len=max_seq_len)
    batch = db.struct()
    ex, ws = G.make_exec(scratch)
    qd = G.to_dev(q)
    out = torch.full((hb.total_tokens + 1, heads, pool.head_dim), SENTINEL, dtype=torch.int16, device=G.DEV)
    lse = torch.full((hb.total_tokens + 1, heads), 77.0, dtype=torch.float32, device=G.DEV)
    scores, keep = scores_struct(G, lse=lse if with_lse else None, **terms)
    fn = G.lib().warp34_paged_attention_scored_bf16 if dt == DT_BF16 else G.lib().warp34_paged_attention_scored_f16
    rc = fn(C.byref(ex), C.byref(layout), C.byref(batch), C.byref(scores), G.ptr(qd), G.ptr(out), heads)
    torch.cuda.synchronize()
    assert rc == 0, rc
    if ws is not None:
        assert bool((ws[scratch:] == 0x5A).all()), "scratch canary overwritten"
    assert bool((out[hb.total_tokens] == SENTINEL).all()) and bool((lse[hb.total_tokens] == 77.0).all())
    assert with_lse or bool((lse == 77.0).all())
    return out[:-1].cpu().numpy().view(np.uint16), lse[:-1].cpu().numpy()


def check_scored(pool, bt, seqs, q, dt, aq, ctx, heads, *, hb=None, scratch=8 << 20, rows=None, with_lse=True, max_q_len=None,
                 max_seq_len=None, **terms):
    """One call against the plain form; rows: the tokens that are computed (all)."""
    kinds = {"window": 0, "noncausal": False}
    kinds.update({k: terms.pop(k) for k in list(terms) if k in kinds})
    if hb is None:
        hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx)
    hb.sliding_window, hb.mask_mode = kinds["window"], 1 if kinds["noncausal"] else 0
    bits, lse = run_scored(pool, hb, q, dt, heads, scratch=scratch, with_lse=with_lse, max_q_len=max_q_len, max_seq_len=max_seq_len, **terms)
    longest = int(np.diff(hb.qsl).max()) if max_q_len is None else max_q_len
    columns = 8 if pool.fmt == oracle.FMT_TQ4 else 16  # of a decode tile, of which a kv head's query heads fill a divisor
    group = next(d for d in range(min(columns, heads // pool.kv_heads), 0, -1) if heads // pool.kv_heads % d == 0)
    chunk = (longest if longest > 0 else hb.total_tokens) * group >= CHUNK_FROM
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, seqs, oracle.bits_to_f32(q, dt).astype(np.float64), aq, ctx,
                                                        scale=hb.sm_scale, dt=dt, chunk=chunk, **kinds, **terms)
    rows = np.ones(hb.total_tokens, dtype=bool) if rows is None else np.asarray(rows, dtype=bool)
    got = oracle.bits_to_f32(bits, dt).astype(np.float64)
    assert (bits[~rows] == SENTINEL).all()
    over = (np.abs(got - want) - bound)[rows]
    assert np.isfinite(got[rows]).all() and over.max() <= 0, ("out", over.max(), np.unravel_index(over.argmax(), over.shape))
    if with_lse:
        assert (lse[~rows] == 77.0).all()
        empty = np.isneginf(want_lse) & rows[:, None]
        assert np.isneginf(lse[empty]).all() and (got[empty] == 0).all()
        full = rows[:, None] & ~empty
        over = np.abs(lse[full] - want_lse[full]) - lse_bound[full]
        assert np.isfinite(lse[full]).all() and (over.size == 0 or over.max() <= 0), ("lse", over.max())
    return bits, lse
