"""warp34_paged_attention_scored_*: score caps, distance slopes, windows, documents and prefixes over every page format, against the
plain form in float64 (tests/plain_kv.py, which derives the tolerances)."""
import ctypes as C

import numpy as np
import pytest

import oracle
from cases import make_case
from oracle import DT_BF16, DT_F16, FMT_BF16, FMT_FP16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_IDENTITY, XF_WHT256
from plain_kv import scored_attention
from scored_harness import CHUNK_FROM, SENTINEL, check_scored, run_scored, scores_struct

gpu = pytest.mark.gpu
FORMS = [(FMT_TQ4, XF_WHT256, XF_WHT256, DT_F16, 256), (FMT_TQ4, XF_WHT256, XF_WHT256, DT_BF16, 256),
         (FMT_TQ4, XF_IDENTITY, XF_WHT256, DT_F16, 256), (FMT_TQ4, XF_WHT256, XF_IDENTITY, DT_BF16, 256),
         (FMT_FP8, XF_IDENTITY, XF_IDENTITY, DT_F16, 256), (FMT_FP8, XF_WHT256, XF_WHT256, DT_BF16, 256),
         (FMT_Q8_0, XF_IDENTITY, XF_IDENTITY, DT_BF16, 256), (FMT_Q8_0, XF_WHT256, XF_WHT256, DT_F16, 256),
         (FMT_FP16, XF_IDENTITY, XF_IDENTITY, DT_F16, 256), (FMT_FP16, XF_IDENTITY, XF_IDENTITY, DT_F16, 128),
         (FMT_BF16, XF_IDENTITY, XF_IDENTITY, DT_BF16, 256), (FMT_BF16, XF_IDENTITY, XF_IDENTITY, DT_BF16, 128)]


def slopes_of(heads):
    return (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)


def case(fmt, block, seqs, qs, seed, dt, **kw):
    return make_case(fmt, block, seqs, qs, seed, dt, **kw)


@gpu
@pytest.mark.parametrize("fmt,xf,v_xf,dt,hd", FORMS)
@pytest.mark.parametrize("seqs,qs,terms", [([1, 17, 300], [1, 1, 1], {"cap": 30.0}), ([40, 700], [3, 5], {"sloped": True}),
                                           ([150, 90], [90, 33], {"cap": 5.0, "window": 50})])
def test_formats(fmt, xf, v_xf, dt, hd, seqs, qs, terms):
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 900 + hd, dt, xf=xf, v_xf=v_xf, head_dim=hd)
    terms = dict(terms)
    if terms.pop("sloped", False):
        terms["slopes"] = slopes_of(8)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, **terms)


@gpu
@pytest.mark.parametrize("scratch", [0, 8 << 20])
@pytest.mark.parametrize("seq", [1, 2, 15, 16, 17, 127, 128, 129, 145, 700, 5003])
def test_lengths(seq, scratch):
    pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 64, [seq], [1], 910, DT_F16)
    check_scored(pool, bt, [seq], q, DT_F16, aq, ctx, 8, scratch=scratch, cap=50.0, slopes=slopes_of(8))


@gpu
@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (4, 4), (2, 16), (1, 24), (1, 17), (2, 32), (3, 9), (1, 64)])
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_FP16, DT_F16)])
def test_head_layouts(fmt, dt, kv_heads, heads):
    seqs, qs = [260, 33], [3, 2]
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 920 + heads, dt, kv_heads=kv_heads, q_heads=heads)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, heads, cap=20.0, slopes=slopes_of(heads))


@gpu
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_F16), (FMT_BF16, DT_BF16), (FMT_Q8_0, DT_F16)])
@pytest.mark.parametrize("scratch", [0, 8 << 20])
def test_documents_prefixes_windows_and_empty_rows(fmt, dt, scratch):
    seqs, qs = [400, 61, 500], [70, 61, 4]
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 930, dt)
    rng = np.random.default_rng(5)
    pos = np.concatenate([np.arange(n) + c for n, c in zip(qs, ctx)])
    doc = (pos // 37 * 37).astype(np.int32)
    doc[::9] = 100000                    # sees nothing
    doc[5] = -4
    pre = rng.integers(-3, 600, pos.size).astype(np.int32)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, documents=doc)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, prefixes=pre)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, documents=doc, prefixes=pre, cap=30.0, slopes=slopes_of(8))
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, window=20, prefixes=pre)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, noncausal=True, window=100, slopes=slopes_of(8))


@gpu
def test_decode_step_with_documents():
    """One token each, its document's start deep in the context: the rest of the keys is not read."""
    seqs = [3000, 129, 700]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 64, seqs, [1, 1, 1], 931, DT_BF16)
    check_scored(pool, bt, seqs, q, DT_BF16, aq, ctx, 8, documents=np.array([2900, 129, 0], dtype=np.int32), cap=30.0)


@gpu
@pytest.mark.parametrize("block", [16, 48, 128])
def test_page_sizes(block):
    seqs, qs = [1000, 47, 48, 49], [1, 2, 1, 30]
    pool, bt, k, v, q, aq, ctx = case(FMT_FP8, block, seqs, qs, 940 + block, DT_BF16)
    check_scored(pool, bt, seqs, q, DT_BF16, aq, ctx, 8, cap=30.0)


@gpu
@pytest.mark.parametrize("scratch", [0, 1 << 16, 1 << 20, 3 << 20, 16 << 20])
def test_scratch_sizes(scratch):
    seqs = [3000, 700, 40, 1]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 64, seqs, [1] * 4, 950, DT_BF16)
    check_scored(pool, bt, seqs, q, DT_BF16, aq, ctx, 8, scratch=scratch, cap=30.0)


@gpu
@pytest.mark.parametrize("n", [33, 64, 65, 200])
def test_many_requests(n):
    """More requests than a wave has lanes, of ragged lengths, some without tokens."""
    rng = np.random.default_rng(n)
    seqs = [int(x) for x in rng.integers(1, 900, n)]
    qs = [0 if i % 7 == 3 else 1 for i in range(n)]
    pool, bt, k, v, q, aq, ctx = case(FMT_BF16, 16, seqs, qs, 960, DT_BF16, kv_heads=1, q_heads=4, head_dim=128)
    check_scored(pool, bt, seqs, q, DT_BF16, aq, ctx, 4, scratch=64 << 20, slopes=slopes_of(4))


@gpu
def test_bounds_unknown():
    """max_q_len and max_seq_len of 0: not known."""
    seqs, qs = [600, 40], [2, 5]
    pool, bt, k, v, q, aq, ctx = case(FMT_Q8_0, 16, seqs, qs, 965, DT_BF16)
    check_scored(pool, bt, seqs, q, DT_BF16, aq, ctx, 8, cap=30.0, max_q_len=0, max_seq_len=0)


@gpu
@pytest.mark.parametrize("qs", [[1, 1, 1], [20, 3, 40]])
def test_masked_tokens_and_requests_stay_untouched(qs):
    seqs = [300, 500, 90]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, seqs, qs, 970, DT_F16)
    n = aq[-1]
    tmask = np.ones(n, dtype=np.uint8)
    tmask[::5] = 0
    rmask = np.array([1, 0, 1], dtype=np.uint8)
    hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx, valid_token_mask=tmask, valid_req_mask=rmask)
    rows = tmask.astype(bool)
    rows[aq[1]:aq[2]] = False
    check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, hb=hb, rows=rows, cap=30.0)


@gpu
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_FP8, DT_F16), (FMT_Q8_0, DT_F16), (FMT_FP16, DT_F16), (FMT_BF16, DT_BF16)])
@pytest.mark.parametrize("qs", [[1], [37]])
def test_what_unseen_rows_hold_does_not_matter(fmt, dt, qs):
    """Bytes of 0xFF (NaN scales, values and codes) behind the sequence and before the window."""
    seq = 213
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, [seq], qs, 980, dt)
    seen_from = seq - qs[0] - 40 + 1
    wild = np.ones(pool.k.size // pool.page * 16, dtype=bool)
    wild[oracle.slot_mapping(bt[0], seen_from, seq - seen_from, 16)] = False
    rows_k, rows_v = (s.reshape(-1, pool.kv_heads, 16, pool.tok) for s in (pool.k, pool.v))
    w = wild.reshape(-1, 16)
    for s in (rows_k, rows_v):
        for h in range(pool.kv_heads):
            s[:, h][w] = 0xFF
    hb = oracle.HostBatch(aq, [seq], bt, context_lens_before=ctx)
    hb.sliding_window = 40
    bits, lse = run_scored(pool, hb, q, dt, 8, cap=30.0)
    for s in (rows_k, rows_v):
        for h in range(pool.kv_heads):
            s[:, h][w] = 0
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [seq], oracle.bits_to_f32(q, dt).astype(np.float64), aq, ctx, cap=30.0,
                                                        window=40, scale=hb.sm_scale, dt=dt, chunk=qs[0] * 4 >= CHUNK_FROM)
    got = oracle.bits_to_f32(bits, dt).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()


@gpu
@pytest.mark.parametrize("cap", [1e-44, 1e-38, 0.5, 512.0, 513.0, 1e4, 1e30])
def test_caps_of_any_size(cap):
    """Far above the scores a cap changes nothing.  (The bound's term for the cap stands for the 2^-23 that tanh is off by up to the
    size from which small arguments go through a series.)"""
    pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 16, [200], [2], 985, DT_F16)
    hb = oracle.HostBatch(aq, [200], bt, context_lens_before=ctx)
    bits, lse = run_scored(pool, hb, q, DT_F16, 8, cap=cap)
    q64 = oracle.bits_to_f32(q, DT_F16).astype(np.float64)
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [200], q64, aq, ctx, cap=min(cap, 1e12), scale=hb.sm_scale, dt=DT_F16)
    if cap > 512.0:
        _, _, bound, lse_bound = scored_attention(pool, bt, [200], q64, aq, ctx, cap=0.0, scale=hb.sm_scale, dt=DT_F16)
    got = oracle.bits_to_f32(bits, DT_F16).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()


@gpu
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_FP16, DT_F16)])
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("scale", [-0.0625, 0.0, 0.5])
def test_scales_of_any_sign(fmt, dt, tokens, scale):
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, [150], [tokens], 984, dt)
    hb = oracle.HostBatch(aq, [150], bt, context_lens_before=ctx)
    hb.sm_scale = scale
    check_scored(pool, bt, [150], q, dt, aq, ctx, 8, hb=hb, cap=20.0)


@gpu
@pytest.mark.parametrize("tokens", [2, 70])
def test_lengths_before_may_be_left_out(tokens):
    """Without context_lens_before a request's tokens are its last ones."""
    seqs, qs = [150, 90], [tokens, 3]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, seqs, qs, 983, DT_F16)
    hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx)
    want = run_scored(pool, hb, q, DT_F16, 8, cap=20.0)
    hb.ctx = None
    got = run_scored(pool, hb, q, DT_F16, 8, cap=20.0)
    assert want[0].tobytes() == got[0].tobytes() and want[1].tobytes() == got[1].tobytes()


@gpu
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_BF16, DT_BF16), (FMT_Q8_0, DT_F16)])
@pytest.mark.parametrize("tokens", [1, 70])
def test_positions_of_any_size(fmt, dt, tokens):
    """A window over the end of 2^30 keys gives the bits of the same keys in a short sequence."""
    block, seq, window = 128, 1000, 300
    pool, bt, k, v, q, aq, ctx = case(fmt, block, [seq], [tokens], 982, dt)
    moved = (1 << 23) - 16
    far = np.zeros((1, bt.shape[1] + moved), dtype=np.int32)
    far[0, moved:] = bt[0]
    results = []
    for table, before in ((bt, 0), (far, moved * block)):
        hb = oracle.HostBatch(aq, [seq + before], table, context_lens_before=[ctx[0] + before])
        hb.sliding_window = window
        documents = np.full(aq[-1], before + 640, dtype=np.int32)
        results.append(run_scored(pool, hb, q, dt, 8, cap=20.0, slopes=slopes_of(8), documents=documents))
    assert results[0][0].tobytes() == results[1][0].tobytes() and results[0][1].tobytes() == results[1][1].tobytes()


@gpu
def test_calls_on_two_streams_at_once():
    """Own workspaces, the same pages: a decode call and a chunk call in turn on each of two streams give what they give alone."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    made = []
    for seqs, qs, seed in (([3000, 100], [1, 2], 980), ([700], [130], 981)):
        pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, seqs, qs, seed, DT_BF16)
        dpool = G.DevPool(pool)
        dpool.upload()
        hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx)
        alone = run_scored(pool, hb, q, DT_BF16, 8, cap=30.0, dpool=dpool, scratch=16 << 20)
        made.append((dpool, G.DevBatch(hb), G.to_dev(q), aq[-1], alone))
    fn = G.lib().warp34_paged_attention_scored_bf16
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.zeros(16 << 20, dtype=torch.uint8, device=G.DEV) for _ in range(2)]
    calls = []
    torch.cuda.synchronize()
    for turn in range(6):
        for stream, space in zip(streams, spaces):
            dpool, db, qd, n, alone = made[(turn + (stream is streams[1])) % 2]
            with torch.cuda.stream(stream):
                out = torch.zeros((n, 8, 256), dtype=torch.int16, device=G.DEV)
                lse = torch.zeros((n, 8), dtype=torch.float32, device=G.DEV)
            layout, batch = dpool.layout(), db.struct()
            scores, keep = scores_struct(G, cap=30.0, lse=lse)
            ex = ffi.Warp34Exec(stream.cuda_stream, space.data_ptr(), space.numel(), 0)
            assert fn(C.byref(ex), C.byref(layout), C.byref(batch), C.byref(scores), G.ptr(qd), G.ptr(out), 8) == 0
            calls.append((out, lse, alone))
    torch.cuda.synchronize()
    for out, lse, alone in calls:
        assert out.cpu().numpy().view(np.uint16).tobytes() == alone[0].tobytes() and lse.cpu().numpy().tobytes() == alone[1].tobytes()


@gpu
def test_queries_of_any_size():
    """bf16 queries beyond fp16's range, and tiny ones, over quantised pages."""
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, [90, 90, 90], [1, 1, 1], 986, DT_BF16)
    x = oracle.bits_to_f32(q, DT_BF16) * np.array([1e20, 1e-20, 1.0], dtype=np.float32)[:, None, None]
    q = oracle.f32_to_bf16_bits(x)
    check_scored(pool, bt, [90] * 3, q, DT_BF16, aq, ctx, 8, cap=10.0)


@gpu
@pytest.mark.parametrize("slope", [-0.5, 0.0, 1000.0])
def test_slopes_of_any_sign(slope):
    pool, bt, k, v, q, aq, ctx = case(FMT_BF16, 64, [3000], [1], 987, DT_BF16)
    check_scored(pool, bt, [3000], q, DT_BF16, aq, ctx, 8, slopes=np.full(8, slope, dtype=np.float32))


@gpu
def test_pages_behind_four_gigabytes():
    """A slab of 5 GiB whose live pages are its last ones: offsets pass 32 bits."""
    import torch

    import gpu_harness as G

    pool, bt, k, v, q, aq, ctx = case(FMT_BF16, 64, [300, 70], [1, 20], 988, DT_BF16)
    pages = (5 << 30) // pool.page
    first = pages - pool.k.size // pool.page
    dpool = G.DevPool(pool)
    for name, host in (("k", pool.k), ("v", pool.v)):
        big = torch.empty(pages * pool.page, dtype=torch.uint8, device=G.DEV)
        big[first * pool.page:first * pool.page + host.size] = torch.from_numpy(host).to(G.DEV)
        setattr(dpool, name, big)
    hb = oracle.HostBatch(aq, [300, 70], bt + first, context_lens_before=ctx)
    bits, lse = run_scored(pool, hb, q, DT_BF16, 8, cap=30.0, dpool=dpool)
    near, near_lse = run_scored(pool, oracle.HostBatch(aq, [300, 70], bt, context_lens_before=ctx), q, DT_BF16, 8, cap=30.0)
    assert bits.tobytes() == near.tobytes() and lse.tobytes() == near_lse.tobytes()


@gpu
def test_same_bits_whatever_the_pages_and_bounds():
    seqs, qs = [2000, 300], [1, 2]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 64, seqs, qs, 989, DT_F16)
    a = check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, cap=30.0)
    b = check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, cap=30.0)
    wide = np.zeros((2, bt.shape[1] + 30), dtype=np.int32)
    wide[:, :bt.shape[1]] = bt
    c = check_scored(pool, wide, seqs, q, DT_F16, aq, ctx, 8, cap=30.0)
    d = check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, cap=30.0, max_seq_len=100000)
    e = check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, cap=30.0, max_seq_len=0)
    for other in (b, c, d, e):
        assert a[0].tobytes() == other[0].tobytes() and a[1].tobytes() == other[1].tobytes()


@gpu
@pytest.mark.parametrize("qs", [[1, 1, 1], [1, 30, 6], [1, 70, 6]])
def test_captured_call_follows_lengths_tables_and_terms(qs):
    """A graph of the call, replayed after lengths, tables, document starts and queries have changed, with eager work between; two
    graphs share the workspace."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    seqs = [1500, 300, 40]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, seqs, qs, 990, DT_BF16)
    dpool = G.DevPool(pool)
    dpool.upload()
    layout = dpool.layout()
    n = aq[-1]
    hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx)
    db = G.DevBatch(hb)
    batch = db.struct()
    ws = torch.zeros(8 << 20, dtype=torch.uint8, device=G.DEV)
    qd = G.to_dev(q)
    outs = [torch.zeros((n, 8, 256), dtype=torch.int16, device=G.DEV) for _ in range(2)]
    lses = [torch.zeros((n, 8), dtype=torch.float32, device=G.DEV) for _ in range(2)]
    doc = np.zeros(n, dtype=np.int32)
    made = [scores_struct(G, cap=30.0, documents=doc, lse=l) for l in lses]
    fn = G.lib().warp34_paged_attention_scored_bf16

    def run(which, stream):
        ex = ffi.Warp34Exec(stream.cuda_stream, ws.data_ptr(), ws.numel(), 0)
        assert fn(C.byref(ex), C.byref(layout), C.byref(batch), C.byref(made[which][0]), G.ptr(qd), G.ptr(outs[which]), 8) == 0

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(0, side)
    torch.cuda.synchronize()
    graphs = []
    for which in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(which, torch.cuda.current_stream())
        graphs.append(graph)
    for turn, lens in enumerate(([1500, 300, 40], [700, 299, 33], [1, 1, 1] if max(qs) == 1 else [800, qs[1] + 1, 7])):
        now_ctx = [s - a for s, a in zip(lens, qs)]
        db.t["seq"].copy_(G.to_dev(np.asarray(lens, dtype=np.int32)))
        db.t["ctx"].copy_(G.to_dev(np.asarray(now_ctx, dtype=np.int32)))
        new_doc = np.full(n, 5 * turn, dtype=np.int32)
        for m in made:
            m[1][1].copy_(G.to_dev(new_doc))
        new_q = np.roll(q, turn, axis=0)
        qd.copy_(G.to_dev(new_q))
        want, want_lse, bound, lse_bound = scored_attention(pool, bt, lens, oracle.bits_to_f32(new_q, DT_BF16).astype(np.float64), aq, now_ctx,
                                                            cap=30.0, documents=new_doc, scale=hb.sm_scale, dt=DT_BF16,
                                                            chunk=max(qs) * 4 >= CHUNK_FROM)
        for which in (0, 1, 0):
            outs[which].zero_()
            graphs[which].replay()
            torch.cuda.synchronize()
            got = oracle.bits_to_f32(outs[which].cpu().numpy().view(np.uint16), DT_BF16).astype(np.float64)
            assert (np.abs(got - want) <= bound).all()
            seen = ~np.isneginf(want_lse)
            assert (np.abs(lses[which].cpu().numpy()[seen] - want_lse[seen]) <= lse_bound[seen]).all()


@gpu
def test_append_read_attention_and_merge_together():
    """A request's keys in two caches: the older ones in TQ4 pages, read back into BF16 pages of a second cache, the newer ones appended
    there too; attention over both halves, joined, equals attention over the whole."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    seq, cut, heads = 700, 432, 8
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, [seq], [1], 995, DT_BF16)
    dpool = G.DevPool(pool)
    dpool.upload()
    slots = oracle.slot_mapping(bt[0], 0, seq, 16)
    lib, layout = G.lib(), dpool.layout()
    rows = [torch.zeros((seq, 512), dtype=torch.bfloat16, device=G.DEV) for _ in range(2)]
    ex, ws = G.make_exec(8 << 20)
    d_slots = G.to_dev(slots)
    assert lib.warp34_kv_cache_read_bf16(C.byref(ex), C.byref(layout), G.ptr(d_slots), seq, G.ptr(rows[0]), G.ptr(rows[1]), 512, 512) == 0
    wide = oracle.HostPool(pool.k.size // pool.page, 2, 256, 16, FMT_BF16, XF_IDENTITY)
    dwide = G.DevPool(wide)
    wide_layout = dwide.layout()
    wb = G.DevBatch(oracle.HostBatch([0, seq], [seq], bt, context_lens_before=[0], write_slot_mapping=slots))
    write = wb.struct()
    assert lib.warp34_kv_cache_write_bf16(C.byref(ex), C.byref(wide_layout), C.byref(write), G.ptr(rows[0]), G.ptr(rows[1])) == 0
    qd = G.to_dev(q)
    parts = torch.zeros((2, heads, 256), dtype=torch.int16, device=G.DEV)
    lses = torch.zeros((2, heads), dtype=torch.float32, device=G.DEV)
    halves = [(0, cut, 1), (cut, seq, 0)]  # (the older keys lie before every position: all of them are seen)
    keep = []
    for i, (a, e, mode) in enumerate(halves):
        hb = oracle.HostBatch([0, 1], [e - a], bt[:, a // 16:(e + 15) // 16], context_lens_before=[e - a - 1], mask_mode=mode)
        db = G.DevBatch(hb)
        batch = db.struct()
        scores = ffi.Warp34AttentionScores(None, None, None, lses[i].data_ptr(), 30.0, 0)
        keep += [db, batch, scores]
        assert lib.warp34_paged_attention_scored_bf16(C.byref(ex), C.byref(wide_layout), C.byref(batch), C.byref(scores), G.ptr(qd),
                                                      G.ptr(parts[i]), heads) == 0
    out = torch.zeros((heads, 256), dtype=torch.int16, device=G.DEV)
    lse = torch.zeros(heads, dtype=torch.float32, device=G.DEV)
    assert lib.warp34_attention_merge_bf16(C.byref(ex), G.ptr(parts), G.ptr(lses), 2, heads * 256, heads, G.ptr(out), G.ptr(lse), heads,
                                           256) == 0
    torch.cuda.synchronize()
    wide.k, wide.v = dwide.download()
    q64 = oracle.bits_to_f32(q, DT_BF16).astype(np.float64)
    scale = 256 ** -0.5
    want, want_lse, bound, lse_bound = scored_attention(wide, bt, [seq], q64, aq, ctx, cap=30.0, scale=scale, dt=DT_BF16)
    # a part's own rounding: half a step of each part, which the weights only average
    half = [scored_attention(wide, bt[:, a // 16:], [e - a], q64, [0, 1], [e - a - 1], cap=30.0, noncausal=True, scale=scale, dt=DT_BF16)
            for a, e, _ in halves]
    room = bound[0] + 2.0 ** -8 * np.maximum(np.abs(half[0][0][0]), np.abs(half[1][0][0])) + 2.0 ** -15 * np.abs(want[0])
    got = oracle.bits_to_f32(out.cpu().numpy().view(np.uint16), DT_BF16).astype(np.float64)
    assert (np.abs(got - want[0]) <= room).all()
    assert (np.abs(lse.cpu().numpy() - want_lse[0]) <= lse_bound[0] + 2.0 ** -20 * (1 + np.abs(want_lse[0]))).all()


def _call(name="warp34_paged_attention_scored_bf16", layout_over=(), batch_over=(), scores_over=(), null=None, heads=16, q=1 << 24, out=1 << 25):
    from warp34_amd import ffi

    ex = ffi.Warp34Exec(0, 0, 0, 0)
    layout = ffi.Warp34KvLayerLayout(1 << 20, 1 << 21, 132 * 32, 132 * 16, 132, 132 * 32, 132 * 16, 132, 0, 0, 2, 256, 16, FMT_TQ4, FMT_TQ4,
                                     XF_WHT256, XF_WHT256, 0)
    batch = ffi.Warp34AttentionBatch(1 << 16, None, 1 << 17, 1 << 18, None, None, None, 1, 1, 4, 1, 64, 0, 0, 0.0625, 0)
    scores = ffi.Warp34AttentionScores(None, None, None, None, 0.0, 0)
    for target, over in ((layout, layout_over), (batch, batch_over), (scores, scores_over)):
        for key, value in dict(over).items():
            setattr(target, key, value)
    args = [C.byref(ex), C.byref(layout), C.byref(batch), C.byref(scores), q, out, heads]
    if null is not None:
        args[null] = None
    return getattr(ffi.load(), name)(*args)


@pytest.mark.parametrize("null", range(6))
def test_null_arguments_are_refused(null):
    assert _call(null=null) == 1


@pytest.mark.parametrize("over,code", [
    (dict(heads=0), 1), (dict(heads=15), 1), (dict(batch_over={"total_tokens": -1}), 1), (dict(batch_over={"total_tokens": 0}), 0),
    (dict(batch_over={"num_reqs": 0}), 1), (dict(batch_over={"query_start_loc": None}), 1), (dict(batch_over={"seq_lens_after": None}), 1),
    (dict(batch_over={"block_tables": None}), 1), (dict(batch_over={"max_blocks_per_req": 0}), 1), (dict(batch_over={"sliding_window": -1}), 1),
    (dict(batch_over={"mask_mode": 2}), 1), (dict(scores_over={"softcap": -1.0}), 1), (dict(scores_over={"softcap": float("nan")}), 1),
    (dict(scores_over={"softcap": float("inf")}), 1), (dict(layout_over={"local_kv_heads": 0}), 1), (dict(layout_over={"k_format": FMT_FP8}), 801),
    (dict(layout_over={"k_format": FMT_FP16, "v_format": FMT_FP16}), 801), (dict(layout_over={"head_dim": 128}), 801),
    (dict(layout_over={"block_size": 24}), 801), (dict(layout_over={"block_size": 0}), 801), (dict(layout_over={"k_token_stride_bytes": 136}), 801),
    (dict(layout_over={"k_base": (1 << 20) + 4}), 801), (dict(layout_over={"k_transform": 7}), 801), (dict(q=(1 << 24) + 8), 801),
    (dict(out=(1 << 25) + 4), 801), (dict(scores_over={"lse_out": (1 << 26) + 2}), 801)])
def test_refusals(over, code):
    assert _call(**over) == code


def test_f16_entry_takes_fp16_pages_and_bf16_entry_bf16_pages():
    sixteen = dict(k_token_stride_bytes=512, v_token_stride_bytes=512, k_transform=0, v_transform=0)
    assert _call("warp34_paged_attention_scored_f16", layout_over=dict(sixteen, k_format=FMT_BF16, v_format=FMT_BF16)) == 801
    assert _call("warp34_paged_attention_scored_bf16", layout_over=dict(sixteen, k_format=FMT_FP16, v_format=FMT_FP16)) == 801


def test_descriptor_has_the_size_that_the_header_states():
    from warp34_amd import ffi

    assert C.sizeof(ffi.Warp34AttentionScores) == 40


@pytest.mark.parametrize("kv_heads,heads", [(1, 8), (2, 16), (4, 32), (40, 40)])
@pytest.mark.parametrize("fmt", [FMT_TQ4, FMT_FP8])
def test_scratch_grows_with_the_batch_and_ends_where_nothing_is_cut(fmt, kv_heads, heads):
    from warp34_amd import ffi

    layout = ffi.Warp34KvLayerLayout(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, kv_heads, 256, 16, fmt, fmt, 1, 1, 0)
    size = ffi.load().warp34_paged_attention_scored_scratch_bytes
    sizes = [size(C.byref(layout), n, n, 1, heads) for n in (100, 300, 1000, 2000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert size(C.byref(layout), 2100, 2100, 1, heads) == 0


def test_scratch_query():
    from warp34_amd import ffi

    layout = ffi.Warp34KvLayerLayout(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 2, 256, 16, FMT_TQ4, FMT_TQ4, 1, 1, 0)
    size = ffi.load().warp34_paged_attention_scored_scratch_bytes
    one = size(C.byref(layout), 1, 1, 1, 16)
    assert 0 < one <= 8 << 20  # what the reference's engine guarantees
    assert size(C.byref(layout), 32, 32, 1, 16) >= one
    for args in ((0, 1, 1, 16), (1, 0, 1, 16), (1, 1, 1, 0), (1, 1, 1, 15)):
        assert size(C.byref(layout), *args) == 0
    assert size(None, 1, 1, 1, 16) == 0
    assert SENTINEL


@gpu
@pytest.mark.parametrize("fmt,xf,v_xf,dt,hd", FORMS)
@pytest.mark.parametrize("seqs,qs,terms", [([70], [70], {"cap": 30.0}), ([333, 1100], [100, 65], {"sloped": True}),
                                           ([200, 90], [150, 90], {"cap": 5.0, "window": 50})])
def test_chunks(fmt, xf, v_xf, dt, hd, seqs, qs, terms):
    """Many query columns: several tiles, ranges that end inside a unit, keys split and joined."""
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 1000 + hd, dt, xf=xf, v_xf=v_xf, head_dim=hd)
    terms = dict(terms)
    if terms.pop("sloped", False):
        terms["slopes"] = slopes_of(8)
    for scratch in (0, 64 << 20):
        check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, **terms)


@gpu
@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (2, 16), (1, 24), (1, 17), (3, 9), (1, 64)])
def test_chunk_head_layouts(kv_heads, heads):
    seqs, qs = [300], [260]
    pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 16, seqs, qs, 1020 + heads, DT_F16, kv_heads=kv_heads, q_heads=heads, head_dim=128)
    check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, heads, cap=20.0, slopes=slopes_of(heads))


@gpu
@pytest.mark.parametrize("block", [16, 48, 128])
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_BF16, DT_BF16)])
def test_chunk_page_sizes_and_odd_starts(fmt, dt, block):
    """Windows that open at odd half units, so that a unit of keys lies in two pages."""
    seqs, qs = [500, 97], [64, 33]
    pool, bt, k, v, q, aq, ctx = case(fmt, block, seqs, qs, 1040 + block, dt)
    for window in (0, 130, 150):
        check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=64 << 20, cap=30.0, window=window)


@gpu
@pytest.mark.parametrize("fmt,xf,dt", [(FMT_TQ4, XF_WHT256, DT_F16), (FMT_BF16, XF_IDENTITY, DT_BF16), (FMT_Q8_0, XF_IDENTITY, DT_F16),
                                       (FMT_FP8, XF_WHT256, DT_F16)])
@pytest.mark.parametrize("scratch", [0, 64 << 20])
def test_chunk_documents_prefixes_windows_and_empty_rows(fmt, xf, dt, scratch):
    seqs, qs = [400, 161, 250], [170, 161, 3]
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 1060, dt, xf=xf)
    rng = np.random.default_rng(6)
    pos = np.concatenate([np.arange(n) + c for n, c in zip(qs, ctx)])
    doc = (pos // 37 * 37).astype(np.int32)
    doc[::9] = 100000
    doc[40:80] = 1 << 30                 # tiles of which whole waves see nothing
    doc[5] = -4
    pre = rng.integers(-3, 600, pos.size).astype(np.int32)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, documents=doc)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, documents=doc, prefixes=pre, cap=30.0, slopes=slopes_of(8))
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, scratch=scratch, noncausal=True, window=100, slopes=slopes_of(8))


@gpu
def test_chunk_whose_tokens_all_see_nothing():
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, [200], [100], 1070, DT_BF16)
    check_scored(pool, bt, [200], q, DT_BF16, aq, ctx, 8, documents=np.full(100, 5000, dtype=np.int32))


@gpu
@pytest.mark.parametrize("scratch", [0, 64 << 20])
def test_chunk_masked_tokens_and_requests_stay_untouched(scratch):
    seqs, qs = [300, 500, 90], [140, 60, 90]
    pool, bt, k, v, q, aq, ctx = case(FMT_TQ4, 16, seqs, qs, 1080, DT_F16)
    tmask = np.ones(aq[-1], dtype=np.uint8)
    tmask[::5] = 0
    tmask[40:100] = 0
    rmask = np.array([1, 0, 1], dtype=np.uint8)
    hb = oracle.HostBatch(aq, seqs, bt, context_lens_before=ctx, valid_token_mask=tmask, valid_req_mask=rmask)
    rows = tmask.astype(bool)
    rows[aq[1]:aq[2]] = False
    check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, hb=hb, rows=rows, cap=30.0, scratch=scratch)


@gpu
@pytest.mark.parametrize("fmt,xf,dt", [(FMT_TQ4, XF_WHT256, DT_BF16), (FMT_FP8, XF_IDENTITY, DT_F16), (FMT_FP8, XF_WHT256, DT_F16),
                                       (FMT_Q8_0, XF_IDENTITY, DT_F16), (FMT_FP16, XF_IDENTITY, DT_F16), (FMT_BF16, XF_IDENTITY, DT_BF16)])
def test_chunk_what_unseen_rows_hold_does_not_matter(fmt, xf, dt):
    """Bytes of 0xFF behind the sequence and before the window, in the pages of a chunk."""
    seq, n = 213, 137
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, [seq], [n], 1090, dt, xf=xf)
    window = 40
    seen_from = seq - n - window + 1
    wild = np.ones(pool.k.size // pool.page * 16, dtype=bool)
    wild[oracle.slot_mapping(bt[0], seen_from, seq - seen_from, 16)] = False
    views = [s.reshape(-1, pool.kv_heads, 16, pool.tok) for s in (pool.k, pool.v)]
    keep = [s.copy() for s in views]
    for s in views:
        for h in range(pool.kv_heads):
            s[:, h][wild.reshape(-1, 16)] = 0xFF
    hb = oracle.HostBatch(aq, [seq], bt, context_lens_before=ctx)
    hb.sliding_window = window
    bits, lse = run_scored(pool, hb, q, dt, 8, cap=30.0)
    for s, old in zip(views, keep):
        s[:] = old
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [seq], oracle.bits_to_f32(q, dt).astype(np.float64), aq, ctx, cap=30.0,
                                                        window=window, scale=hb.sm_scale, dt=dt, chunk=True)
    got = oracle.bits_to_f32(bits, dt).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()


@gpu
@pytest.mark.parametrize("fmt,dt", [(FMT_FP16, DT_F16), (FMT_TQ4, DT_BF16)])
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 31, 32, 33, 64, 65])
def test_requests_of_any_number_of_tokens(fmt, dt, tokens):
    """From one kernel's range into the other's: 8 query heads of a kv head, so 128 columns at 16 tokens, 256 at 32."""
    seqs, qs = [tokens + 200, tokens], [tokens, tokens]
    pool, bt, k, v, q, aq, ctx = case(fmt, 16, seqs, qs, 1100 + tokens, dt, kv_heads=1)
    check_scored(pool, bt, seqs, q, dt, aq, ctx, 8, cap=30.0)


@gpu
@pytest.mark.parametrize("kv_heads,heads", [(1, 8), (4, 8), (16, 16), (40, 40)])
@pytest.mark.parametrize("seqs,qs", [([6000], [1]), ([500] * 20, [1] * 20), ([700, 90], [300, 40])])
def test_kv_heads_share_the_chip(kv_heads, heads, seqs, qs):
    """The cut of a batch goes by the number of kv heads: from 512 chunks for one of them to 16 for each of 40."""
    pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 16, seqs, qs, 1220, DT_F16, kv_heads=kv_heads, q_heads=heads, head_dim=128)
    check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, heads, scratch=64 << 20, cap=30.0)


@gpu
def test_one_long_request_among_many_short_ones():
    """More tiles than a wave has lanes, most of them short: the long one is cut, in both kernels."""
    seqs = [9000] + [40] * 150
    for tokens in (1, 33):
        qs = [tokens] * len(seqs)
        pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 16, seqs, qs, 1200, DT_F16, kv_heads=1, q_heads=8, head_dim=128)
        check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 8, scratch=64 << 20, cap=30.0)


@gpu
@pytest.mark.parametrize("n", [520, 2100])
def test_more_tiles_than_are_cut(n):
    seqs = [int(x) for x in np.random.default_rng(n).integers(1, 60, n)]
    pool, bt, k, v, q, aq, ctx = case(FMT_FP16, 16, seqs, [1] * n, 1210, DT_F16, kv_heads=1, q_heads=2, head_dim=128)
    check_scored(pool, bt, seqs, q, DT_F16, aq, ctx, 2, scratch=64 << 20, cap=30.0)
