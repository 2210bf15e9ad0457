"""Scored attention at the ends of its arguments' ranges: scales of the scores that leave 32 bits, caps beyond every score."""
import numpy as np
import pytest

import oracle
from cases import make_case
from oracle import DT_BF16, DT_F16, FMT_BF16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_IDENTITY, XF_WHT256
from plain_kv import scored_attention
from scored_harness import CHUNK_FROM, check_scored, run_scored

FORMS = [(FMT_TQ4, XF_WHT256), (FMT_TQ4, XF_IDENTITY), (FMT_FP8, XF_WHT256), (FMT_FP8, XF_IDENTITY), (FMT_Q8_0, XF_WHT256), (FMT_Q8_0, XF_IDENTITY),
         (FMT_BF16, XF_IDENTITY)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf", FORMS)
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("scale,size", [(0.0, 2.0 ** -60), (0.0, 2.0 ** -30), (1e-25, 2.0 ** -90), (0.0, 1.0)])
def test_scores_that_are_all_zero(fmt, xf, tokens, scale, size):
    """sm_scale 0 or tiny, tiny queries, no cap: hidden keys stay hidden and the rest count alike."""
    pool, bt, k, v, q, aq, ctx = make_case(fmt, 16, [150], [tokens], 1500, DT_BF16, xf=xf)
    q = oracle.f32_to_bf16_bits(oracle.bits_to_f32(q, DT_BF16) * np.float32(size))
    hb = oracle.HostBatch(aq, [150], bt, context_lens_before=ctx)
    hb.sm_scale = scale
    check_scored(pool, bt, [150], q, DT_BF16, aq, ctx, 8, hb=hb, window=100)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf", FORMS)
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("cap", [1e30, 1e34, 1e36, 1.5e38, 3.4e38])
def test_caps_beyond_every_score_change_nothing(fmt, xf, tokens, cap):
    pool, bt, k, v, q, aq, ctx = make_case(fmt, 16, [200], [tokens], 1501, DT_BF16, xf=xf)
    hb = oracle.HostBatch(aq, [200], bt, context_lens_before=ctx)
    bits, lse = run_scored(pool, hb, q, DT_BF16, 8, cap=cap)
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [200], oracle.bits_to_f32(q, DT_BF16).astype(np.float64), aq, ctx,
                                                        scale=hb.sm_scale, dt=DT_BF16, chunk=tokens * 4 >= CHUNK_FROM)
    got = oracle.bits_to_f32(bits, DT_BF16).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf", [f for f in FORMS if f[0] != FMT_BF16])
@pytest.mark.parametrize("dt", [DT_F16, DT_BF16])
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("size", [1e2, 1e-3, 1e-4, 1e-5, 1e-6])
def test_values_of_any_size(fmt, xf, dt, tokens, size):
    """Quantised values have fp16's relative and absolute steps.  The rotation back in the chunk kernel splits the row's average, and the average
    times a Hadamard matrix of 16, into two fp16 parts each: 2^-25 of an element is left out twice, and 256 of them come together with 1 / 16."""
    pool, bt, k, v, q, aq, ctx = make_case(fmt, 16, [300], [tokens], 1502, dt, xf=xf)
    x = oracle.bits_to_f32(v, dt) * np.float32(size)
    v = oracle.f32_to_bf16_bits(x) if dt == DT_BF16 else oracle.f32_to_f16_bits(x)
    write = oracle.HostBatch([0, 300], [300], bt, context_lens_before=[0], write_slot_mapping=oracle.slot_mapping(bt[0], 0, 300, 16))
    oracle.kv_cache_write(pool, write, k, v, dt)
    hb = oracle.HostBatch(aq, [300], bt, context_lens_before=ctx)
    bits, lse = run_scored(pool, hb, q, dt, 8)
    chunk = tokens * 4 >= CHUNK_FROM
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [300], oracle.bits_to_f32(q, dt).astype(np.float64), aq, ctx,
                                                        scale=hb.sm_scale, dt=dt, chunk=chunk)
    if chunk and xf == XF_WHT256:
        bound = bound + 2 * 16 * 2.0 ** -25
    got = oracle.bits_to_f32(bits, dt).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,xf", FORMS)
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("cap,size", [(1e-30, 1e20), (1e-20, 1e25), (1e-38, 1.0)])
def test_scores_of_zero_under_small_caps_of_large_queries(fmt, xf, tokens, cap, size):
    """Keys of zeros, whose scores are 0 whatever their factor: all keys count alike, and lse is the logarithm of their number."""
    pool, bt, k, v, q, aq, ctx = make_case(fmt, 16, [150], [tokens], 1503, DT_BF16, xf=xf)
    pool.k[:] = 0
    q = oracle.f32_to_bf16_bits(oracle.bits_to_f32(q, DT_BF16) * np.float32(size))
    hb = oracle.HostBatch(aq, [150], bt, context_lens_before=ctx)
    bits, lse = run_scored(pool, hb, q, DT_BF16, 8, cap=cap)
    want, want_lse, bound, lse_bound = scored_attention(pool, bt, [150], oracle.bits_to_f32(q, DT_BF16).astype(np.float64), aq, ctx,
                                                        scale=hb.sm_scale, dt=DT_BF16, chunk=tokens * 4 >= CHUNK_FROM)
    got = oracle.bits_to_f32(bits, DT_BF16).astype(np.float64)
    assert (np.abs(got - want) <= bound).all() and (np.abs(lse - want_lse) <= lse_bound).all()
