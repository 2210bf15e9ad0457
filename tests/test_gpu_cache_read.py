"""warp34_kv_cache_read_*: rows that the append wrote (oracle bytes), decoded, against float64.

Tolerance: the result is rounded once, half a step of |want|.  Plain rows are a product of two exact numbers in 32 bits (2^-24, far
below a 16-bit half step; 2^-10 of that half step covers it).  Rotated rows: with x the stored values relative to the row's largest
block scale, the two fp16 parts of an operand leave at most 2^-22 |x| + 2^-25 (the second part's smallest step), and so do those of
the 16-term sums of the first product; 256 stored values of at most c (TQ4 0.17, E4M3 448, Q8_0 127 scales) give
(256 * (2^-22 c + 2^-25) + 16 * 2^-22 * 16 c + 256 c * 2^-22) / 16 <= 14.3e-6 c for every c >= 0.17: 1.5e-5 of the row's largest
stored magnitude bound."""
import ctypes as C

import numpy as np
import pytest

import oracle
from cases import make_case
from oracle import (DT_BF16, DT_F16, FMT_BF16, FMT_FP16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_IDENTITY, XF_WHT256)
from plain_kv import HALF_STEP, HALF_TINY, decoded_rows, slab_rows

SENTINEL = 0x5500
LARGEST = {FMT_TQ4: 0.1694104124, FMT_FP8: 448.0, FMT_Q8_0: 127.0}


def call(pool, dt, slots, want_k=True, want_v=True, stride=None, layout_over=(), k=None, v=None):
    import torch

    import gpu_harness as G

    dpool = G.DevPool(pool)
    dpool.upload()
    layout = dpool.layout()
    for name, value in layout_over:
        setattr(layout, name, value)
    width = pool.kv_heads * pool.head_dim
    stride = width if stride is None else stride
    n = len(slots)
    d_slots = G.to_dev(np.asarray(slots, dtype=np.int32))
    outs = [torch.full((max(n, 1), stride), SENTINEL, dtype=torch.int16, device=G.DEV) for _ in range(2)]
    fn = G.lib().warp34_kv_cache_read_bf16 if dt == DT_BF16 else G.lib().warp34_kv_cache_read_f16
    ex, _ = G.make_exec(0)
    rc = fn(C.byref(ex), C.byref(layout), G.ptr(d_slots), n, G.ptr(outs[0]) if want_k else None,
            G.ptr(outs[1]) if want_v else None, stride, stride)
    torch.cuda.synchronize()
    assert rc == 0
    return [o.cpu().numpy().view(np.uint16) for o in outs]


def stored_scale(rows, fmt, head_dim):
    """The row's largest block scale times the format's largest code value; 0 for 16-bit rows."""
    if fmt == FMT_TQ4:
        d = np.ascontiguousarray(rows.reshape(*rows.shape[:-1], head_dim // 128, 66)[..., :2]).view(np.float16)
    elif fmt == FMT_FP8:
        d = np.ascontiguousarray(rows[..., 256:264]).view(np.float32)
    elif fmt == FMT_Q8_0:
        d = np.ascontiguousarray(rows.reshape(*rows.shape[:-1], 4, 68)[..., :4]).view(np.float32)
    else:
        return np.zeros(rows.shape[:-1])
    return np.abs(d.astype(np.float64)).reshape(*rows.shape[:-1], -1).max(-1) * LARGEST[fmt]


def check(got, dt, rows, fmt, xf, head_dim):
    with np.errstate(invalid="ignore"):
        want = decoded_rows(rows, fmt, xf, head_dim)
    got = oracle.bits_to_f32(np.ascontiguousarray(got), dt).astype(np.float64).reshape(want.shape)
    bound = HALF_STEP[dt] * (1 + 2.0 ** -10) * np.abs(want) + HALF_TINY[dt]
    if xf == XF_WHT256:
        bound = bound + 1.5e-5 * stored_scale(rows, fmt, head_dim)[..., None]
    fine = np.isfinite(want)  # (a row whose scale has left fp16's range has no values)
    assert not np.isfinite(got[~fine]).any()
    with np.errstate(invalid="ignore"):
        worst = np.where(fine, np.abs(got - want) - bound, -1.0)
    assert worst.max() <= 0, (worst.max(), np.unravel_index(worst.argmax(), worst.shape))


FORMS = [(FMT_TQ4, XF_WHT256, 256), (FMT_TQ4, XF_IDENTITY, 256), (FMT_TQ4, XF_IDENTITY, 128), (FMT_FP8, XF_IDENTITY, 256),
         (FMT_FP8, XF_WHT256, 256), (FMT_Q8_0, XF_IDENTITY, 256), (FMT_Q8_0, XF_WHT256, 256), (FMT_FP16, XF_IDENTITY, 256),
         (FMT_FP16, XF_IDENTITY, 128), (FMT_BF16, XF_IDENTITY, 256), (FMT_BF16, XF_IDENTITY, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [DT_F16, DT_BF16])
@pytest.mark.parametrize("fmt,xf,hd", FORMS)
@pytest.mark.parametrize("rows,block,kv_heads", [(1, 16, 2), (37, 16, 1), (333, 64, 3)])
def test_rows_come_back(fmt, xf, hd, dt, rows, block, kv_heads):
    in_dt = dt if fmt in (FMT_TQ4, FMT_FP8, FMT_Q8_0) else DT_BF16 if fmt == FMT_BF16 else DT_F16
    pool, bt, *_ = make_case(fmt, block, [rows], [1], 700 + rows, in_dt, kv_heads=kv_heads, q_heads=kv_heads, xf=xf, head_dim=hd)
    slots = oracle.slot_mapping(bt[0], 0, rows, block)
    for got, slab in zip(call(pool, dt, slots), (pool.k, pool.v)):
        check(got, dt, slab_rows(slab, pool, slots), fmt, xf, hd)


@pytest.mark.gpu
def test_negative_slots_repeats_strides_and_single_slabs():
    pool, bt, *_ = make_case(FMT_TQ4, 16, [200], [1], 811, DT_BF16)
    slots = np.concatenate([oracle.slot_mapping(bt[0], 0, 200, 16)[::-3], [-1, 5, 5, -7, 5]]).astype(np.int32)
    for k, v in ((True, True), (True, False), (False, True)):
        outs = call(pool, DT_F16, slots, k, v, stride=2 * 256 + 40)
        for wanted, got, slab in zip((k, v), outs, (pool.k, pool.v)):
            assert (got[:, 512:] == SENTINEL).all()
            live = (slots >= 0) & wanted
            assert (got[~live] == SENTINEL).all()
            if wanted:
                check(got[live][:, :512], DT_F16, slab_rows(slab, pool, slots[live]), FMT_TQ4, XF_WHT256, 256)


@pytest.mark.gpu
def test_slabs_of_different_transforms():
    """K rotated, V as it is: two launches."""
    pool, bt, *_ = make_case(FMT_TQ4, 64, [90], [1], 812, DT_BF16, v_xf=XF_IDENTITY)
    slots = oracle.slot_mapping(bt[0], 0, 90, 64)
    k, v = call(pool, DT_BF16, slots)
    check(k, DT_BF16, slab_rows(pool.k, pool, slots), FMT_TQ4, XF_WHT256, 256)
    check(v, DT_BF16, slab_rows(pool.v, pool, slots), FMT_TQ4, XF_IDENTITY, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [FMT_TQ4, FMT_Q8_0])
def test_rows_of_zeros_and_of_extreme_scales(fmt):
    """Rotated rows whose scales are zero, or as small and as large as fp16 inputs make them, out of fp16's range too."""
    pool, bt, *_ = make_case(fmt, 16, [64], [1], 813, DT_F16, kv_heads=1, q_heads=1, xf=XF_WHT256)
    x = np.random.default_rng(3).standard_normal((64, 1, 256)).astype(np.float32)
    x *= np.array([0.0, 1e-6, 3e-5, 1.0, 1000.0, 4000.0], dtype=np.float32)[np.arange(64) % 6][:, None, None]
    bits = oracle.f32_to_f16_bits(x)
    wb = oracle.HostBatch([0, 64], [64], bt, context_lens_before=[0], write_slot_mapping=oracle.slot_mapping(bt[0], 0, 64, 16))
    oracle.kv_cache_write(pool, wb, bits, bits, DT_F16)
    slots = oracle.slot_mapping(bt[0], 0, 64, 16)
    for got, slab in zip(call(pool, DT_F16, slots), (pool.k, pool.v)):
        check(got, DT_F16, slab_rows(slab, pool, slots), fmt, XF_WHT256, 256)


@pytest.mark.gpu
def test_written_rows_read_back_are_the_values_attention_uses():
    """Append, read, append the read rows into BF16 pages: attention over both caches agrees within the parity bound."""
    import gpu_harness as G

    pool, bt, k, v, q, aq, ctx = make_case(FMT_FP8, 16, [150], [2], 814, DT_BF16)
    slots = oracle.slot_mapping(bt[0], 0, 150, 16)
    kr, vr = call(pool, DT_BF16, slots)
    wide = oracle.HostPool(pool.k.size // pool.page, 2, 256, 16, FMT_BF16, XF_IDENTITY)
    wb = oracle.HostBatch([0, 150], [150], bt, context_lens_before=[0], write_slot_mapping=slots)
    oracle.kv_cache_write(wide, wb, kr.reshape(150, 2, 256), vr.reshape(150, 2, 256), DT_BF16)
    hb = oracle.HostBatch(aq, [150], bt, context_lens_before=ctx)
    dwide = G.DevPool(wide)
    dwide.upload()
    rc, got, _ = G.dev_attention(dwide, hb, q, DT_BF16, 8, scratch_bytes=8 << 20)
    assert rc == 0
    want = oracle.paged_attention(wide, hb, q, DT_BF16, 8)
    G.assert_close(got, DT_BF16, want, what="read rows", scale=G.channel_scale(v, DT_BF16, hb, 8))


@pytest.mark.gpu
def test_captured_read_follows_pages_and_slots():
    """A graph of the call, replayed after pages and slots have changed, with eager work between."""
    import torch

    import gpu_harness as G

    pool, bt, *_ = make_case(FMT_TQ4, 16, [64], [1], 815, DT_BF16)
    dpool = G.DevPool(pool)
    dpool.upload()
    layout = dpool.layout()
    slots = oracle.slot_mapping(bt[0], 0, 64, 16)
    d_slots = G.to_dev(slots)
    outs = [torch.zeros((64, 512), dtype=torch.bfloat16, device=G.DEV) for _ in range(2)]

    def run(stream):
        from warp34_amd import ffi

        ex = ffi.Warp34Exec(stream.cuda_stream, 0, 0, 0)
        assert G.lib().warp34_kv_cache_read_bf16(C.byref(ex), C.byref(layout), G.ptr(d_slots), 64, G.ptr(outs[0]), G.ptr(outs[1]),
                                                 512, 512) == 0

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(torch.cuda.current_stream())
    for turn in range(3):
        d_slots.copy_(G.to_dev(np.roll(slots, 5 * turn)))
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, slab in zip(outs, (pool.k, pool.v)):
            bits = got.view(torch.int16).cpu().numpy().view(np.uint16)
            check(bits, DT_BF16, slab_rows(slab, pool, np.roll(slots, 5 * turn)), FMT_TQ4, XF_WHT256, 256)


def _layout(**over):
    from warp34_amd import ffi

    fields = dict(k_base=1 << 20, v_base=1 << 21, k_page_stride_bytes=132 * 32, k_head_stride_bytes=132 * 16, k_token_stride_bytes=132,
                  v_page_stride_bytes=132 * 32, v_head_stride_bytes=132 * 16, v_token_stride_bytes=132, local_kv_heads=2, head_dim=256,
                  block_size=16, k_format=FMT_TQ4, v_format=FMT_TQ4, k_transform=XF_WHT256, v_transform=XF_WHT256)
    fields.update(over)
    return ffi.Warp34KvLayerLayout(**fields)


@pytest.mark.parametrize("over,args,code", [
    ({}, dict(slots=None), 1), ({}, dict(k=None, v=None), 1), ({}, dict(k_stride=511), 1), ({}, dict(v_stride=256), 1),
    ({"block_size": 0}, {}, 1), ({"k_base": 0}, {}, 1), ({"head_dim": 0}, {}, 1), ({"head_dim": 264}, {}, 1),
    ({"k_format": 9}, {}, 801), ({"k_format": FMT_FP16}, {}, 801), ({"v_format": FMT_FP8, "v_base": (1 << 21) + 2}, {}, 801),
    ({"k_base": (1 << 20) + 1}, {}, 801), ({}, dict(k_stride=516), 801), ({}, dict(k=(1 << 22) + 8), 801),
    ({"head_dim": 64}, {}, 801), ({"local_kv_heads": 65536}, dict(k_stride=1 << 25, v_stride=1 << 25), 1),
    ({}, dict(rows=0), 0), ({}, dict(rows=-3), 0), ({"local_kv_heads": 0}, {}, 0)])
@pytest.mark.parametrize("name", ["warp34_kv_cache_read_f16", "warp34_kv_cache_read_bf16"])
def test_refusals(name, over, args, code):
    """Arguments that are refused, or leave nothing to do, before anything is launched."""
    from warp34_amd import ffi

    a = dict(slots=1 << 23, rows=5, k=1 << 22, v=3 << 22, k_stride=512, v_stride=512)
    a.update(args)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    layout = _layout(**over)
    fn = getattr(ffi.load(), name)
    assert fn(C.byref(ex), C.byref(layout), a["slots"], a["rows"], a["k"], a["v"], a["k_stride"], a["v_stride"]) == code


def test_null_descriptors_are_refused():
    from warp34_amd import ffi

    fn = ffi.load().warp34_kv_cache_read_f16
    ex, layout = ffi.Warp34Exec(0, 0, 0, 0), _layout()
    assert fn(None, C.byref(layout), 1 << 23, 5, 1 << 22, None, 512, 512) == 1
    assert fn(C.byref(ex), None, 1 << 23, 5, 1 << 22, None, 512, 512) == 1
