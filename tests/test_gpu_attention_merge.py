"""warp34_attention_merge_*: partial attention results joined, against float64.

Tolerance: with w_p the exact weights, sums in 32 bits of num_parts terms and weights from exp2 of arguments up to 2^7 that are
rounded in 32 bits (an argument's rounding of 2^-24 * 2^7 is 2^-17 of the weight, the same in numerator and denominator only for
equal parts): 2^-16 of sum_p w_p |out_p|, and the output's half step.  lse: 2^-22 of its size and of 1."""
import ctypes as C

import numpy as np
import pytest

import oracle
from oracle import DT_BF16, DT_F16
from plain_kv import HALF_STEP, HALF_TINY


def plain(parts, lse):
    with np.errstate(all="ignore"):
        top = lse.max(0)
        top = np.where(np.isfinite(top), top, 0.0)
        w = np.where(lse == -np.inf, 0.0, np.exp(lse - top))
        total = w.sum(0)
        share = w / np.where(total > 0, total, 1.0)
        seen = np.where((lse == -np.inf)[..., None], 0.0, parts)
        return (share[..., None] * seen).sum(0), np.log(total) + top, (share[..., None] * np.abs(seen)).sum(0)


def call(bits, lse, dt, out=None, with_lse=True, part_pad=0, lse_pad=0):
    import torch

    import gpu_harness as G

    n, rows, hd = bits.shape
    d = torch.full((n, rows * hd + part_pad), 0x7FFF, dtype=torch.int16, device=G.DEV)
    d[:, :rows * hd] = torch.from_numpy(bits.reshape(n, -1).view(np.int16)).to(G.DEV)
    dl = torch.full((n, rows + lse_pad), float("nan"), dtype=torch.float32, device=G.DEV)
    dl[:, :rows] = torch.from_numpy(lse.astype(np.float32)).to(G.DEV)
    got = torch.full((rows + 1, hd), 0x5500, dtype=torch.int16, device=G.DEV)
    got_lse = torch.full((rows + 1,), 77.0, dtype=torch.float32, device=G.DEV)
    target = got if out is None else d[out]
    ex, _ = G.make_exec(0)
    fn = G.lib().warp34_attention_merge_bf16 if dt == DT_BF16 else G.lib().warp34_attention_merge_f16
    rc = fn(C.byref(ex), G.ptr(d), G.ptr(dl), n, rows * hd + part_pad, rows + lse_pad, G.ptr(target),
            G.ptr(got_lse) if with_lse else None, rows, hd)
    torch.cuda.synchronize()
    assert rc == 0
    assert bool((got[rows] == 0x5500).all()) and float(got_lse[rows]) == 77.0
    res = target.reshape(-1)[:rows * hd].reshape(rows, hd).cpu().numpy().view(np.uint16)
    return oracle.bits_to_f32(np.ascontiguousarray(res), dt).astype(np.float64), got_lse[:rows].cpu().numpy().astype(np.float64)


def make(n, rows, hd, dt, seed, spread=2.0, none=0.0):
    rng = np.random.default_rng(seed)
    bits = oracle.fill_normal(n * rows * hd, seed, dt).reshape(n, rows, hd)
    lse = (rng.standard_normal((n, rows)) * spread + 6).astype(np.float32).astype(np.float64)
    lse[rng.random((n, rows)) < none] = -np.inf
    return bits, lse


def check(got, bits, lse, dt, with_lse=True):
    want, want_lse, size = plain(oracle.bits_to_f32(bits, dt).astype(np.float64), lse)
    out, out_lse = got
    bound = HALF_STEP[dt] * np.abs(want) + 2.0 ** -16 * size + HALF_TINY[dt]
    assert (np.abs(out - want) <= bound).all(), np.max(np.abs(out - want) - bound)
    if with_lse:
        empty = np.isneginf(want_lse)
        assert np.isneginf(out_lse[empty]).all()
        assert (np.abs(out_lse[~empty] - want_lse[~empty]) <= 2.0 ** -22 * (np.abs(want_lse[~empty]) + 1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [DT_F16, DT_BF16])
@pytest.mark.parametrize("n,rows,hd", [(1, 1, 256), (2, 16, 256), (3, 7, 128), (5, 1001, 256), (8, 33, 64), (9, 5, 8), (16, 3, 2048),
                                       (4, 11, 96), (33, 65, 256)])
def test_parts_are_joined(n, rows, hd, dt):
    bits, lse = make(n, rows, hd, dt, 40 + n, none=0.2)
    check(call(bits, lse, dt), bits, lse, dt)


@pytest.mark.gpu
def test_far_apart_sums_padded_strides_and_no_lse():
    bits, lse = make(4, 50, 256, DT_BF16, 71, spread=40.0)
    check(call(bits, lse, DT_BF16, part_pad=8, lse_pad=3), bits, lse, DT_BF16)
    check(call(bits, lse, DT_BF16, with_lse=False), bits, lse, DT_BF16, with_lse=False)


@pytest.mark.gpu
def test_rows_that_no_part_saw_and_what_unseen_parts_hold():
    bits, lse = make(6, 40, 256, DT_F16, 72, none=0.5)
    lse[:, ::5] = -np.inf
    bits[lse == -np.inf] = 0x7E00  # NaN
    got = call(bits, lse, DT_F16)
    check(got, bits, lse, DT_F16)
    assert (got[0][::5] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("part", [0, 2])
def test_into_the_memory_of_a_part(part):
    bits, lse = make(3, 200, 128, DT_BF16, 73)
    check(call(bits, lse, DT_BF16, out=part), bits, lse, DT_BF16)


@pytest.mark.gpu
def test_one_part_comes_back_as_it_is():
    bits, lse = make(1, 30, 256, DT_F16, 74)
    out, out_lse = call(bits, lse, DT_F16)
    assert (out == oracle.bits_to_f32(bits[0], DT_F16)).all()
    assert (np.abs(out_lse - lse[0]) <= 2.0 ** -22 * (np.abs(lse[0]) + 1)).all()


@pytest.mark.parametrize("args,code", [
    (dict(parts=None), 1), (dict(lse=None), 1), (dict(out=None), 1), (dict(n=0), 1), (dict(hd=0), 1), (dict(rows=0), 0),
    (dict(rows=-1), 0), (dict(hd=12, stride=60), 801), (dict(hd=2056, stride=5 * 2056), 801), (dict(parts=(1 << 20) + 8), 801),
    (dict(out=(1 << 22) + 2), 801), (dict(stride=1284), 801), (dict(stride=1272), 1), (dict(lse_stride=4), 1),
    (dict(rows=1 << 45, stride=1 << 60, lse_stride=1 << 46), 1)])
@pytest.mark.parametrize("name", ["warp34_attention_merge_f16", "warp34_attention_merge_bf16"])
def test_refusals(name, args, code):
    from warp34_amd import ffi

    a = dict(parts=1 << 20, lse=1 << 21, n=2, stride=1280, lse_stride=5, out=1 << 22, rows=5, hd=256)
    a.update(args)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    fn = getattr(ffi.load(), name)
    assert fn(C.byref(ex), a["parts"], a["lse"], a["n"], a["stride"], a["lse_stride"], a["out"], None, a["rows"], a["hd"]) == code
    assert fn(None, a["parts"], a["lse"], a["n"], a["stride"], a["lse_stride"], a["out"], None, a["rows"], a["hd"]) == 1
