"""Plain implementations in 64 bits that the tests of the cache read, the scored attention and the merge compare with."""
import numpy as np

import oracle
from oracle import DT_BF16, DT_F16, FMT_BF16, FMT_FP16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_WHT256

# relative error of one rounding to the type: half a step
HALF_STEP = {DT_F16: 2.0 ** -11, DT_BF16: 2.0 ** -8}
# half the distance of its smallest numbers
HALF_TINY = {DT_F16: 2.0 ** -25, DT_BF16: 2.0 ** -134}


def _hadamard():
    h = np.ones((1, 1))
    while h.shape[0] < 256:
        h = np.block([[h, h], [h, -h]])
    return h / 16.0


def stored_rows(rows, fmt, head_dim):
    """Bytes [..., row bytes] -> the values as they are stored (in the rotated domain where the slab is rotated), float64."""
    rows = np.ascontiguousarray(rows)
    lead = rows.shape[:-1]
    if fmt == FMT_FP16:
        return rows.view(np.float16).astype(np.float64)
    if fmt == FMT_BF16:
        return oracle.bits_to_f32(rows.view(np.uint16), DT_BF16).astype(np.float64)
    if fmt == FMT_TQ4:
        blocks = rows.reshape(*lead, head_dim // 128, 66)
        d = np.ascontiguousarray(blocks[..., :2]).view(np.float16).astype(np.float64)
        table = oracle.centroids().astype(np.float64)
        codes = np.stack([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], axis=-1).reshape(*lead, head_dim // 128, 128)
        return (d * table[codes]).reshape(*lead, head_dim)
    if fmt == FMT_FP8:
        table = np.array([oracle.e4m3_to_f32(c) for c in range(256)], dtype=np.float64)
        d = np.ascontiguousarray(rows[..., 256:264]).view(np.float32).astype(np.float64)
        return table[rows[..., :256]] * np.repeat(d, 128, axis=-1)
    assert fmt == FMT_Q8_0
    blocks = rows.reshape(*lead, head_dim // 64, 68)
    d = np.ascontiguousarray(blocks[..., :4]).view(np.float32).astype(np.float64)
    return (np.ascontiguousarray(blocks[..., 4:]).view(np.int8).astype(np.float64) * d).reshape(*lead, head_dim)


def decoded_rows(rows, fmt, transform, head_dim):
    """Bytes [..., row bytes] -> the values they stand for, float64."""
    x = stored_rows(rows, fmt, head_dim)
    if transform == XF_WHT256 and head_dim == 256 and fmt in (FMT_TQ4, FMT_FP8, FMT_Q8_0):
        x = (x @ _hadamard()) * oracle.signs().astype(np.float64)
    return x


def slab_rows(slab, pool, slots):
    """Bytes of the rows of `slots` of a HostPool's slab: [slots, kv heads, row bytes]."""
    slots = np.asarray(slots)
    page, at = slots // pool.block_size, slots % pool.block_size
    base = page * pool.page + at * pool.tok
    where = base[:, None, None] + np.arange(pool.kv_heads)[None, :, None] * pool.head + np.arange(pool.tok)[None, None, :]
    return slab[where]
