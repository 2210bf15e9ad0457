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


def scored_attention(pool, bt, seqs, q, qsl, ctx, *, cap=0.0, slopes=None, window=0, noncausal=False, documents=None, prefixes=None,
                     scale=None, dt=DT_BF16, chunk=False):
    """Scored attention of q (float64 [tokens, heads, head_dim]) over a HostPool's pages, in float64.

    Returns (out, lse, out_bound, lse_bound).  The bounds are what 16-bit operands and 32-bit sums may do, worst case:
      score    the products are summed in 32 bits (2^-20 of sum |q_i k_i|), the terms are rounded a few times (2^-20 of their sizes);
               rotated queries and TQ4 keys have two fp16 parts, 2^-21 of them missing: of sum |q_i k_i| in the stored domain
      weight   two 16-bit parts: 2^-21 (fp16), 2^-16 (bf16); with an error d_k of a score, a weight p_k moves by p_k (d_k + sum p d)
      value    TQ4: 9.4e-5 of each stored element, which the rotation back adds up with 1 / 16
      small    fp16 weights have an absolute error of 2^-25 as well (half the distance of fp16's smallest numbers), relative to the
               row's largest, which is 1, and so its sum at least 1: 2^-25 of each |v_k| over that sum.  Where block scales ride on
               the weights it is 2^-25 of the largest code (in the units of the weights: TQ4 0.17, E4M3 448 / 256, Q8_0 127 / 128),
               which the rotation back adds up to 16 times that.  Values of their own below 2^-14: 2^-25 once more
      output   half a step.
    chunk: the call's chunk kernel, whose rotated queries and TQ4 keys are one fp16 part (2^-11 and 9.4e-5 of sum |q_i k_i|), whose
    weights are one 16-bit part (half a step) and whose quantised values are fp16(scale * code): 2^-11 of each stored element, or 2^-25
    below 2^-14, which the rotation back adds up with 1 / 16."""
    fmt, hd, kvh, bs = pool.fmt, pool.head_dim, pool.kv_heads, pool.block_size
    heads = q.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    rot_k = pool.transform == XF_WHT256 and fmt not in (FMT_FP16, FMT_BF16)
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    out_bound, lse_bound = np.zeros(q.shape), np.zeros(q.shape[:2])
    table = 9.4e-5 if fmt == FMT_TQ4 else 0.0
    weight = 2.0 ** -16 if fmt == FMT_BF16 else 2.0 ** -21
    operand = 2.0 ** -20
    rounded = 0.0  # of a stored value
    if chunk:
        operand = (2.0 ** -11 if rot_k else 0.0) + table
        weight = HALF_STEP[dt] if fmt in (FMT_FP16, FMT_BF16) else 2.0 ** -11
        rounded = 0.0 if fmt in (FMT_FP16, FMT_BF16) else 2.0 ** -11
    rotated_back = pool.v_transform == XF_WHT256 and fmt not in (FMT_FP16, FMT_BF16)
    ride = {FMT_TQ4: 0.17, FMT_FP8: 1.75, FMT_Q8_0: 1.0}.get(fmt, 0.0) * (16.0 if pool.v_transform == XF_WHT256 else 1.0)
    if chunk:
        ride = 0.0
    for r, s in enumerate(seqs):
        slots = oracle.slot_mapping(bt[r], 0, s, bs) if s else np.zeros(0, dtype=np.int64)
        kb, vb = slab_rows(pool.k, pool, slots), slab_rows(pool.v, pool, slots)
        ks = stored_rows(kb, fmt, hd)
        k, v = decoded_rows(kb, fmt, pool.transform, hd), decoded_rows(vb, fmt, pool.v_transform, hd)
        v_sum = np.abs(stored_rows(vb, fmt, hd)).sum(-1) / 16.0
        pos = np.arange(qsl[r + 1] - qsl[r]) + ctx[r]
        key = np.arange(s)
        for t in range(qsl[r], qsl[r + 1]):
            p_t = pos[t - qsl[r]]
            hi = s - 1 if noncausal else p_t
            if prefixes is not None:
                hi = max(hi, prefixes[t] - 1)
            hi = min(hi, s - 1)
            lo = max(0, p_t - window + 1) if window else 0
            if documents is not None:
                lo = max(lo, documents[t])
            if lo > hi:
                continue
            seen = slice(lo, hi + 1)
            for h in range(heads):
                g = h // (heads // kvh)
                qs = q[t, h]
                if rot_k:
                    qs = (qs * oracle.signs()) @ _hadamard()
                raw = (k[seen, g] @ q[t, h]) * scale
                size = (np.abs(ks[seen, g]) @ np.abs(qs)) * abs(scale)
                x = cap * np.tanh(raw / cap) if cap else raw
                far = slopes[h] * np.abs(p_t - key[seen]) if slopes is not None else np.zeros_like(x)
                d = size * (2.0 ** -20 + operand) + 2.0 ** -20 * (np.abs(x) + np.abs(far) + cap)
                x = x - far
                top = x.max()
                p = np.exp(x - top)
                total = p.sum()
                small = 2.0 ** -25 * (ride * p.size if ride else np.abs(v[seen, g]).sum(0)) / total + 2.0 ** -25 * (16.0 if rotated_back else 1.0)
                p = p / total
                lse[t, h] = top + np.log(total)
                out[t, h] = p @ v[seen, g]
                mean = p @ d
                moved = p * (d + mean + weight)
                lse_bound[t, h] = mean + 2.0 ** -20 * (np.abs(lse[t, h]) + np.abs(top) + 1)
                out_bound[t, h] = moved @ np.abs(v[seen, g]) + HALF_STEP[dt] * np.abs(out[t, h]) + HALF_TINY[dt]
                if fmt != FMT_BF16:
                    out_bound[t, h] += small
                if rotated_back:
                    out_bound[t, h] += (table + rounded) * (p @ v_sum[seen, g])
                else:
                    out_bound[t, h] += (table + rounded) * (p @ np.abs(v[seen, g]))
    return out, lse, out_bound, lse_bound
