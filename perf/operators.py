"""Performance cases of the scored attention, the cache read and the merge of partial attentions.

A case is a dict of plain values; its "kind" says which operator one pass runs:

  attention  paged attention whose scores are capped by a tanh (cap > 0), fall with the distance by a slope for each head
             (slopes), and whose rows see the keys of a sliding window (window > 0), of their own document (docs > 0: mean
             document length) or a prefix that is visible in both directions (prefix > 0: its largest length); with the
             logarithms of the rows' sums where lse is true
  read       rows of a paged cache, decoded, by their slots
  merge      attention results over disjoint key sets joined by the logarithms of their sums

Context lengths are drawn uniformly from [ctx_min, ctx_max] and the numbers of new tokens from [q_min, q_max] by a generator
seeded with "lens", and so are document borders and prefix lengths: they belong to the case.  The values and the page order
come from the seed.  Pages are made here, by the formats' definitions, from rows with the values that real caches show.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
NO_KEY = -1.0e30  # a score that no key has
# TQ4: the centroids of a code, and the signs of the rotated domain (bit i of word i / 32: element i is negated)
CENTROIDS = (-1.694104124e-1, -1.285881878e-1, -1.006979993e-1, -7.824930800e-2, -5.873210384e-2, -4.094919437e-2,
             -2.420087619e-2, -8.008373692e-3, 8.008373692e-3, 2.420087619e-2, 4.094919437e-2, 5.873210384e-2,
             7.824930800e-2, 1.006979993e-1, 1.285881878e-1, 1.694104124e-1)
SIGN_WORDS = (0x29e1d357, 0x48974752, 0xeebc0de4, 0xf1297e2a, 0xba639274, 0xe2eb25d0, 0xfde0ee14, 0x36b5bda1)
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SCRATCH_BYTES = 64 << 20  # an engine's workspace


def row_bytes(fmt, head_dim):
    return {"fp16": 2 * head_dim, "bf16": 2 * head_dim, "tq4": 66 * head_dim // 128, "q8_0": 68 * head_dim // 64,
            "fp8": 264 * head_dim // 256}[fmt]


def _attention(fmt, act, requests, ctx_min, ctx_max, q_min, q_max, *, block=64, q_heads=16, kv_heads=2, head_dim=256, cap=0.0,
               slopes=False, window=0, docs=0, prefix=0, lse=True, lens=1):
    return {"kind": "attention", "fmt": fmt, "act": act, "requests": requests, "ctx_min": ctx_min, "ctx_max": ctx_max,
            "q_min": q_min, "q_max": q_max, "block": block, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "cap": cap, "slopes": slopes, "window": window, "docs": docs, "prefix": prefix, "lse": lse, "lens": lens}


def _read(fmt, act, rows, *, block=64, kv_heads=2, head_dim=256):
    return {"kind": "read", "fmt": fmt, "act": act, "rows": rows, "block": block, "kv_heads": kv_heads, "head_dim": head_dim}


def _merge(act, parts, rows, *, head_dim=256):
    return {"kind": "merge", "act": act, "parts": parts, "rows": rows, "head_dim": head_dim}


def listed():
    named = [
        # one user, a short chat, unquantised pages, capped scores: nothing but latency
        ("decode_fp16_1x700_cap", _attention("fp16", "fp16", 1, 700, 700, 1, 1, block=16, cap=50.0)),
        # one user at 128K context
        ("decode_tq4_1x131072_cap", _attention("tq4", "bf16", 1, 131072, 131072, 1, 1, cap=30.0)),
        # a full decode batch of users with contexts of any length, scores that fall with the distance
        ("decode_tq4_32x1k_64k_slopes", _attention("tq4", "fp16", 32, 1024, 65536, 1, 1, slopes=True)),
        # local layers of a decode batch: capped scores inside a window, head dimension 128
        ("decode_bf16_16x9k_window_cap", _attention("bf16", "bf16", 16, 1000, 9000, 1, 1, block=16, kv_heads=4, head_dim=128,
                                                    cap=50.0, window=4096)),
        # a few users, one token and three drafted ones verified, over 8-bit pages
        ("verify_q8_0_5x4_3k_21k_cap", _attention("q8_0", "fp16", 5, 3000, 21000, 4, 4, block=16, cap=50.0)),
        # chunked prefill in full swing, capped scores
        ("chunk_tq4_4x2048_16384_cap", _attention("tq4", "bf16", 4, 18432, 18432, 2048, 2048, cap=50.0, lse=False)),
        # documents packed into one row of tokens, as an embedding or scoring pass sends them
        ("packed_bf16_1x8192_documents", _attention("bf16", "bf16", 1, 8192, 8192, 8192, 8192, docs=700)),
        # prompts of odd lengths that open with images, which see each other both ways; slopes
        ("prefix_fp8_3x200_1900_slopes", _attention("fp8", "fp16", 3, 1900, 7000, 200, 1900, block=16, slopes=True, prefix=600)),
        # a long prefix read back to be handed on
        ("read_tq4_32768", _read("tq4", "bf16", 32768)),
        # some rows of a short request
        ("read_q8_0_333", _read("q8_0", "fp16", 333, block=16)),
        # a decode batch whose keys are spread over eight cards
        ("merge_bf16_8x512", _merge("bf16", 8, 512)),
        # a prefill chunk: shared prefix and private rest
        ("merge_fp16_2x131072", _merge("fp16", 2, 131072)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges the listed ones stand for; never more bytes or operations than the largest of those."""
    kind = rng.choice(["decode"] * 4 + ["chunk"] * 3 + ["read", "merge"])
    if kind == "read":
        fmt = rng.choice(["tq4", "tq4", "fp8", "q8_0", "fp16", "bf16"])
        hd = rng.choice([256, 128]) if fmt in TYPES else 256
        return _read(fmt, fmt if fmt in TYPES else rng.choice(["fp16", "bf16"]), _log_int(rng, 1, 60000),
                     block=rng.choice([16, 64, 128]), kv_heads=rng.choice([1, 2, 4]), head_dim=hd)
    if kind == "merge":
        parts = rng.randint(2, 16)
        return _merge(rng.choice(["fp16", "bf16"]), parts, _log_int(rng, 8, 262144 // parts), head_dim=rng.choice([128, 256]))
    while True:
        fmt = rng.choice(["tq4"] * 3 + ["q8_0", "fp8", "fp16", "bf16"])
        hd = rng.choice([256, 256, 128]) if fmt in TYPES else 256
        q_heads, kv_heads = rng.choice([(16, 2), (16, 2), (8, 1), (8, 2), (16, 4), (32, 4)])
        act = fmt if fmt in TYPES else rng.choice(["fp16", "bf16"])
        shape = {"block": rng.choice([16, 64, 64, 128]), "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": hd,
                 "lens": rng.randrange(1 << 20)}
        terms = {"cap": rng.choice([0.0, 30.0, 50.0]), "slopes": rng.random() < 0.3}
        if kind == "decode":
            ctx_max = _log_int(rng, 1, 131072)
            q = min(ctx_max, rng.choice([1, 1, 1, 2, 4, 7]))
            terms["window"] = rng.choice([0, 0, 1024, 4096])
            c = _attention(fmt, act, _log_int(rng, 1, 32), max(q, int(ctx_max * rng.uniform(0.02, 1.0))), ctx_max, q, q,
                           **shape, **terms)
        else:
            q_max = _log_int(rng, 20, 4096)
            part = rng.choice(["", "window", "docs", "prefix"])
            if part:
                terms[part] = _log_int(rng, 16, 4096)
            c = _attention(fmt, act, _log_int(rng, 1, 8), q_max, q_max + rng.choice([0, rng.randrange(16384)]),
                           max(1, int(q_max * rng.uniform(0.2, 1.0))), q_max, lse=fmt in TYPES, **shape, **terms)
        w = work(c)
        seqs, news = _lengths(c)[:2]
        padded = c["requests"] * max(seqs)
        if w["bytes"] > 5.0e8 or w["flops"] > 1.2e12:
            continue
        if padded * max(news) * q_heads > 2.4e9 or padded * kv_heads * hd > 1.1e9:  # what the plain form holds at once
            continue
        return c


def _lengths(case):
    """Per request: tokens after the step, new tokens, prefix length; per request the sorted starts of its documents."""
    rng = random.Random(case["lens"])
    seqs, news, prefixes, starts = [], [], [], []
    for _ in range(case["requests"]):
        s = rng.randint(case["ctx_min"], case["ctx_max"])
        seqs.append(s)
        news.append(min(rng.randint(case["q_min"], case["q_max"]), s))
        prefixes.append(rng.randint(1, min(s, case["prefix"])) if case["prefix"] else 0)
        borders = [0]
        while case["docs"] and borders[-1] < s:
            borders.append(borders[-1] + rng.randint(1, 2 * case["docs"]))
        starts.append([b for b in borders if b < s])
    return seqs, news, prefixes, starts


def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _hadamard(dtype):
    h = torch.ones((1, 1), dtype=dtype, device=DEV)
    while h.shape[0] < 256:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / 16.0


def _signs(dtype):
    return torch.tensor([-1.0 if SIGN_WORDS[i // 32] >> (i % 32) & 1 else 1.0 for i in range(256)], dtype=dtype, device=DEV)


def _encode(x, fmt):
    """Rows [..., head_dim] in 32 bits as the bytes [..., row_bytes] of a format."""
    lead, hd = x.shape[:-1], x.shape[-1]
    if fmt in TYPES:
        return x.to(TYPES[fmt]).contiguous().view(torch.uint8)
    if fmt == "tq4":
        y = ((x * _signs(x.dtype)) @ _hadamard(x.dtype)).reshape(*lead, 2, 128)
        d = y.square().sum((-2, -1), keepdim=True).sqrt().to(torch.float16).expand(*lead, 2, 1)
        table = torch.tensor(CENTROIDS, dtype=x.dtype, device=DEV)
        code = torch.bucketize(y / d.float(), (table[1:] + table[:-1]) / 2).to(torch.uint8)
        packed = code[..., 0::2] | code[..., 1::2] << 4
        return torch.cat([d.contiguous().view(torch.uint8), packed], -1).reshape(*lead, 132)
    if fmt == "fp8":
        y = x.reshape(*lead, 2, 128)
        d = y.abs().amax(-1, keepdim=True) / 448.0
        code = (y / d).to(torch.float8_e4m3fn).view(torch.uint8).reshape(*lead, 256)
        return torch.cat([code, d.reshape(*lead, 2).contiguous().view(torch.uint8)], -1)
    y = x.reshape(*lead, hd // 64, 64)
    d = y.abs().amax(-1, keepdim=True) / 127.0
    code = (y / d).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return torch.cat([d.contiguous().view(torch.uint8), code], -1).reshape(*lead, 68 * hd // 64)


def _decode(rows, fmt, hd):
    """Bytes [..., row_bytes] as values [..., head_dim] in 32 bits."""
    lead = rows.shape[:-1]
    if fmt in TYPES:
        return rows.view(TYPES[fmt]).float()
    if fmt == "tq4":
        r = rows.reshape(*lead, 2, 66)
        d = r[..., :2].contiguous().view(torch.float16).float()
        table = torch.tensor(CENTROIDS, device=DEV)
        pairs = torch.stack([table.repeat(16), table.repeat_interleave(16)], -1)  # of a byte: low code, high code
        y = (pairs[r[..., 2:].int()].flatten(-2) * d).reshape(*lead, 256)
        return (y @ _hadamard(torch.float32)) * _signs(torch.float32)
    if fmt == "fp8":
        d = rows[..., 256:].contiguous().view(torch.float32)[..., None]
        code = rows[..., :256].contiguous().view(torch.float8_e4m3fn).float()
        return (code.reshape(*lead, 2, 128) * d).reshape(*lead, 256)
    r = rows.reshape(*lead, hd // 64, 68)
    return (r[..., 4:].contiguous().view(torch.int8).float() * r[..., :4].contiguous().view(torch.float32)).reshape(*lead, hd)


def _pages(gen, case, pool):
    """One slab [pages, kv heads, block, row bytes]: rows N(0, 1) with three channels of every head twenty times as large."""
    kvh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
    slab = torch.empty((pool, kvh, bs, row_bytes(case["fmt"], hd)), dtype=torch.uint8, device=DEV)
    for part in slab.split(max(1, (1 << 27) // (kvh * bs * hd))):
        x = _normal(gen, (part.shape[0], kvh, bs, hd))
        x[..., [7, hd // 2 + 13, hd - 30]] *= 20.0
        part.copy_(_encode(x.to(TYPES[case["act"]]).float(), case["fmt"]))
    return slab


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"case": dict(case)}
    dtype = TYPES[case["act"]]
    if case["kind"] == "merge":
        n, rows, hd = case["parts"], case["rows"], case["head_dim"]
        st["parts"] = _normal(gen, (n, rows, hd), dtype)
        st["lse_parts"] = _normal(gen, (n, rows)) * 2.0 + 8.0
        nothing = torch.rand((n, rows), generator=gen, device=DEV) < 0.05  # a part without a visible key
        st["lse_parts"][nothing] = -math.inf
        st["parts"][nothing] = 0
        st["out"] = torch.zeros((rows, hd), dtype=dtype, device=DEV)
        st["lse"] = torch.zeros(rows, device=DEV)
        return st
    kvh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
    if case["kind"] == "read":
        rows = case["rows"]
        pool = (rows + bs - 1) // bs + 3
        st["k"], st["v"] = _pages(gen, case, pool), _pages(gen, case, pool)
        slots = torch.randperm(pool, generator=gen, device=DEV)[:, None] * bs + torch.arange(bs, device=DEV)
        st["slots"] = slots.reshape(-1)[:rows].to(torch.int32)
        st["slots"][torch.rand(rows, generator=gen, device=DEV) < 0.01] = -1  # padding of the list
        st["k_out"], st["v_out"] = (torch.zeros((rows, kvh, hd), dtype=dtype, device=DEV) for _ in range(2))
        return st
    seqs, news, prefixes, starts = _lengths(case)
    pages_per = [(s + bs - 1) // bs for s in seqs]
    pool, n = sum(pages_per) + 3, sum(news)
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    st["block_tables"] = torch.zeros((len(seqs), max(pages_per)), dtype=torch.int32, device=DEV)
    at = 0
    for r, p in enumerate(pages_per):
        st["block_tables"][r, :p] = order[at:at + p]
        at += p
    st["k"], st["v"] = _pages(gen, case, pool), _pages(gen, case, pool)
    first = [0]
    for q in news:
        first.append(first[-1] + q)
    st["qsl"] = torch.tensor(first, dtype=torch.int32, device=DEV)
    st["seq"] = torch.tensor(seqs, dtype=torch.int32, device=DEV)
    st["ctx"] = torch.tensor([s - q for s, q in zip(seqs, news)], dtype=torch.int32, device=DEV)
    # per token: its request, its place among the request's new tokens
    st["req"] = torch.repeat_interleave(torch.arange(len(news), device=DEV), torch.tensor(news, device=DEV))
    st["place"] = torch.arange(n, device=DEV) - st["qsl"][st["req"]]
    pos = st["ctx"][st["req"]] + st["place"]
    st["doc"] = st["pre"] = st["slopes"] = None
    if case["docs"]:
        st["doc"] = torch.empty(n, dtype=torch.int32, device=DEV)
        for r, s in enumerate(starts):
            b = torch.tensor(s, dtype=torch.int32, device=DEV)
            mine = slice(first[r], first[r + 1])
            st["doc"][mine] = b[torch.searchsorted(b, pos[mine].to(torch.int32), right=True) - 1]
    if case["prefix"]:
        st["pre"] = torch.tensor(prefixes, dtype=torch.int32, device=DEV)[st["req"]].contiguous()
    if case["slopes"]:
        heads = torch.arange(1, case["q_heads"] + 1, device=DEV)
        st["slopes"] = 2.0 ** (-8.0 * heads.float() / case["q_heads"])
    st["q"] = _normal(gen, (n, case["q_heads"], hd), dtype)
    st["out"] = torch.zeros_like(st["q"])
    st["lse"] = torch.zeros((n, case["q_heads"]), device=DEV) if case["lse"] else None
    st["scratch"] = torch.empty(SCRATCH_BYTES, dtype=torch.uint8, device=DEV)
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------------


def _merge_plain(st):
    lse_parts = st["lse_parts"]
    top = lse_parts.amax(0)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = (lse_parts - top).exp()
    total = w.sum(0)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    return (w[..., None] * st["parts"].float()).sum(0).to(st["out"].dtype), total.log() + top


def _read_plain(st):
    c, slots = st["case"], st["slots"].long()
    page, at = slots.clamp(min=0) // c["block"], slots.clamp(min=0) % c["block"]
    wanted = (slots >= 0)[:, None, None]
    return [torch.where(wanted, _decode(st[s][page, :, at], c["fmt"], c["head_dim"]).to(TYPES[c["act"]]),
                        torch.zeros_like(st[s + "_out"])) for s in ("k", "v")]


def _attention_plain(st):
    """All requests at once, padded to the longest; [request, kv head, query head of it x new token, key]."""
    c = st["case"]
    kvh, hd, qh = c["kv_heads"], c["head_dim"], c["q_heads"]
    n, keys, g = int(st["block_tables"].shape[0]), int(st["block_tables"].shape[1]) * c["block"], qh // kvh
    most = c["q_max"]
    values = [_decode(st[s][st["block_tables"].long()].transpose(2, 3).reshape(n, keys, kvh, -1).transpose(1, 2), c["fmt"], hd)
              for s in ("k", "v")]
    q = torch.zeros((n, most, qh, hd), device=DEV)
    q[st["req"], st["place"]] = st["q"].float()
    q = q.reshape(n, most, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * most, hd)
    x = torch.matmul(q, values[0].transpose(-1, -2).contiguous()) * hd ** -0.5
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    x = x.reshape(n, kvh, g, most, keys)
    key = torch.arange(keys, device=DEV)
    pos = st["ctx"][:, None] + torch.arange(most, device=DEV)  # [request, new token]
    if c["slopes"]:
        x = x - st["slopes"].reshape(kvh, g, 1, 1) * (pos[..., None] - key).abs()[:, None, None].float()
    low, high = torch.zeros_like(pos), torch.minimum(pos, st["seq"][:, None] - 1)
    if c["window"]:
        low = (pos - c["window"] + 1).clamp(min=0)
    if c["docs"]:
        low[st["req"], st["place"]] = torch.maximum(low[st["req"], st["place"]], st["doc"].long()).to(low.dtype)
    if c["prefix"]:
        reach = torch.zeros_like(high)
        reach[st["req"], st["place"]] = st["pre"].to(reach.dtype) - 1
        high = torch.minimum(torch.maximum(high, reach), st["seq"][:, None] - 1)
    seen = ((key >= low[..., None]) & (key <= high[..., None]))[:, None, None]
    x = torch.where(seen, x, torch.full((), NO_KEY, device=DEV))
    top = x.amax(-1, keepdim=True)
    x = (x - top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.reshape(n, kvh, g * most, keys), values[1]).reshape(n, kvh, g, most, hd) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, qh, hd)[st["req"], st["place"]].to(TYPES[c["act"]])
    if not c["lse"]:
        return [out]
    lse = (total.log() + top).squeeze(-1).permute(0, 3, 1, 2).reshape(n, most, qh)
    return [out, lse[st["req"], st["place"]]]


# ---- the framework's calls ------------------------------------------------------------------------------------------------


def _calls(st):
    """The descriptors of a state's call and the call, as an engine keeps them for a layer: (function, arguments)."""
    import ctypes as C

    from warp34_amd import ffi

    lib, c = ffi.load(), st["case"]
    act = "f16" if c["act"] == "fp16" else "bf16"
    if c["kind"] == "merge":
        ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, 0, 0, 0)
        return getattr(lib, "warp34_attention_merge_" + act), (
            C.pointer(ex), st["parts"].data_ptr(), st["lse_parts"].data_ptr(), c["parts"], c["rows"] * c["head_dim"], c["rows"],
            st["out"].data_ptr(), st["lse"].data_ptr(), c["rows"], c["head_dim"])
    fmt = {"fp16": ffi.WARP34_KV_FORMAT_FP16, "bf16": ffi.WARP34_KV_FORMAT_BF16, "tq4": ffi.WARP34_KV_FORMAT_TQ4,
           "q8_0": ffi.WARP34_KV_FORMAT_Q8_0, "fp8": ffi.WARP34_KV_FORMAT_FP8_E4M3}[c["fmt"]]
    xf = ffi.WARP34_KV_TRANSFORM_RADEMACHER_WHT256 if c["fmt"] == "tq4" else ffi.WARP34_KV_TRANSFORM_IDENTITY
    tok = row_bytes(c["fmt"], c["head_dim"])
    strides = (c["kv_heads"] * c["block"] * tok, c["block"] * tok, tok)
    layout = ffi.Warp34KvLayerLayout(st["k"].data_ptr(), st["v"].data_ptr(), *strides, *strides, 0, 0, c["kv_heads"],
                                     c["head_dim"], c["block"], fmt, fmt, xf, xf, 0)
    if c["kind"] == "read":
        ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, 0, 0, 0)
        stride = c["kv_heads"] * c["head_dim"]
        return getattr(lib, "warp34_kv_cache_read_" + act), (
            C.pointer(ex), C.pointer(layout), st["slots"].data_ptr(), c["rows"], st["k_out"].data_ptr(), st["v_out"].data_ptr(),
            stride, stride)
    ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, st["scratch"].data_ptr(), st["scratch"].numel(), 0)
    seqs, news = _lengths(c)[:2]
    batch = ffi.Warp34AttentionBatch(
        st["qsl"].data_ptr(), st["ctx"].data_ptr(), st["seq"].data_ptr(), st["block_tables"].data_ptr(), None, None, None,
        c["requests"], sum(news), st["block_tables"].shape[1], max(news), max(seqs), ffi.WARP34_ATTN_MASK_CAUSAL, c["window"],
        c["head_dim"] ** -0.5, 0)
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    scores = ffi.Warp34AttentionScores(at(st["slopes"]), at(st["doc"]), at(st["pre"]), at(st["lse"]), c["cap"], 0)
    return getattr(lib, "warp34_paged_attention_scored_" + act), (
        C.pointer(ex), C.pointer(layout), C.pointer(batch), C.pointer(scores), st["q"].data_ptr(), st["out"].data_ptr(),
        c["q_heads"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        call, args = state["call"]
        rc = call(*args)
        if rc:
            raise RuntimeError("%s: %d" % (call.__name__, rc))
        if kind == "read":
            return [state["k_out"], state["v_out"]]
        return [state["out"]] if state["lse"] is None else [state["out"], state["lse"]]
    return list({"attention": _attention_plain, "read": _read_plain, "merge": _merge_plain}[kind](state))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    hd = case["head_dim"]
    if case["kind"] == "merge":
        return {"bytes": (case["parts"] + 1.0) * case["rows"] * (2 * hd + 4), "flops": 2.0 * case["parts"] * case["rows"] * hd}
    row = row_bytes(case["fmt"], hd)
    if case["kind"] == "read":
        return {"bytes": case["rows"] * (2.0 * case["kv_heads"] * (row + 2 * hd) + 4), "flops": 0.0}
    seqs, news, prefixes, starts = _lengths(case)
    pairs = keys = 0.0
    for s, q, p, doc in zip(seqs, news, prefixes, starts):
        at, lowest, highest = 0, s, -1
        for pos in range(s - q, s):
            while at + 1 < len(doc) and doc[at + 1] <= pos:
                at += 1
            lo = max(pos - case["window"] + 1 if case["window"] else 0, doc[at] if case["docs"] else 0, 0)
            hi = min(s - 1, max(pos, p - 1))
            pairs += max(0, hi - lo + 1)
            lowest, highest = min(lowest, lo), max(highest, hi)
        keys += max(0, highest - lowest + 1)
    n = sum(news)
    return {"bytes": keys * 2.0 * case["kv_heads"] * row + n * case["q_heads"] * (4.0 * hd + (4 if case["lse"] else 0)),
            "flops": 4.0 * hd * case["q_heads"] * pairs}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------


def _rows64(rows, fmt):
    if fmt in TYPES:
        return rows.view(TYPES[fmt]).double()
    if fmt == "tq4":
        out = torch.empty((*rows.shape[:-1], 256), dtype=torch.float64, device=DEV)
        table = torch.tensor(CENTROIDS, dtype=torch.float32, device=DEV).double()
        for h in range(2):
            d = rows[..., 66 * h:66 * h + 2].contiguous().view(torch.float16).double()
            codes = rows[..., 66 * h + 2:66 * h + 66]
            out[..., 128 * h:128 * h + 128:2] = d * table[(codes & 15).int()]
            out[..., 128 * h + 1:128 * h + 128:2] = d * table[(codes >> 4).int()]
        step = 1
        while step < 256:  # the fast transform, its 1/16 at the end
            pairs = out.reshape(-1, 256 // (2 * step), 2, step)
            out = torch.stack([pairs[:, :, 0] + pairs[:, :, 1], pairs[:, :, 0] - pairs[:, :, 1]], 2).reshape(out.shape)
            step *= 2
        return out / 16.0 * _signs(torch.float64)
    if fmt == "fp8":
        d = rows[..., 256:264].contiguous().view(torch.float32).double()
        return rows[..., :256].contiguous().view(torch.float8_e4m3fn).double() * d.repeat_interleave(128, -1)
    blocks = [rows[..., 68 * b + 4:68 * b + 68].contiguous().view(torch.int8).double() *
              rows[..., 68 * b:68 * b + 4].contiguous().view(torch.float32).double() for b in range(rows.shape[-1] // 68)]
    return torch.cat(blocks, -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "merge":
        lse = torch.logsumexp(st["lse_parts"].double(), 0)
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEV)
        for part, l in zip(st["parts"], st["lse_parts"].double()):
            w = torch.where(l == -math.inf, torch.zeros_like(l), torch.exp(l - lse))
            out += w[:, None] * part.double()
        return [out, lse]
    bs, fmt = case["block"], case["fmt"]
    if case["kind"] == "read":
        outs = []
        for slab in (st["k"], st["v"]):
            out = torch.zeros((case["rows"], case["kv_heads"], case["head_dim"]), dtype=torch.float64, device=DEV)
            live = (st["slots"] >= 0).nonzero()[:, 0]
            slot = st["slots"][live].long()
            out[live] = _rows64(slab[torch.div(slot, bs, rounding_mode="floor"), :, slot % bs], fmt)
            outs.append(out)
        return outs
    seqs, news, prefixes, starts = _lengths(case)
    qh, kvh, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((sum(news), qh, hd), dtype=torch.float64, device=DEV)
    lse = torch.full((sum(news), qh), -math.inf, dtype=torch.float64, device=DEV)
    at = 0
    for r, (s, q) in enumerate(zip(seqs, news)):
        pages = st["block_tables"][r, :(s + bs - 1) // bs].long()
        i = torch.arange(s, device=DEV)[None, :]
        p = torch.arange(s - q, s, device=DEV)[:, None]
        seen = (i <= p) | (i < prefixes[r])
        if case["window"]:
            seen &= i > p - case["window"]
        if case["docs"]:
            b = torch.tensor(starts[r], device=DEV)
            seen &= torch.bucketize(i, b, right=True) >= torch.bucketize(p, b, right=True)
        for h in range(kvh):
            k, v = (_rows64(slab[pages, h].reshape(-1, slab.shape[-1])[:s], fmt) for slab in (st["k"], st["v"]))
            for a in range(h * (qh // kvh), (h + 1) * (qh // kvh)):
                x = (st["q"][at:at + q, a].double() @ k.t()) / math.sqrt(hd)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x - st["slopes"][a].double() * (p - i).abs()
                x = x.masked_fill(~seen, -math.inf)
                lse[at:at + q, a] = torch.logsumexp(x, 1)
                out[at:at + q, a] = torch.softmax(x, 1) @ v
        at += q
    return [out, lse] if case["lse"] else [out]
