"""Performance cases of linear attention, the verification of drafted tokens and the copying of cache pages.

A case is a dict of plain values; its "kind" says which operator one pass runs:

  linear   attention whose keys and values are summed up in one state per value head, which fades by a factor for each head
           (decay "head") or each head and token (decay "token"): a prompt's tokens, one token of every request, or a few drafted
           ones of which the state keeps the first (kept true)
  drafts   drafted tokens accepted or refused by the target's probabilities, and one more token drawn
  pages    pages of a paged cache copied in all layers, whole ones or their first rows (partly true)

Lengths are drawn uniformly from [q_min, q_max] by a generator seeded with "lens": they belong to the case, and so do the numbers
of kept tokens and rows.  The values and the page order come from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SCRATCH_BYTES = 64 << 20  # an engine's workspace
CHUNK = 64  # tokens that the plain form takes at once


def row_bytes(fmt, head_dim):
    return {"fp16": 2 * head_dim, "bf16": 2 * head_dim, "tq4": 66 * head_dim // 128, "q8_0": 68 * head_dim // 64,
            "fp8": 264 * head_dim // 256}[fmt]


def _linear(act, requests, q_min, q_max, *, k_heads=16, v_heads=32, k_dim=128, v_dim=128, decay="token", resumed=True, kept=False,
            lens=1):
    return {"kind": "linear", "act": act, "requests": requests, "q_min": q_min, "q_max": q_max, "k_heads": k_heads,
            "v_heads": v_heads, "k_dim": k_dim, "v_dim": v_dim, "decay": decay, "resumed": resumed, "kept": kept, "lens": lens}


def _drafts(requests, q_min, q_max, vocab, *, certain=False, lens=1):
    return {"kind": "drafts", "requests": requests, "q_min": q_min, "q_max": q_max, "vocab": vocab, "certain": certain, "lens": lens}


def _pages(fmt, layers, pairs, *, block=64, kv_heads=2, head_dim=256, partly=False, lens=1):
    return {"kind": "pages", "fmt": fmt, "layers": layers, "pairs": pairs, "block": block, "kv_heads": kv_heads,
            "head_dim": head_dim, "partly": partly, "lens": lens}


def listed():
    named = [
        # one long prompt from its beginning
        ("prompt_bf16_1x8192", _linear("bf16", 1, 8192, 8192, resumed=False)),
        # a prefill step in full swing: chunks of several prompts
        ("prompt_bf16_8x4096", _linear("bf16", 8, 4096, 4096)),
        # prompts of odd lengths, decays that belong to the heads
        ("prompt_fp16_6x100_1900_heads", _linear("fp16", 6, 100, 1900, k_heads=16, v_heads=16, decay="head")),
        # one user's short question
        ("prompt_bf16_1x333", _linear("bf16", 1, 333, 333, k_heads=8, v_heads=16)),
        # one user, one token: nothing but latency
        ("step_bf16_1x1", _linear("bf16", 1, 1, 1)),
        # a full decode batch
        ("step_fp16_64x1", _linear("fp16", 64, 1, 1)),
        # one token and four drafted ones, of which the state keeps those that were accepted
        ("step_bf16_16x5_kept", _linear("bf16", 16, 5, 5, kept=True)),
        # one user's three drafted tokens, vocabulary of ordinary size
        ("drafts_1x4_128000", _drafts(1, 4, 4, 128000)),
        # a verify batch with any number of drafts, odd vocabulary
        ("drafts_32x1_8_150001", _drafts(32, 1, 8, 150001)),
        # drafts that were each the draft model's most likely token, taken as certain
        ("drafts_16x5_65536_certain", _drafts(16, 5, 5, 65536, certain=True)),
        # requests that fork behind a prompt: the last page of each, its first rows, in the layers of a model
        ("pages_tq4_40_layers_24_partly", _pages("tq4", 40, 24, partly=True)),
        # a pool that is packed together
        ("pages_bf16_24_layers_128", _pages("bf16", 24, 128)),
    ]
    return [dict(c, name=n) for n, c in named]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges the listed ones stand for; never more bytes or operations than the largest of those."""
    kind = rng.choice(["prompt"] * 4 + ["step"] * 3 + ["drafts"] * 2 + ["pages"] * 2)
    lens = rng.randrange(1 << 20)
    while True:
        if kind == "drafts":
            q_max = rng.randint(1, 12)
            return _drafts(_log_int(rng, 1, 64), rng.randint(1, q_max), q_max, _log_int(rng, 1000, 260000),
                           certain=rng.random() < 0.3, lens=lens)
        if kind == "pages":
            fmt = rng.choice(["tq4", "tq4", "fp8", "q8_0", "fp16", "bf16"])
            c = _pages(fmt, _log_int(rng, 1, 64), _log_int(rng, 1, 400), block=rng.choice([16, 64, 128]),
                       kv_heads=rng.choice([1, 2, 4]), head_dim=rng.choice([256, 128]) if fmt in TYPES else 256,
                       partly=rng.random() < 0.5, lens=lens)
            if work(dict(c, partly=False))["bytes"] > 8.0e8:
                continue
            return c
        shape = {"decay": rng.choice(["token", "token", "head"]), "resumed": rng.random() < 0.7, "lens": lens}
        shape["k_heads"], shape["v_heads"] = rng.choice([(16, 32), (16, 32), (16, 16), (8, 16), (4, 12), (2, 16)])
        shape["k_dim"], shape["v_dim"] = rng.choice([(128, 128)] * 4 + [(64, 64), (64, 128), (128, 64)])
        act = rng.choice(["fp16", "bf16", "bf16"])
        if kind == "step":
            q_max = rng.choice([1, 1, 1, 2, 3, 5, 8])
            return _linear(act, _log_int(rng, 1, 128), rng.randint(1, q_max), q_max, kept=q_max > 1 and rng.random() < 0.7, **shape)
        q_max = _log_int(rng, 17, 8192)
        c = _linear(act, _log_int(rng, 1, 16), max(1, int(q_max * rng.uniform(0.05, 1.0))), q_max, kept=rng.random() < 0.1, **shape)
        if c["requests"] * q_max * c["v_heads"] > 8 * 4096 * 32:
            continue
        return c


def _lengths(case):
    """Per request (or pair of pages): tokens of the step, and how many of them (of a page's rows) are kept."""
    rng = random.Random(case["lens"])
    if case["kind"] == "pages":
        return [], [rng.randint(1, case["block"]) if case["partly"] else case["block"] for _ in range(case["pairs"])]
    news = [rng.randint(case["q_min"], case["q_max"]) for _ in range(case["requests"])]
    return news, [rng.randint(1, n) if case.get("kept") else n for n in news]


def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _starts(news):
    first = [0]
    for q in news:
        first.append(first[-1] + q)
    return torch.tensor(first, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"case": dict(case)}
    news, kept = _lengths(case)
    if case["kind"] == "pages":
        pairs, n = case["pairs"], case["pairs"] * 2 + 5
        order = torch.randperm(n, generator=gen, device=DEV).to(torch.int32)
        st["src"], st["dst"] = order[:pairs].contiguous(), order[pairs:2 * pairs].contiguous()
        st["rows"] = torch.tensor(kept, dtype=torch.int32, device=DEV) if case["partly"] else None
        # [layer, K or V, page, kv head, row, four bytes]
        words = row_bytes(case["fmt"], case["head_dim"]) // 4
        st["slabs"] = torch.randint(-(1 << 31), (1 << 31) - 1, (case["layers"], 2, n, case["kv_heads"], case["block"], words),
                                    generator=gen, device=DEV, dtype=torch.int32)
        return st
    st["qsl"], n = _starts(news), sum(news)
    st["req"] = torch.repeat_interleave(torch.arange(len(news), device=DEV), torch.tensor(news, device=DEV))
    st["place"] = torch.arange(n, device=DEV) - st["qsl"][st["req"]]
    st["scratch"] = torch.empty(SCRATCH_BYTES, dtype=torch.uint8, device=DEV)
    if case["kind"] == "drafts":
        vocab = case["vocab"]
        logits = _normal(gen, (n, vocab)) * 3.0
        st["target"] = torch.softmax(logits, -1)
        draft = torch.softmax(logits + _normal(gen, (n, vocab)), -1)
        if case["certain"]:
            drawn = draft.argmax(-1)
        else:
            drawn = (draft.log() - torch.log(-torch.log(torch.rand((n, vocab), generator=gen, device=DEV)))).argmax(-1)
        # the token fed behind row i is the one drafted from row i
        st["tokens"] = torch.randint(0, vocab, (n + 1,), generator=gen, device=DEV, dtype=torch.int32)
        st["tokens"][1:] = torch.where(torch.arange(1, n + 1, device=DEV) == st["qsl"][1:].long()[st["req"]], st["tokens"][1:],
                                       drawn.to(torch.int32))
        st["tokens"] = st["tokens"][:n].contiguous()
        st["draft"] = None if case["certain"] else draft
        st["u"] = torch.rand(n, generator=gen, device=DEV)
        st["u_draw"] = torch.rand(len(news), generator=gen, device=DEV)
        st["out"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        st["counts"] = torch.zeros(len(news), dtype=torch.int32, device=DEV)
        return st
    dtype, hk, hv = TYPES[case["act"]], case["k_heads"], case["v_heads"]
    unit = lambda x: x / x.square().sum(-1, keepdim=True).sqrt()  # noqa: E731  queries and keys arrive at length one
    st["q"] = unit(_normal(gen, (n, hk, case["k_dim"]))).to(dtype)
    st["k"] = unit(_normal(gen, (n, hk, case["k_dim"]))).to(dtype)
    st["v"] = _normal(gen, (n, hv, case["v_dim"]), dtype)
    heads = torch.arange(1, hv + 1, device=DEV)
    if case["decay"] == "head":
        st["g"] = -(2.0 ** (-8.0 * heads.float() / hv))[None].contiguous()
    else:  # a head's rate times a token's step
        step = torch.nn.functional.softplus(_normal(gen, (n, hv)) + torch.linspace(-6.0, -1.0, hv, device=DEV))
        st["g"] = -step * torch.linspace(1.0, 16.0, hv, device=DEV)[torch.randperm(hv, generator=gen, device=DEV)]
    r = len(news)
    slots = torch.randperm(2 * r, generator=gen, device=DEV).to(torch.int32)
    st["state_in"] = slots[:r].contiguous() if case["resumed"] else torch.full((r,), -1, dtype=torch.int32, device=DEV)
    st["state_out"] = slots[r:].contiguous()
    st["kept"] = torch.tensor(kept, dtype=torch.int32, device=DEV) if case["kept"] else None
    st["states"] = _normal(gen, (2 * r, hv, case["k_dim"], case["v_dim"])) * 0.3
    st["out"] = torch.zeros((n, hv, case["v_dim"]), dtype=dtype, device=DEV)
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------------


def _pages_plain(st):
    slabs, src, dst = st["slabs"], st["src"].long(), st["dst"].long()
    rows = slabs[:, :, src]
    if st["rows"] is not None:
        mine = torch.arange(st["case"]["block"], device=DEV) < st["rows"][:, None]
        rows = torch.where(mine[:, None, :, None], rows, slabs[:, :, dst])
    slabs[:, :, dst] = rows
    return [slabs]


def _drafts_plain(st):
    c = st["case"]
    n, first, counts = c["requests"], st["qsl"][:-1].long(), (st["qsl"][1:] - st["qsl"][:-1]).long()
    judged = torch.arange(c["q_max"] - 1, device=DEV)
    row = (first[:, None] + judged).clamp(max=st["out"].shape[0] - 1)  # [request, draft]
    token = st["tokens"][(row + 1).clamp(max=st["out"].shape[0] - 1)].long()
    p = st["target"][row, token].double()
    q = torch.ones_like(p) if st["draft"] is None else st["draft"][row, token].double()
    good = (st["u"][row].double() * q < p) & (judged < counts[:, None] - 1)
    accepted = torch.cumprod(good.long(), 1).sum(1)
    at = first + accepted
    refused = accepted < counts - 1
    p = st["target"][at].double()
    token_at = st["tokens"][(at + 1).clamp(max=st["out"].shape[0] - 1)].long()
    vocab = torch.arange(c["vocab"], device=DEV)
    if st["draft"] is None:
        rest = torch.where(vocab == token_at[:, None], torch.zeros_like(p), p)
    else:
        rest = (p - st["draft"][at].double()).clamp(min=0)
    w = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, p)
    running = torch.cumsum(w, 1)
    drawn = (running <= st["u_draw"].double()[:, None] * running[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
    follow = st["tokens"][(torch.arange(st["out"].shape[0], device=DEV) + 1).clamp(max=st["out"].shape[0] - 1)]
    mine = accepted[st["req"]]
    out = torch.where(st["place"] < mine, follow, torch.where(st["place"] == mine, drawn[st["req"]].to(torch.int32),
                                                              torch.full_like(follow, -1)))
    return [out, (accepted + 1).to(torch.int32).reshape(n)]


def _linear_plain(st):
    """All requests at once, padded to the longest, in chunks; [request, chunk, value head, token of the chunk, channel]."""
    c = st["case"]
    n, hk, hv, dk, dv = c["requests"], c["k_heads"], c["v_heads"], c["k_dim"], c["v_dim"]
    size = min(CHUNK, c["q_max"])
    chunks = (c["q_max"] + size - 1) // size
    req, place = st["req"], st["place"]

    def padded(x, heads, width):
        y = torch.zeros((n, chunks * size, heads, width), device=DEV)
        y[req, place] = x.float()
        y = y.reshape(n, chunks, size, heads, width).transpose(2, 3)
        return y.repeat_interleave(hv // heads, 2)

    q, k, v = padded(st["q"], hk, dk), padded(st["k"], hk, dk), padded(st["v"], hv, dv)
    g = torch.zeros((n, chunks * size, hv), dtype=torch.float64, device=DEV)
    g[req, place] = (st["g"] if c["decay"] == "token" else st["g"].expand(place.shape[0], hv)).double()
    total = torch.cumsum(g, 1)  # up to and with the token
    before = torch.zeros((n, 1, hv), dtype=torch.float64, device=DEV)
    upto = torch.cat([before, total[:, size - 1::size]], 1)  # at the borders of the chunks
    inside = total.reshape(n, chunks, size, hv).transpose(2, 3)
    start = torch.zeros((n, hv, dk, dv), device=DEV)
    if c["resumed"]:
        start = st["states"][st["state_in"].long()]
    # the chunks' own sums, and the states that they begin with
    to_end = torch.exp((upto[:, 1:, :, None] - inside)).float()
    sums = torch.matmul((k * to_end[..., None]).transpose(-1, -2).contiguous(), v)
    gap = (upto[:, :-1, None] - upto[:, None, 1:]).permute(0, 3, 1, 2)  # [request, head, chunk, chunk before it]
    earlier = torch.arange(chunks, device=DEV)[:, None] > torch.arange(chunks, device=DEV)
    weight = torch.exp(torch.where(earlier, gap, torch.full_like(gap, -math.inf))).float()
    begins = torch.matmul(weight, sums.transpose(1, 2).reshape(n, hv, chunks, dk * dv)).reshape(n, hv, chunks, dk, dv)
    begins = begins + torch.exp(upto[:, :-1]).float().transpose(1, 2)[..., None, None] * start[:, :, None]
    # what a chunk's tokens see of each other, and of the state
    gap = inside[..., :, None] - inside[..., None, :]
    seen = torch.arange(size, device=DEV)[:, None] >= torch.arange(size, device=DEV)
    weight = torch.exp(torch.where(seen, gap, torch.full_like(gap, -math.inf))).float()
    out = torch.matmul(torch.matmul(q, k.transpose(-1, -2).contiguous()) * weight, v)
    from_start = torch.exp(inside - upto[:, :-1, :, None]).float()
    out = out + torch.matmul(q * from_start[..., None], begins.transpose(1, 2))
    out = (out * dk ** -0.5).transpose(2, 3).reshape(n, chunks * size, hv, dv)[req, place].to(TYPES[c["act"]])
    # the state behind the kept tokens
    kept = st["kept"].long() if st["kept"] is not None else (st["qsl"][1:] - st["qsl"][:-1]).long()
    last = torch.gather(total, 1, (kept - 1)[:, None, None].expand(n, 1, hv))
    gap = torch.where((torch.arange(chunks * size, device=DEV) < kept[:, None])[..., None], last - total,
                      torch.full_like(total, -math.inf))
    weight = torch.exp(gap).float().reshape(n, chunks, size, hv).transpose(2, 3)[..., None]
    flat = lambda x: x.transpose(1, 2).reshape(n, hv, chunks * size, -1)  # noqa: E731
    end = torch.matmul(flat(k * weight).transpose(-1, -2).contiguous(), flat(v))
    st["states"][st["state_out"].long()] = end + torch.exp(last[:, 0]).float()[..., None, None] * start
    return [out, st["states"]]


# ---- the framework's calls ------------------------------------------------------------------------------------------------


def _calls(st):
    """The descriptors of a state's call and the call, as an engine keeps them: (function, arguments)."""
    import ctypes as C

    from warp34_amd import ffi

    lib, c = ffi.load(), st["case"]
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    scratch = st.get("scratch")
    ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, at(scratch) or 0, 0 if scratch is None else scratch.numel(), 0)
    if c["kind"] == "pages":
        fmt = {"fp16": ffi.WARP34_KV_FORMAT_FP16, "bf16": ffi.WARP34_KV_FORMAT_BF16, "tq4": ffi.WARP34_KV_FORMAT_TQ4,
               "q8_0": ffi.WARP34_KV_FORMAT_Q8_0, "fp8": ffi.WARP34_KV_FORMAT_FP8_E4M3}[c["fmt"]]
        xf = ffi.WARP34_KV_TRANSFORM_RADEMACHER_WHT256 if c["fmt"] == "tq4" else ffi.WARP34_KV_TRANSFORM_IDENTITY
        tok = row_bytes(c["fmt"], c["head_dim"])
        strides = (c["kv_heads"] * c["block"] * tok, c["block"] * tok, tok)
        layers = [ffi.Warp34KvLayerLayout(s[0].data_ptr(), s[1].data_ptr(), *strides, *strides, 0, i, c["kv_heads"],
                                          c["head_dim"], c["block"], fmt, fmt, xf, xf, 0) for i, s in enumerate(st["slabs"])]
        return lib.warp34_kv_cache_copy_pages, (C.pointer(ex), (ffi.Warp34KvLayerLayout * len(layers))(*layers), len(layers),
                                                at(st["src"]), at(st["dst"]), at(st["rows"]), c["pairs"])
    news = _lengths(c)[0]
    if c["kind"] == "drafts":
        batch = ffi.Warp34DraftBatch(at(st["qsl"]), at(st["tokens"]), None, c["vocab"], c["vocab"], c["requests"], sum(news),
                                     max(news), c["vocab"])
        return lib.warp34_verify_drafts, (C.pointer(ex), C.pointer(batch), at(st["target"]), at(st["draft"]), at(st["u"]),
                                          at(st["u_draw"]), at(st["out"]), at(st["counts"]))
    k_row, v_row = c["k_heads"] * c["k_dim"], c["v_heads"] * c["v_dim"]
    layout = ffi.Warp34LinearStateLayout(at(st["states"]), 4 * c["v_heads"] * c["k_dim"] * c["v_dim"], c["k_heads"], c["v_heads"],
                                         c["k_dim"], c["v_dim"])
    batch = ffi.Warp34LinearBatch(at(st["qsl"]), at(st["state_in"]), None, at(st["state_out"]), at(st["kept"]), None, c["requests"],
                                  sum(news), max(news), c["k_dim"] ** -0.5, k_row, k_row, v_row, v_row,
                                  c["v_heads"] if c["decay"] == "token" else 0, 0)
    return lib.warp34_linear_attention_f16 if c["act"] == "fp16" else lib.warp34_linear_attention_bf16, (
        C.pointer(ex), C.pointer(layout), C.pointer(batch), at(st["q"]), at(st["k"]), at(st["v"]), at(st["g"]), at(st["out"]))


def run(state):
    kind = state["case"]["kind"]
    if own:
        if "call" not in state:
            state["call"] = _calls(state)
        call, args = state["call"]
        rc = call(*args)
        if rc:
            raise RuntimeError("%s: %d" % (call.__name__, rc))
        return {"pages": lambda: [state["slabs"]], "drafts": lambda: [state["out"], state["counts"]],
                "linear": lambda: [state["out"], state["states"]]}[kind]()
    return {"pages": _pages_plain, "drafts": _drafts_plain, "linear": _linear_plain}[kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    news, kept = _lengths(case)
    n = sum(news)
    if case["kind"] == "pages":
        return {"bytes": 4.0 * case["layers"] * case["kv_heads"] * sum(kept) * row_bytes(case["fmt"], case["head_dim"]), "flops": 0.0}
    if case["kind"] == "drafts":  # one row of the target's probabilities a request, and one of the draft's
        rows = 1.0 if case["certain"] else 2.0
        return {"bytes": 4.0 * rows * case["requests"] * case["vocab"] + 20.0 * n, "flops": 2.0 * case["requests"] * case["vocab"]}
    hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    state = 4.0 * case["requests"] * hv * dk * dv * (2 if case["resumed"] else 1)
    decay = 4.0 * hv * (n if case["decay"] == "token" else 1)
    return {"bytes": n * 4.0 * (hk * dk + hv * dv) + decay + state, "flops": 4.0 * n * hv * dk * dv}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    news, kept = _lengths(case)
    first = st["qsl"].tolist() if "qsl" in st else None
    if case["kind"] == "pages":
        was = st["slabs"].clone()
        for s, d, rows in zip(st["src"].tolist(), st["dst"].tolist(), kept):
            st["slabs"][:, :, d, :, :rows] = was[:, :, s, :, :rows]
        return [st["slabs"]]
    if case["kind"] == "drafts":
        out, counts = torch.full_like(st["out"], -1), torch.zeros_like(st["counts"])
        for r, n in enumerate(news):
            i, lo = 0, first[r]
            while i < n - 1:
                x = int(st["tokens"][lo + i + 1])
                p = float(st["target"][lo + i, x])
                if not float(st["u"][lo + i]) * (1.0 if case["certain"] else float(st["draft"][lo + i, x])) < p:
                    break
                out[lo + i] = x
                i += 1
            w = st["target"][lo + i].double()
            if i < n - 1:
                rest = w.clone()
                if case["certain"]:
                    rest[int(st["tokens"][lo + i + 1])] = 0
                else:
                    rest = torch.relu(rest - st["draft"][lo + i].double())
                w = rest if float(rest.sum()) > 0 else w
            running = torch.cumsum(w, 0)
            above = (running > float(st["u_draw"][r]) * running[-1]).nonzero()
            out[lo + i] = int(above[0]) if len(above) else int(w.nonzero()[-1])
            counts[r] = i + 1
        return [out, counts]
    hk, hv = case["k_heads"], case["v_heads"]
    wide = lambda x: x.double().repeat_interleave(hv // x.shape[1], 1)  # noqa: E731
    q, k, v = wide(st["q"]), wide(st["k"]), wide(st["v"])
    g = st["g"].double().expand(q.shape[0], hv)
    state = torch.zeros(st["states"][:len(news)].shape, dtype=torch.float64, device=DEV)
    if case["resumed"]:
        state += st["states"][st["state_in"].long()]
    out = torch.zeros(v.shape, dtype=torch.float64, device=DEV)
    states = st["states"].double()
    n, keep = torch.tensor(news, device=DEV), torch.tensor(kept, device=DEV)
    for t in range(max(news)):
        row = (st["qsl"][:-1].long() + t).clamp(max=q.shape[0] - 1)
        state = state * torch.exp(g[row])[..., None, None] + k[row][..., :, None] * v[row][..., None, :]
        o = torch.matmul(q[row][..., None, :], state)[..., 0, :] / math.sqrt(case["k_dim"])
        live, done = n > t, keep == t + 1
        out[row[live]] = o[live]
        states[st["state_out"].long()[done]] = state[done]
    return [out, states]
