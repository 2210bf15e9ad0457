"""warp34_kv_cache_copy_pages: every byte of the slabs against plain indexing."""
import ctypes as C

import numpy as np
import pytest

from oracle import FMT_BF16, FMT_FP16, FMT_FP8, FMT_Q8_0, FMT_TQ4, XF_IDENTITY, XF_WHT256

ROW = {FMT_FP16: lambda d: 2 * d, FMT_BF16: lambda d: 2 * d, FMT_TQ4: lambda d: 66 * d // 128, FMT_Q8_0: lambda d: 68 * d // 64, FMT_FP8: lambda d: 264 * d // 256}


class Pool:
    """Layers of slabs with any strides; formats: (K format, V format) of each layer."""

    def __init__(self, formats, pages, *, heads=2, hd=256, bs=16, token_pad=0, head_pad=0, page_pad=0, offset=0, token_major=False, seed=1):
        rng = np.random.default_rng(seed)
        self.formats, self.pages, self.heads, self.hd, self.bs, self.offset = formats, pages, heads, hd, bs, offset
        self.strides, self.bytes = [], []
        for kf, vf in formats:
            for f in (kf, vf):
                row = ROW[f](hd)
                if token_major:  # [page][row][head]
                    head, token = row + head_pad, heads * (row + head_pad) + token_pad
                    page = bs * token + page_pad
                else:
                    token = row + token_pad
                    head = bs * token + head_pad
                    page = heads * head + page_pad
                self.strides.append((page, head, token, row))
                self.bytes.append(rng.integers(0, 256, offset + pages * page + 64, dtype=np.uint8))

    def rows_of(self, slab):
        """Index of the bytes [page, head, row, byte]."""
        page, head, token, row = self.strides[slab]
        ix = lambda n, s: np.arange(n) * s  # noqa: E731
        return (self.offset + ix(self.pages, page)[:, None, None, None] + ix(self.heads, head)[None, :, None, None] + ix(self.bs, token)[None, None, :, None] +
                np.arange(row))

    def want(self, src, dst, rows):
        out = []
        for i, b in enumerate(self.bytes):
            at, new = self.rows_of(i), b.copy()
            for p, (s, d) in enumerate(zip(src, dst)):
                if s < 0 or d < 0 or s == d:
                    continue
                n = self.bs if rows is None else min(max(rows[p], 0), self.bs)
                new[at[d, :, :n]] = b[at[s, :, :n]]
            out.append(new)
        return out

    def check(self, src, dst, rows=None, stream=None):
        import torch

        import gpu_harness as G
        from warp34_amd import ffi

        dev = [torch.from_numpy(b.copy()).to(G.DEV) for b in self.bytes]
        layers = []
        for l, (kf, vf) in enumerate(self.formats):
            k, v = 2 * l, 2 * l + 1
            layers.append(ffi.Warp34KvLayerLayout(dev[k].data_ptr() + self.offset, dev[v].data_ptr() + self.offset, *self.strides[k][:3], *self.strides[v][:3],
                                                  0, l, self.heads, self.hd, self.bs, kf, vf, XF_IDENTITY, XF_WHT256, 0))
        i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=G.DEV)  # noqa: E731
        s, d, r = i32(src), i32(dst), i32(rows)
        torch.cuda.synchronize()
        ex = ffi.Warp34Exec(stream or torch.cuda.current_stream().cuda_stream, 0, 0, 0)
        rc = G.lib().warp34_kv_cache_copy_pages(C.byref(ex), (ffi.Warp34KvLayerLayout * len(layers))(*layers), len(layers), G.ptr(s), G.ptr(d), G.ptr(r), len(src))
        torch.cuda.synchronize()
        assert rc == 0
        for got, want in zip(dev, self.want(src, dst, rows)):
            assert (got.cpu().numpy() == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd", [(FMT_FP16, 256), (FMT_BF16, 128), (FMT_BF16, 8), (FMT_TQ4, 256), (FMT_TQ4, 128), (FMT_Q8_0, 256), (FMT_Q8_0, 64), (FMT_FP8, 256)])
@pytest.mark.parametrize("bs", [1, 16, 64])
def test_whole_pages_and_first_rows(fmt, hd, bs):
    p = Pool([(fmt, fmt)] * 3, 9, hd=hd, bs=bs, seed=bs + hd)
    p.check([7, 0, 3], [1, 8, 2])
    p.check([7, 0, 3, 5], [1, 8, 2, 4], rows=[1, bs, 0, bs // 2 + 1])


@pytest.mark.gpu
def test_pairs_that_copy_nothing():
    """Negative pages, a page onto itself, rows below zero and beyond the page; one source for two destinations."""
    p = Pool([(FMT_TQ4, FMT_TQ4)] * 2, 10, seed=3)
    p.check([-1, 4, 5, 6, 6, 8, 2], [0, -7, 5, 1, 3, 9, 7], rows=[16, 16, 16, 16, 5, -3, 1000])
    p.check([], [])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(token_pad=16), dict(token_pad=4), dict(token_pad=2), dict(head_pad=2), dict(page_pad=6), dict(page_pad=4), dict(offset=2),
                                dict(offset=4), dict(offset=16), dict(token_major=True), dict(token_major=True, head_pad=4, token_pad=12)])
@pytest.mark.parametrize("fmt", [FMT_BF16, FMT_TQ4, FMT_FP8])
def test_strides_and_alignments(fmt, kw):
    p = Pool([(fmt, fmt)] * 2, 6, seed=4, **kw)
    p.check([0, 5, 2], [3, 1, 4], rows=[16, 7, 3])


@pytest.mark.gpu
def test_models_of_many_layers_and_mixed_formats():
    """More layers than one launch takes; tail layers in another format, K and V each in its own."""
    p = Pool([(FMT_TQ4, FMT_TQ4)] * 45 + [(FMT_FP8, FMT_Q8_0)] * 9 + [(FMT_BF16, FMT_TQ4)] * 47, 5, heads=1, seed=5)
    p.check([0, 4], [2, 1], rows=[16, 9])


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_heads_and_many_pairs(heads):
    n = 60
    order = np.random.default_rng(6).permutation(2 * n)
    p = Pool([(FMT_TQ4, FMT_TQ4)], 2 * n, heads=heads, seed=7)
    p.check(order[:n].tolist(), order[n:].tolist(), rows=np.random.default_rng(8).integers(0, 18, n).tolist())


@pytest.mark.gpu
def test_more_pairs_than_a_launch_takes():
    """A whole pool's pairs, nearly all of them without work: of 96 slabs and 16 heads a launch takes 10 922."""
    n, src, dst = 25000, [3, 0, 7], [1, 5, 6]
    p = Pool([(FMT_TQ4, FMT_TQ4)] * 48, 8, heads=16, hd=128, bs=4, seed=10)
    at = [0, 10921, n - 1]
    pairs = [[-1] * n for _ in range(3)]
    for i, s, d in zip(at, src, dst):
        pairs[0][i], pairs[1][i], pairs[2][i] = s, d, 3
    p.check(pairs[0], pairs[1], rows=pairs[2])


@pytest.mark.gpu
def test_pages_far_into_a_large_slab():
    """Page offsets beyond 2^32 bytes."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    page, pages = 2 * 64 * 512, (1 << 32) // (2 * 64 * 512) + 9
    k = torch.zeros(page * pages, dtype=torch.uint8, device=G.DEV)
    v = torch.zeros(page * pages, dtype=torch.uint8, device=G.DEV)
    src, dst = [3, pages - 1], [pages - 3, pages - 2]
    for s in src:
        k[s * page:(s + 1) * page] = torch.randint(0, 256, (page,), dtype=torch.uint8, device=G.DEV)
        v[s * page:(s + 1) * page] = torch.randint(0, 256, (page,), dtype=torch.uint8, device=G.DEV)
    lay = ffi.Warp34KvLayerLayout(k.data_ptr(), v.data_ptr(), page, page // 2, 512, page, page // 2, 512, 0, 0, 2, 256, 64, FMT_BF16, FMT_BF16, 0, 0, 0)
    s, d = (torch.tensor(x, dtype=torch.int32, device=G.DEV) for x in (src, dst))
    ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, 0, 0, 0)
    assert G.lib().warp34_kv_cache_copy_pages(C.byref(ex), C.byref(lay), 1, G.ptr(s), G.ptr(d), None, 2) == 0
    torch.cuda.synchronize()
    for slab in (k, v):
        for a, b in zip(src, dst):
            assert torch.equal(slab[a * page:(a + 1) * page], slab[b * page:(b + 1) * page])
        assert not bool(slab[(pages - 4) * page:(pages - 3) * page].any()) and not bool(slab[:3 * page].any())


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    p = Pool([(FMT_TQ4, FMT_TQ4)] * 2, 6, seed=9)
    p.check([0, 5], [3, 1], stream=torch.cuda.Stream().cuda_stream)
    slab = torch.randint(0, 256, (4, 6, 2, 16, 132), dtype=torch.uint8, device=G.DEV)
    lays = (ffi.Warp34KvLayerLayout * 2)(*[ffi.Warp34KvLayerLayout(slab[2 * l].data_ptr(), slab[2 * l + 1].data_ptr(), 4224, 2112, 132, 4224, 2112, 132, 0, l, 2,
                                                                   256, 16, FMT_TQ4, FMT_TQ4, 1, 1, 0) for l in range(2)])
    src, dst = (torch.tensor(x, dtype=torch.int32, device=G.DEV) for x in ([0], [1]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, 0, 0, 0)
        assert G.lib().warp34_kv_cache_copy_pages(C.byref(ex), lays, 2, G.ptr(src), G.ptr(dst), None, 1) == 0
    del lays  # the descriptors belong to the caller again when the call returns
    for s, d in ((0, 1), (2, 3), (1, 5)):
        want = slab.clone()
        want[:, d] = want[:, s]
        src.fill_(s)
        dst.fill_(d)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(slab, want)


@pytest.mark.parametrize("args,code", [
    (dict(ex=False), 1), (dict(layouts=False), 1), (dict(n=-1), 1), (dict(src=None), 1), (dict(dst=None), 1), (dict(kb=0), 1), (dict(vb=0), 1),
    (dict(heads=0), 1), (dict(bs=0), 1), (dict(bs=-16), 1), (dict(hd=0), 1), (dict(pairs=(1 << 31) - 1, heads=8), 1),
    (dict(pairs=(1 << 24) + 1), 1), (dict(heads=180000), 1),
    (dict(fmt=9), 801), (dict(fmt=-1), 801), (dict(hd=192), 801), (dict(fmt=FMT_FP8, hd=128), 801), (dict(fmt=FMT_Q8_0, hd=96), 801), (dict(tok=130), 801),
    (dict(kb=(1 << 20) + 1), 801), (dict(page=16 * 132 * 2 + 1), 801), (dict(tok=133), 801), (dict(tok=1 << 32), 801),
    (dict(n=0), 0), (dict(pairs=0), 0), (dict(pairs=-2), 0), (dict(pairs=0, src=None, dst=None), 0)])
def test_refusals(args, code):
    from warp34_amd import ffi

    a = dict(ex=True, layouts=True, n=2, src=1 << 12, dst=1 << 13, pairs=3, kb=1 << 20, vb=1 << 30, heads=2, bs=16, hd=256, fmt=FMT_TQ4, tok=132,
             page=16 * 132 * 2)
    a.update(args)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    good = (16 * 132 * 2, 16 * 132, 132)
    first = ffi.Warp34KvLayerLayout(1 << 20, 1 << 30, *good, *good, 0, 0, 2, 256, 16, FMT_TQ4, FMT_TQ4, 1, 1, 0)
    second = ffi.Warp34KvLayerLayout(a["kb"], a["vb"], a["page"], 16 * 132, a["tok"], *good, 0, 1, a["heads"], a["hd"], a["bs"], a["fmt"], FMT_TQ4, 1, 1, 0)
    lays = (ffi.Warp34KvLayerLayout * 2)(first, second)
    assert ffi.load().warp34_kv_cache_copy_pages(C.byref(ex) if a["ex"] else None, lays if a["layouts"] else None, a["n"], a["src"], a["dst"], None,
                                                 a["pairs"]) == code
