"""warp34_verify_drafts: accepted drafts and drawn tokens, equal to those of plain 64-bit arithmetic on the same numbers.

A drawn token depends on where u * total falls between running sums; two orders of a 64-bit sum of V terms differ by at most V 2^-53 of the
total, so the plain form says where its borders are nearer than 2^-34 and the test's inputs have none there."""
import ctypes as C

import numpy as np
import pytest


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


class Drafts:
    def __init__(self, lens, vocab, seed, certain=False, target_pad=0, draft_pad=0, spread=3.0, mask=None):
        rng = np.random.default_rng(seed)
        n, r = sum(lens), len(lens)
        self.lens, self.vocab, self.mask = lens, vocab, mask
        logits = rng.standard_normal((n, vocab)) * spread
        self.p = softmax(logits)
        self.q = softmax(logits + rng.standard_normal((n, vocab)))
        self.starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        self.tokens = rng.integers(0, vocab, n).astype(np.int32)
        for i in range(n - 1):
            if i + 1 not in self.starts:
                self.tokens[i + 1] = self.q[i].argmax() if certain else rng.choice(vocab, p=self.q[i].astype(np.float64) / self.q[i].astype(np.float64).sum())
        self.u, self.u_draw = rng.random(n).astype(np.float32), rng.random(r).astype(np.float32)
        self.certain, self.pads = certain, (target_pad, draft_pad)

    def want(self):
        out, counts = np.full(sum(self.lens), 77, np.int32), np.full(len(self.lens), 77, np.int32)
        proper = lambda x: np.where(np.isfinite(x) & (x > 0), x, 0).astype(np.float64)  # noqa: E731
        with np.errstate(all="ignore"):
            for r, n in enumerate(self.lens):
                if self.mask is not None and not self.mask[r]:
                    continue
                lo = self.starts[r]
                out[lo:lo + n] = -1
                counts[r] = 0
                if n == 0:
                    continue
                i, refused = 0, -1
                while i < n - 1:
                    x = self.tokens[lo + i + 1]
                    if not 0 <= x < self.vocab:
                        break
                    q = 1.0 if self.certain else float(self.q[lo + i, x])
                    if not float(self.u[lo + i]) * q < float(self.p[lo + i, x]):
                        refused = x
                        break
                    out[lo + i] = x
                    i += 1
                counts[r] = i + 1
                p = proper(self.p[lo + i])
                w = p
                if refused >= 0:
                    rest = p.copy()
                    if self.certain:
                        rest[refused] = 0
                    else:
                        rest = np.maximum(p - proper(self.q[lo + i]), 0)
                    w = rest if rest.sum() > 0 else p
                if not w.sum() > 0:
                    continue
                running = np.cumsum(w)
                at = float(self.u_draw[r]) * running[-1]
                assert at in (0, running[-1]) or np.abs(running[w > 0] / running[-1] - float(self.u_draw[r])).min() > 2.0 ** -34
                above = np.nonzero((running > at) & (w > 0))[0]
                out[lo + i] = above[0] if len(above) else np.nonzero(w)[0][-1]
        return out, counts

    def device(self):
        import torch

        import gpu_harness as G
        from warp34_amd import ffi

        d = {}
        for name, x, pad in (("p", self.p, self.pads[0]), ("q", self.q, self.pads[1])):
            rows = np.full((x.shape[0], self.vocab + pad), np.nan, np.float32)
            rows[:, :self.vocab] = x
            d[name] = torch.from_numpy(rows).to(G.DEV)
        if self.certain:
            d["q"] = None
        for name in ("tokens", "u", "u_draw", "starts"):
            d[name] = torch.from_numpy(np.ascontiguousarray(getattr(self, name))).to(G.DEV)
        d["mask"] = None if self.mask is None else torch.tensor(self.mask, dtype=torch.uint8, device=G.DEV)
        d["out"] = torch.full((sum(self.lens) + 1,), 77, dtype=torch.int32, device=G.DEV)
        d["counts"] = torch.full((len(self.lens) + 1,), 77, dtype=torch.int32, device=G.DEV)
        d["batch"] = ffi.Warp34DraftBatch(d["starts"].data_ptr(), d["tokens"].data_ptr(), None if self.mask is None else d["mask"].data_ptr(),
                                          self.vocab + self.pads[0], self.vocab + self.pads[1], len(self.lens), sum(self.lens), max(self.lens), self.vocab)
        return d

    def call(self, d, scratch="queried", stream=None):
        import torch

        import gpu_harness as G
        from warp34_amd import ffi

        need = G.lib().warp34_verify_drafts_scratch_bytes(len(self.lens), self.vocab)
        size = need if scratch == "queried" else scratch
        work = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device=G.DEV)
        torch.cuda.synchronize()
        ex = ffi.Warp34Exec(stream or torch.cuda.current_stream().cuda_stream, work.data_ptr() if size else 0, size, 0)
        rc = G.lib().warp34_verify_drafts(C.byref(ex), C.byref(d["batch"]), G.ptr(d["p"]), G.ptr(d["q"]), G.ptr(d["u"]), G.ptr(d["u_draw"]), G.ptr(d["out"]),
                                          G.ptr(d["counts"]))
        torch.cuda.synchronize()
        assert rc == 0 and bool((work[size:] == 0xA5).all())
        assert int(d["out"][-1]) == 77 and int(d["counts"][-1]) == 77
        return d["out"][:-1].cpu().numpy(), d["counts"][:-1].cpu().numpy()

    def check(self, **kw):
        want = self.want()
        got = self.call(self.device(), **kw)
        assert (got[1] == want[1]).all(), (got[1], want[1])
        assert (got[0] == want[0]).all(), (got[0], want[0])
        return want


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("lens,vocab", [([1], 1), ([4], 1), ([3, 2], 2), ([4], 1023), ([5, 1, 8, 2], 1024), ([2, 7, 1], 1025), ([6] * 9, 5000), ([3, 4], 32768),
                                        ([4, 2], 150001), ([1, 70, 130], 700), ([2] * 40, 3001)])
def test_accepted_and_drawn_tokens(lens, vocab, certain):
    for seed in range(3):
        d = Drafts(lens, vocab, seed * 100 + vocab % 97 + len(lens), certain=certain, target_pad=seed * 3, draft_pad=seed)
        d.check()
        d.check(scratch=0)


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", ["queried", 0])
def test_rows_far_apart(scratch):
    """Rows beyond 2^31 elements."""
    import torch

    import gpu_harness as G

    d = Drafts([4], 3000, 11)
    d.u[:2] = 0
    want, dev, stride = d.want(), d.device(), (1 << 30) + 5
    for name in ("p", "q"):
        far = torch.empty(3 * stride + 3000, dtype=torch.float32, device=G.DEV)
        for i in range(4):
            far[i * stride:i * stride + 3000] = dev[name][i]
        dev[name] = far
    dev["batch"].target_row_stride = dev["batch"].draft_row_stride = stride
    got = d.call(dev, scratch=scratch)
    assert want[1][0] >= 3 and (got[0] == want[0]).all() and (got[1] == want[1]).all()


@pytest.mark.gpu
def test_every_draft_accepted_and_every_draft_refused():
    d = Drafts([5, 5, 1, 3], 4000, 7)
    d.u[:] = 0
    _, counts = d.check()
    assert (counts == d.lens).all()
    d.u[:] = 0.999
    d.q[:] = 1.0  # more than any p: refused, and nothing is left of p - q, so that the token is drawn from p
    _, counts = d.check()
    assert (counts == 1).all()


@pytest.mark.gpu
def test_equal_distributions_accept_and_have_no_rest():
    """q = p: every draft is accepted for u < 1; with the same u * q = p a draft is refused and the rest is zero everywhere: drawn from p."""
    d = Drafts([6, 4], 3000, 8)
    d.q[:] = d.p
    d.u[:] = 0.75
    assert (d.check()[1] == d.lens).all()
    d.u[:] = 1.0
    assert (d.check()[1] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("certain", [False, True])
def test_drafts_outside_the_vocabulary_end_them(certain):
    d = Drafts([4, 4, 4, 3], 2500, 9, certain=certain)
    d.u[:] = 0
    for row, token in ((1, -1), (6, 2500), (11, -(1 << 31)), (13, (1 << 31) - 1)):
        d.tokens[row] = token
    _, counts = d.check()
    assert counts.tolist() == [1, 2, 3, 1]


@pytest.mark.gpu
def test_entries_that_are_no_probabilities():
    d = Drafts([3, 3, 1, 1], 1500, 10)
    d.p[:, 7::50] = np.nan
    d.p[:, 9::50] = -1
    d.p[:, 11::50] = np.inf
    d.q[:, 13::50] = np.nan
    d.q[:, 17::50] = -2
    d.q[:, 19::50] = np.inf
    d.p[6] = 0  # nothing to draw
    d.p[7] = np.nan
    out, _ = d.check()
    assert out[6] == -1 and out[7] == -1
    d.check(scratch=0)


@pytest.mark.gpu
def test_one_hot_rows_decode_greedily():
    rng = np.random.default_rng(11)
    d = Drafts([5, 5], 2000, 11)
    best = rng.integers(0, 2000, 10)
    d.p[:] = 0
    d.p[np.arange(10), best] = 1
    d.tokens[[1, 2]], d.tokens[3] = best[[0, 1]], (best[2] + 1) % 2000  # two right, one wrong
    d.q[:] = 0
    for row in range(9):
        d.q[row, d.tokens[row + 1]] = 1
    d.tokens[6:10], d.q[5:9] = best[5:9], d.p[5:9]
    out, counts = d.check()
    assert counts.tolist() == [3, 5] and out[:3].tolist() == best[:3].tolist() and out[5:].tolist() == best[5:].tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0])
def test_draws_at_the_ends(u):
    """u = 0 takes the first entry with any weight, u next to 1 (or 1, which is out of range) the last one."""
    d = Drafts([1, 1, 1], 4100, 12)
    d.p[:] = 0
    for r, entries in enumerate(([5, 6, 4099], [1023, 1024, 2050], [0, 4096])):
        d.p[r, entries] = 0.25
    d.u_draw[:] = u
    out, _ = d.check()
    assert out.tolist() == ([5, 1023, 0] if u == 0 else [4099, 2050, 4096])


@pytest.mark.gpu
def test_masked_requests_and_requests_without_rows():
    d = Drafts([4, 0, 3, 2, 0], 1200, 13, mask=[1, 1, 0, 1, 0])
    out, counts = d.check()
    assert counts[1] == 0 and counts[2] == 77 and counts[4] == 77 and (out[4:7] == 77).all()


@pytest.mark.gpu
def test_sums_that_32_bits_would_lose():
    """One large entry in front of many small ones: the draw falls among the small ones."""
    d = Drafts([1, 1], 200000, 14)
    d.p[:] = np.float32(1e-9)
    d.p[:, 3] = 1.0
    d.u_draw[:] = [np.float32(0.99990), np.float32(0.99985)]
    out, _ = d.check()
    assert (out > 1000).all()


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    d = Drafts([4, 3, 5], 9001, 15)
    want = d.want()
    s = torch.cuda.Stream()
    got = d.call(d.device(), stream=s.cuda_stream)
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()
    t = d.device()
    need = G.lib().warp34_verify_drafts_scratch_bytes(3, 9001)
    work = torch.zeros(need, dtype=torch.uint8, device=G.DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, work.data_ptr(), need, 0)
        rc = G.lib().warp34_verify_drafts(C.byref(ex), C.byref(t["batch"]), G.ptr(t["p"]), G.ptr(t["q"]), G.ptr(t["u"]), G.ptr(t["u_draw"]),
                                          G.ptr(t["out"]), G.ptr(t["counts"]))
    assert rc == 0
    rng = np.random.default_rng(16)
    for _ in range(4):  # new numbers into the captured step's buffers
        d.u, d.u_draw = rng.random(12).astype(np.float32), rng.random(3).astype(np.float32)
        t["u"].copy_(torch.from_numpy(d.u))
        t["u_draw"].copy_(torch.from_numpy(d.u_draw))
        graph.replay()
        torch.cuda.synchronize()
        want = d.want()
        assert (t["out"][:-1].cpu().numpy() == want[0]).all() and (t["counts"][:-1].cpu().numpy() == want[1]).all()


@pytest.mark.parametrize("args,code", [
    (dict(ex=False), 1), (dict(batch=False), 1), (dict(qsl=None), 1), (dict(tokens=None), 1), (dict(p=None), 1), (dict(u=None), 1), (dict(u_draw=None), 1),
    (dict(out=None), 1), (dict(counts=None), 1), (dict(vocab=0), 1), (dict(vocab=-5), 1), (dict(ps=999), 1), (dict(qs=999), 1), (dict(reqs=(1 << 20) + 1), 1),
    (dict(reqs=0), 0), (dict(reqs=-3), 0), (dict(total=0), 0)])
def test_refusals(args, code):
    from warp34_amd import ffi

    a = dict(ex=True, batch=True, qsl=1 << 12, tokens=1 << 13, p=1 << 20, q=1 << 21, u=1 << 14, u_draw=1 << 15, out=1 << 16, counts=1 << 17, vocab=1000,
             ps=1000, qs=1000, reqs=2, total=6)
    a.update(args)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    batch = ffi.Warp34DraftBatch(a["qsl"], a["tokens"], None, a["ps"], a["qs"], a["reqs"], a["total"], 3, a["vocab"])
    assert ffi.load().warp34_verify_drafts(C.byref(ex) if a["ex"] else None, C.byref(batch) if a["batch"] else None, a["p"], a["q"], a["u"], a["u_draw"],
                                           a["out"], a["counts"]) == code


def test_scratch_sizes():
    from warp34_amd import ffi

    size = ffi.load().warp34_verify_drafts_scratch_bytes
    assert size(0, 1000) == size(3, 0) == size(-1, 5) == 0
    assert size(1, 1) >= 16 and size(3, 200000) <= 1 << 20
