"""The operators of a branching step in a row, as a serving loop makes the calls: prompts into state slots and pages, a request forked (its pages
copied, its state carried over by a request without tokens), drafted tokens run through a linear layer, verified, and the accepted part committed to
the states by counts that never leave the device; all of it captured and replayed with other drafts."""
import ctypes as C

import numpy as np
import pytest
import torch

import oracle
from oracle import DT_BF16, FMT_TQ4, XF_WHT256

pytestmark = pytest.mark.gpu

HK, HV, D, VOCAB = 2, 4, 128, 3000
LENS = [70, 33]   # prompts of two requests; the second one is forked
DRAFTED = 4       # tokens of the step: the last one known and three drafts


def recurrence(state, q, k, v, g, scale):
    """Rows [n, heads, dim] in 64 bits from a state; (out, state behind each number of rows)."""
    states, outs = [state.clone()], []
    k, q = (x.double().repeat_interleave(HV // HK, 1) for x in (k, q))
    for t in range(q.shape[0]):
        state = state * torch.exp(g[t].double())[:, None, None] + k[t][:, :, None] * v[t].double()[:, None, :]
        outs.append((q[t][:, :, None] * state).sum(1) * scale)
        states.append(state.clone())
    return outs, states


def test_fork_verify_commit():
    import gpu_harness as G
    from warp34_amd import ffi

    lib, dev = G.lib(), G.DEV
    gen = torch.Generator(device=dev)
    gen.manual_seed(5)
    scale = D ** -0.5
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731

    def rows(n):
        q, k = (torch.randn((n, HK, D), generator=gen, device=dev) for _ in range(2))
        return ((q / q.norm(dim=-1, keepdim=True)).bfloat16(), (k / k.norm(dim=-1, keepdim=True)).bfloat16(),
                torch.randn((n, HV, D), generator=gen, device=dev).bfloat16(), -torch.rand((n, HV), generator=gen, device=dev))

    states = torch.zeros((8, HV, D, D), device=dev)
    layout = ffi.Warp34LinearStateLayout(states.data_ptr(), 4 * HV * D * D, HK, HV, D, D)
    work = torch.zeros(32 << 20, dtype=torch.uint8, device=dev)

    def linear(stream, x, qsl, s_in, s_out, kept=None, out=None, most=0):
        reqs, n = qsl.numel() - 1, x[0].shape[0]
        batch = ffi.Warp34LinearBatch(qsl.data_ptr(), s_in.data_ptr(), None, None if s_out is None else s_out.data_ptr(),
                                      None if kept is None else kept.data_ptr(), None, reqs, n, most, scale, HK * D, HK * D, HV * D, HV * D, HV, 0)
        ex = ffi.Warp34Exec(stream, work.data_ptr(), work.numel(), 0)
        assert lib.warp34_linear_attention_bf16(C.byref(ex), C.byref(layout), C.byref(batch), *(G.ptr(t) for t in x), G.ptr(out)) == 0

    stream = torch.cuda.current_stream().cuda_stream
    # prompts: states 0 and 1
    prompt = rows(sum(LENS))
    out = torch.zeros((sum(LENS), HV, D), dtype=torch.bfloat16, device=dev)
    linear(stream, prompt, i32([0, LENS[0], sum(LENS)]), i32([-1, -1]), i32([0, 1]), out=out, most=max(LENS))
    want = []
    for lo, hi in ((0, LENS[0]), (LENS[0], sum(LENS))):
        outs, after = recurrence(torch.zeros((HV, D, D), dtype=torch.float64, device=dev), *(x[lo:hi] for x in prompt), scale)
        want.append(after[-1])
        assert float((out[lo:hi].double() - torch.stack(outs)).abs().max()) < 2.0 ** -8
    torch.cuda.synchronize()
    for r in range(2):
        assert float((states[r].double() - want[r]).abs().max()) < 1e-5
    # the cache of a layer: rows of both prompts, then the second request forks: pages copied, state 1 to slot 2 by a request without tokens
    pool = oracle.HostPool(8, 2, 256, 16, FMT_TQ4, XF_WHT256)
    dpool = G.DevPool(pool)
    tables = [[0, 1, 2, 3, 4], [5, 6, 7]]
    bits = oracle.fill_normal(LENS[1] * 2 * 256, 9, DT_BF16).reshape(LENS[1], 2, 256)
    hb = oracle.HostBatch([0, LENS[1]], [LENS[1]], np.array([tables[1]], dtype=np.int32), context_lens_before=[0],
                          write_slot_mapping=[tables[1][p // 16] * 16 + p % 16 for p in range(LENS[1])])
    assert G.dev_write(dpool, hb, bits, bits, DT_BF16) == 0
    lay = dpool.layout()
    ex = ffi.Warp34Exec(stream, 0, 0, 0)
    src, dst, count = i32(tables[1]), i32([1, 3, 0]), i32([16, 16, 1])
    assert lib.warp34_kv_cache_copy_pages(C.byref(ex), C.byref(lay), 1, G.ptr(src), G.ptr(dst), G.ptr(count), 3) == 0
    back = [torch.zeros((LENS[1], 512), dtype=torch.bfloat16, device=dev) for _ in range(2)]
    for table, to in ((tables[1], back[0]), ([1, 3, 0], back[1])):
        slots = i32([table[p // 16] * 16 + p % 16 for p in range(LENS[1])])
        assert lib.warp34_kv_cache_read_bf16(C.byref(ex), C.byref(lay), G.ptr(slots), LENS[1], G.ptr(to), None, 512, 512) == 0
        torch.cuda.synchronize()
    assert torch.equal(back[0], back[1]) and bool(back[0].any())
    linear(stream, rows(1), i32([0, 0]), i32([1]), i32([2]), most=1)
    torch.cuda.synchronize()
    assert torch.equal(states[1], states[2])

    # three requests' drafted step, in a graph: rows of the linear layer (no state written), the verification, the states behind what it accepted
    n, reqs = 3 * DRAFTED, 3
    qsl, s_in, s_out = i32([0, DRAFTED, 2 * DRAFTED, n]), i32([0, 1, 2]), i32([3, 4, 5])
    step = rows(n)
    step_out = torch.zeros((n, HV, D), dtype=torch.bfloat16, device=dev)
    p = torch.zeros((n, VOCAB), device=dev)
    q = torch.zeros((n, VOCAB), device=dev)
    tokens, emitted, counts = i32([0] * n), i32([0] * n), i32([0] * reqs)
    u, u_draw = torch.zeros(n, device=dev), torch.zeros(reqs, device=dev)
    drafts = ffi.Warp34DraftBatch(qsl.data_ptr(), tokens.data_ptr(), None, VOCAB, VOCAB, reqs, n, DRAFTED, VOCAB)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        linear(s, step, qsl, s_in, None, out=step_out, most=DRAFTED)
        ex = ffi.Warp34Exec(s, work.data_ptr(), work.numel(), 0)
        assert lib.warp34_verify_drafts(C.byref(ex), C.byref(drafts), G.ptr(p), G.ptr(q), G.ptr(u), G.ptr(u_draw), G.ptr(emitted), G.ptr(counts)) == 0
        linear(s, step, qsl, s_in, s_out, kept=counts, most=DRAFTED)
    seen = set()
    for turn in range(5):
        logits = torch.randn((n, VOCAB), generator=gen, device=dev) * 2
        p.copy_(torch.softmax(logits, -1))
        q.copy_(torch.softmax(logits + 0.7 * torch.randn((n, VOCAB), generator=gen, device=dev), -1))
        drawn = torch.multinomial(q, 1, generator=gen)[:, 0].int()
        tokens.copy_(torch.cat([drawn[:1] * 0, drawn[:-1]]))
        u.copy_(torch.rand(n, generator=gen, device=dev))
        u_draw.copy_(torch.rand(reqs, generator=gen, device=dev))
        for t, x in zip(step, rows(n)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(reqs):
            lo, accepted = r * DRAFTED, 0
            while accepted < DRAFTED - 1:
                row, x = lo + accepted, int(tokens[lo + accepted + 1])
                if not float(u[row]) * float(q[row, x]) < float(p[row, x]):
                    break
                accepted += 1
            assert int(counts[r]) == accepted + 1
            assert emitted[lo:lo + accepted].tolist() == tokens[lo + 1:lo + 1 + accepted].tolist() and int(emitted[lo + accepted]) >= 0
            assert (emitted[lo + accepted + 1:lo + DRAFTED] == -1).all()
            seen.add(accepted)
            outs, after = recurrence(states[int(s_in[r])].double(), *(x[lo:lo + DRAFTED] for x in step), scale)
            assert float((step_out[lo:lo + DRAFTED].double() - torch.stack(outs)).abs().max()) < 2.0 ** -8
            assert float((states[int(s_out[r])].double() - after[accepted + 1]).abs().max()) < 1e-5
    assert len(seen) > 1, "drafts of several lengths were accepted"
