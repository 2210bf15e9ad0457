"""warp34_linear_attention_*: against the recurrence in 64 bits, with the bounds linear_harness derives."""
import ctypes as C

import pytest

from oracle import DT_BF16, DT_F16

BOTH = pytest.mark.parametrize("dt", [DT_F16, DT_BF16])


def make(*args, **kw):
    from linear_harness import Case

    return Case(*args, **kw)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [5, 3, 8], [2, 1, 7, 1], [4, 3, 1], [4] * 3 + [8] * 70])
def test_single_tokens_and_drafts(lens, dk, dv, dt):
    c = make(lens, dt, dk=dk, dv=dv, seed=len(lens) + dk)
    c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("lens", [[17], [64], [65], [63, 1, 130], [200, 333, 31], [700]])
def test_prompts(lens, dk, dv, dt):
    c = make(lens, dt, dk=dk, dv=dv, seed=len(lens) + dk + lens[0])
    c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("k_heads,v_heads", [(1, 1), (1, 8), (3, 3), (2, 6), (5, 10)])
def test_heads(k_heads, v_heads, dt):
    for lens in ([3, 1], [150, 90]):
        c = make(lens, dt, k_heads=k_heads, v_heads=v_heads, seed=v_heads)
        c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("max_q_len", [None, 0, 1, 1 << 20])
def test_the_bound_changes_the_order_only(max_q_len, dt):
    """A bound that is wrong, or not known, chooses another kernel and nothing else."""
    c = make([70, 1, 200, 4], dt, seed=9)
    c.check(c.call(max_q_len=max_q_len))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[4, 2], [100, 260]])
def test_rows_of_packed_projections(lens, dt):
    """Strides that are wider than the rows, with NaN between them; what lies between output rows stays."""
    c = make(lens, dt, seed=11, pads=(8, 264, 1024, 40, 3))
    c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[3, 1, 5, 0, 2], [3, 1, 4, 0, 2], [80, 1, 300, 0, 129], [600, 0, 1, 700, 0]])
def test_slots(lens, dt):
    """A slot read by two requests, one moved on in place, none to start from, none to go to, a request without tokens."""
    c = make(lens, dt, seed=12, slots=7, state_in=[0, 0, 2, 5, -1], state_out=[3, -1, 2, 6, 4])
    c.check(c.call())
    c = make(lens, dt, seed=13, slots=7, state_in=[0, 1, 2, 5, 6], state_out=[0, 1, 2, 5, 6], has_initial=[1, 0, 1, 0, 1])
    c.check(c.call())
    c = make(lens, dt, seed=14, slots=5, state_in=None, state_out=[0, 1, 2, 3, 4])
    c.check(c.call())
    c = make(lens, dt, seed=15, slots=5, state_in=[0, 1, 2, 3, 4], state_out=None)
    c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[3, 2, 5], [3, 2, 4], [80, 70, 300]])
def test_masked_requests_stay(lens, dt):
    c = make(lens, dt, seed=16, mask=[1, 0, 1])
    c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens,kept", [([5, 5, 5, 5], [1, 0, 5, 3]), ([4, 4, 2, 4], [1, 0, 2, 7]), ([8, 1, 4, 2], [9, -1, 2, 1]), ([200, 130, 64, 300], [64, 129, 63, 0]),
                                       ([500, 65, 128, 129], [257, 64, 1000, 128])])
def test_states_behind_the_kept_tokens(lens, kept, dt):
    c = make(lens, dt, seed=17, kept=kept)
    want = c.want()
    c.check(c.call(), want=want)
    c.check(c.call(with_out=False), with_out=False, want=want)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens,kept,mask", [([5, 4, 3], [2, 0, 3], [1, 1, 0]), ([4, 4, 3], [2, 0, 3], [1, 1, 0]), ([200, 130, 64], [70, 128, 3], [1, 1, 0]),
                                            ([700, 65, 300], [333, 1, 299], [1, 1, 0])])
def test_what_is_not_kept_may_hold_anything(lens, kept, mask, dt):
    """No number in the rows behind the kept tokens, of a masked request and in the slots that requests of zeros would have: the states are unmoved by them."""
    c = make(lens, dt, seed=24, kept=kept, mask=mask, has_initial=[1, 0, 1], slots=6)
    want = c.want()
    for r, length in enumerate(lens):
        left = 0 if not mask[r] else kept[r]
        for x in (c.q, c.k, c.v, c.g):
            x[c.starts[r] + left:c.starts[r] + length] = float("nan")
    c.states[1] = float("nan")
    want[2][1] = 0.0
    for with_out in (False, True):
        out, states = c.call(with_out=with_out)
        assert bool(states[1].isnan().all())
        states[1] = 0.0
        c.check((out, states), with_out=False, want=want)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[6, 1], [4, 1], [333, 128]])
def test_decays(lens, dt):
    import torch

    def forgets(n, h):  # tokens that forget everything, some that forget nothing, and everything between
        g = -torch.rand(n, h).pow(3) * 30
        g[torch.rand(n, h) < 0.05] = -float("inf")
        g[torch.rand(n, h) < 0.1] = 0
        return g

    torch.manual_seed(3)
    for decay in (None, "head", forgets, lambda n, h: torch.full((n, h), -200.0), lambda n, h: torch.full((n, h), -1e-5),
                  lambda n, h: torch.full((n, h), -1e38), lambda n, h: torch.full((n, h), -float("inf"))):
        c = make(lens, dt, seed=18, decay=decay)
        c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[4, 1], [260, 70]])
def test_sizes_of_values_and_states(lens, dt):
    """Large and small values, keys that are not of length one, states far larger than what is added to them."""
    for seed, kw in enumerate([dict(value_scale=200.0), dict(value_scale=2.0 ** -12, state_scale=0.0), dict(unit=False, value_scale=0.1),
                               dict(state_scale=2000.0), dict(state_scale=1e-6, value_scale=1e-3)]):
        c = make(lens, dt, seed=30 + seed, **kw)
        c.check(c.call())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens,heads", [([1000], 2), ([513, 700, 64], 4), ([40, 2000], 2)])
def test_scratch_of_any_size(lens, heads, dt):
    c = make(lens, dt, k_heads=heads // 2, v_heads=heads, seed=19)
    want = c.want()
    for scratch in ("queried", 0, 16, 4 * 128 * 128 * heads * 5, 8 << 20):
        c.check(c.call(scratch=scratch), want=want)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,pad", [([3, 300], 1), ([2, 4], 1), ([300], 4)])
def test_rows_and_slots_far_into_memory(lens, pad):
    """Rows beyond 2^31 elements, slots beyond 2^32 bytes."""
    far = (1 << 23) - 512
    c = make(lens, DT_BF16, seed=25, pads=(0, 0, far, 0, 0) if pad == 1 else (0, far // 8 * 8, 0, far, 0), v_heads=4, slots=2 * len(lens))
    c.check(c.call())
    if pad != 1:
        return
    c = make(lens, DT_BF16, seed=26, k_heads=2, v_heads=32, slots=2300, state_in=[2290, 2291], state_out=[2298, 2299])
    out, bound, states, s_bound = c.want()
    got = c.call()
    c.check((got[0], got[1][2280:]), want=(out, bound, states[2280:], s_bound[2280:]))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("lens", [[3, 4], [700, 300]])
def test_same_call_same_bits(lens, dt):
    import torch

    c = make(lens, dt, seed=20)
    first = c.call()
    for _ in range(3):
        again = c.call()
        assert torch.equal(first[0].view(torch.int16), again[0].view(torch.int16)) and torch.equal(first[1], again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[2, 3], [400, 90]])
def test_on_another_stream(lens):
    import torch

    c = make(lens, DT_BF16, seed=21)
    s = torch.cuda.Stream()
    c.check(c.call(stream=s.cuda_stream))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [([700, 64], [300, 200]), ([4, 2], [900]), ([8] * 5, [1] * 40)])
def test_two_calls_at_once(lens):
    """On two streams, each with a workspace of its own, one behind the other many times: the bits of calls alone."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    cases = [make(x, dt, seed=27 + i, slots=2 * len(x)) for i, (x, dt) in enumerate(zip(lens, (DT_BF16, DT_F16)))]
    alone = [c.call() for c in cases]
    calls, keep = [], []
    for c in cases:
        out, states = c.fresh()
        layout, batch = c.structs(states)
        need = G.lib().warp34_linear_attention_scratch_bytes(C.byref(layout), len(c.lens), c.n, max(c.lens))
        work, stream = torch.zeros(max(16, need), dtype=torch.uint8, device=G.DEV), torch.cuda.Stream()
        ex = ffi.Warp34Exec(stream.cuda_stream, work.data_ptr(), need, 0)
        fn = G.lib().warp34_linear_attention_f16 if c.dt == DT_F16 else G.lib().warp34_linear_attention_bf16
        keep.append((out, states, layout, batch, work, stream, ex))
        calls.append((fn, (C.byref(ex), C.byref(layout), C.byref(batch), G.ptr(c.q), G.ptr(c.k), G.ptr(c.v), G.ptr(c.g), G.ptr(out))))
    torch.cuda.synchronize()
    for _ in range(20):
        for fn, args in calls:
            assert fn(*args) == 0
    torch.cuda.synchronize()
    for c, (want, states), mine in zip(cases, alone, keep):
        got = mine[0][:c.n, :c.hv * c.dv].reshape(want.shape)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and torch.equal(mine[1], states)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1, 4, 2], [8, 1, 5], [300, 65, 400], [300, 65, 640]])
def test_captured(lens):
    """In place in a captured graph: every replay moves the states on, as eager calls do, with eager work between."""
    import torch

    import gpu_harness as G
    from warp34_amd import ffi

    r = len(lens)
    c = make(lens, DT_BF16, seed=22, slots=r, state_in=list(range(r)), state_out=list(range(r)))
    out, states = c.fresh()
    layout, batch = c.structs(states)
    need = G.lib().warp34_linear_attention_scratch_bytes(C.byref(layout), r, c.n, max(lens))
    work = torch.zeros(max(16, need), dtype=torch.uint8, device=G.DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ex = ffi.Warp34Exec(torch.cuda.current_stream().cuda_stream, work.data_ptr(), need, 0)
        rc = G.lib().warp34_linear_attention_bf16(C.byref(ex), C.byref(layout), C.byref(batch), G.ptr(c.q), G.ptr(c.k), G.ptr(c.v), G.ptr(c.g), G.ptr(out))
    assert rc == 0
    eager = c.fresh()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want, _ = c.call(into=eager)
        assert torch.equal(out[:c.n].reshape(want.shape).view(torch.int16), want.view(torch.int16))
        assert torch.equal(states, eager[1])


@pytest.mark.gpu
def test_bounds_that_are_larger_than_the_batch():
    """A captured step's bounds: more tokens than there are, requests without any behind the last."""
    c = make([70, 3, 0, 0], DT_F16, seed=23, slots=9, state_in=[0, 1, -1, -1], state_out=[4, 5, -1, -1])
    c.check(c.call(max_q_len=512))


OK = dict(ex=True, layout=True, batch=True, qsl=1 << 12, q=1 << 20, k=1 << 21, v=1 << 22, g=1 << 23, out=1 << 24, base=1 << 25, slot=4 * 4 * 128 * 128, hk=2,
          hv=4, dk=128, dv=128, s_in=1 << 13, s_out=1 << 14, reqs=3, tokens=10, most=5, scale=0.1, qs=256, ks=256, vs=512, os=512, gs=4)


@pytest.mark.parametrize("args,code", [
    (dict(ex=False), 1), (dict(layout=False), 1), (dict(batch=False), 1), (dict(qsl=None), 1), (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1),
    (dict(hk=0), 1), (dict(hv=0), 1), (dict(hv=3), 1), (dict(hk=-2), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(qs=248), 1), (dict(ks=0), 1), (dict(vs=504), 1), (dict(os=504), 1), (dict(gs=3), 1), (dict(gs=-4), 1), (dict(base=0), 1),
    (dict(slot=4 * 4 * 128 * 128 - 16), 1), (dict(hv=1 << 21, hk=1 << 21), 1),
    (dict(qs=(1 << 23) + 8), 1), (dict(ks=(1 << 23) + 8), 1), (dict(vs=(1 << 23) + 8), 1), (dict(os=(1 << 23) + 8), 1),
    (dict(dk=96), 801), (dict(dv=256, vs=1024, os=1024), 801), (dict(qs=260), 801), (dict(ks=257), 801), (dict(vs=516), 801), (dict(os=513), 801),
    (dict(q=(1 << 20) + 8), 801), (dict(k=(1 << 21) + 2), 801), (dict(v=(1 << 22) + 4), 801), (dict(out=(1 << 24) + 8), 801),
    (dict(base=(1 << 25) + 4), 801), (dict(slot=4 * 4 * 128 * 128 + 8), 801), (dict(g=(1 << 23) + 2), 801),
    (dict(reqs=0), 0), (dict(reqs=-1), 0), (dict(tokens=-1), 0), (dict(out=None, s_out=None), 0), (dict(reqs=1 << 30), 1)])
@pytest.mark.parametrize("name", ["warp34_linear_attention_f16", "warp34_linear_attention_bf16"])
def test_refusals(name, args, code):
    from warp34_amd import ffi

    a = dict(OK)
    a.update(args)
    ex = ffi.Warp34Exec(0, 0, 0, 0)
    layout = ffi.Warp34LinearStateLayout(a["base"], a["slot"], a["hk"], a["hv"], a["dk"], a["dv"])
    batch = ffi.Warp34LinearBatch(a["qsl"], a["s_in"], None, a["s_out"], None, None, a["reqs"], a["tokens"], a["most"], a["scale"], a["qs"], a["ks"], a["vs"],
                                  a["os"], a["gs"], 0)
    assert getattr(ffi.load(), name)(C.byref(ex) if a["ex"] else None, C.byref(layout) if a["layout"] else None, C.byref(batch) if a["batch"] else None,
                                     a["q"], a["k"], a["v"], a["g"], a["out"]) == code


@pytest.mark.parametrize("args", [dict(reqs=0), dict(tokens=0), dict(tokens=16), dict(most=16), dict(hv=0), dict(hv=1 << 21), dict(dk=96), dict(dv=32)])
def test_no_scratch(args):
    from warp34_amd import ffi

    a = dict(OK, reqs=1, tokens=5000, most=5000)
    need = lambda a: ffi.load().warp34_linear_attention_scratch_bytes(  # noqa: E731
        C.byref(ffi.Warp34LinearStateLayout(a["base"], a["slot"], a["hk"], a["hv"], a["dk"], a["dv"])), a["reqs"], a["tokens"], a["most"])
    assert need(a) > 0 and ffi.load().warp34_linear_attention_scratch_bytes(None, 1, 5000, 5000) == 0
    assert need(dict(a, **args)) == 0
