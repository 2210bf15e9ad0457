"""Linear attention of numbers of very different sizes beside each other: each within linear_harness's bound of its own terms, whatever its neighbours are.

What numbers of limited range add to that bound (floors()): weights below 2^-126 count as zero, and so may the parts of operands below that; fp16 operands,
scaled to put the largest of their column (of weighted values in a chunk, of states) or row (of weights) at 2^14 or more, are a number whose last place is
2^-24 or more and a rest of it, which is held times 2^11 and rounded by 2^-25 at most: 2^-36 of 2^14, 2^-50 of the largest."""
import pytest

from oracle import DT_BF16, DT_F16

BOTH = pytest.mark.parametrize("dt", [DT_F16, DT_BF16])
LENS = pytest.mark.parametrize("lens", [[64], [200, 333], [70, 1, 900]])
DIMS = pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])


def make(*args, **kw):
    from linear_harness import Case

    return Case(*args, **kw)


def put(c, name, x):
    """Rows of q, k or v of a case without gaps, [tokens, heads, channels]."""
    getattr(c, name)[:c.n] = x.reshape(c.n, -1).to(c.q.dtype)


def plain(shape, seed):
    """Numbers between 0.5 and 1.5 of either sign: none is near zero."""
    import torch

    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.rand(shape, generator=gen, device="cuda")
    return (0.5 + x) * torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.5, -1.0, 1.0)


def one_hot(c, heads, by):
    """Rows with a single one, in channel (by * token) % dk."""
    import torch

    x = torch.zeros((c.n, heads, c.dk), device="cuda")
    t = torch.arange(c.n, device="cuda")
    x[t, :, by * t % c.dk] = 1.0
    return x


def floors(c):
    """(of outputs, of states): what the smallest numbers that operands can hold add to the bounds; sizes of a request's keys, values and states are taken over
    all of its tokens, and weights as one."""
    import torch

    n = c.n
    heads = lambda x, h, d: x[:n, :h * d].double().abs().reshape(n, h, d).repeat_interleave(c.hv // h, 1)  # noqa: E731
    q, k, v = heads(c.q, c.hk, c.dk), heads(c.k, c.hk, c.dk), heads(c.v, c.hv, c.dv)
    least = 2.0 ** -126 + (2.0 ** -50 if c.dt == DT_F16 else 0.0)
    out, states = torch.zeros(v.shape, dtype=torch.float64, device="cuda"), torch.zeros(c.states.shape, dtype=torch.float64, device="cuda")
    for r, length in enumerate(c.lens):
        rows = slice(c.starts[r], c.starts[r] + length)
        keys, values = k[rows].sum(0), v[rows].sum(0)  # [head, channel], [head, column]
        began = c.states[c.in_list[r]].double().abs()
        floor = least * keys[:, :, None] * (1 + v[rows].amax(0))[:, None, :] + 2.0 ** -126 * began
        largest = (began + keys[:, :, None] * v[rows].amax(0)[:, None, :]).amax(1)  # of a column of the state
        product = (q[rows].sum(2) * k[rows].amax((0, 2)))[:, :, None]  # of a query and a key, at most
        out[rows] = c.scale * ((q[rows][:, :, :, None] * floor).sum(2) + least * q[rows].sum(2)[:, :, None] * (1 + largest) + least * product * (1 + values))
        states[c.out_list[r]] = floor
    return out, states


def check(c, more=None):
    """By chunks whatever the lengths, with the workspace and without."""
    want = c.want()
    if more is not None:
        want = (want[0], want[1] + more[0], want[2], want[3] + more[1])
    for scratch in ("queried", 0):
        c.check(c.call(scratch=scratch, max_q_len=c.n + 1 if max(c.lens) < 17 else None), want=want)
    c.check(c.call(with_out=False), with_out=False, want=want)


@pytest.mark.gpu
@BOTH
@LENS
@DIMS
@pytest.mark.parametrize("fade", [-float("inf"), -30.0, -18.0])
def test_small_values_behind_large_ones_that_are_gone(lens, dk, dv, dt, fade):
    """Inside a chunk: large values, a token that lets them go, small values."""
    import torch

    c = make(lens, dt, dk=dk, dv=dv, seed=40, state_scale=1e-4)
    t = torch.arange(c.n, device="cuda")
    large = (t % 50 < 20)[:, None, None]
    put(c, "v", plain((c.n, c.hv, dv), 1) * torch.where(large, 3e3, 1e-4))
    c.g[:c.n][t % 50 == 20] = fade
    check(c)


@pytest.mark.gpu
@BOTH
@LENS
@DIMS
def test_columns_of_different_sizes(lens, dk, dv, dt):
    import torch

    c = make(lens, dt, dk=dk, dv=dv, seed=41)
    size = torch.where(torch.arange(dv, device="cuda") % 2 == 0, 3e3, 1e-4)
    put(c, "v", plain((c.n, c.hv, dv), 2) * size)
    c.states *= size
    check(c)


@pytest.mark.gpu
@BOTH
@LENS
@DIMS
def test_channels_of_different_sizes(lens, dk, dv, dt):
    """Keys that each go to one channel: tokens of large and of small values never meet in a sum; queries that read one channel each."""
    import torch

    c = make(lens, dt, dk=dk, dv=dv, seed=42)
    t = torch.arange(c.n, device="cuda")
    put(c, "k", one_hot(c, c.hk, 1))
    put(c, "q", one_hot(c, c.hk, 3))
    put(c, "v", plain((c.n, c.hv, dv), 3) * torch.where(t % 2 == 0, 3e3, 1e-4)[:, None, None])
    c.states = plain(c.states.shape, 4) * torch.where(torch.arange(dk, device="cuda") % 2 == 0, 3e3, 1e-4)[:, None]
    check(c, floors(c))


@pytest.mark.gpu
@BOTH
@LENS
@pytest.mark.parametrize("state", [2.0 ** 60, 2.0 ** 100, 2.0 ** -60, 2.0 ** -100])
def test_states_far_from_their_values(lens, dt, state):
    """Values of 10^-4 join states of any size; outputs are looked at behind a token that forgets them."""
    import torch

    c = make(lens, dt, seed=43, state_scale=state, value_scale=1e-4)
    c.g[:c.n].clamp_(min=-0.05)  # what is left of the state stays the larger part, or the smaller one
    want = c.want()
    c.check(c.call(with_out=False), with_out=False, want=want)
    c.check(c.call(with_out=False, scratch=0), with_out=False, want=want)
    c.g[torch.tensor(c.starts[:-1], device="cuda").long()] = -float("inf")
    check(c)


@pytest.mark.gpu
@BOTH
def test_values_that_have_faded_far(dt):
    """A value at the start of a chunk alone, of which 2^-100 is left at its end: the state keeps that."""
    import torch

    c = make([64, 128], dt, seed=44, state_scale=0.0, decay=lambda n, h: torch.full((n, h), -1.1))
    v = c.v.clone()
    c.v[:c.n] = 0
    for first in (0, 64, 128):
        c.v[first] = v[first]
    check(c)


def sizes(c):
    """Sums of the outputs' terms without their signs."""
    import torch

    heads = lambda x, h, d: x[:c.n, :h * d].double().abs().reshape(c.n, h, d).repeat_interleave(c.hv // h, 1)  # noqa: E731
    q, k, v = heads(c.q, c.hk, c.dk), heads(c.k, c.hk, c.dk), heads(c.v, c.hv, c.dv)
    got = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for r, length in enumerate(c.lens):
        a = c.states[c.in_list[r]].double().abs()
        for row in range(c.starts[r], c.starts[r] + length):
            a = torch.exp(c.g[row, :c.hv].double())[:, None, None] * a + k[row][:, :, None] * v[row][:, None, :]
            got[row] = c.scale * (q[row][:, :, None] * a).sum(1)
    return got


@pytest.mark.gpu
@BOTH
@LENS
@DIMS
def test_terms_that_cancel(lens, dk, dv, dt):
    """Tokens that take back what the ones before them added, but for a little.  Of fp16 the operands' 22 bits show: 2^-22 of states, of weights, and 20 roundings of 2^-24
    (eight products of a state, four of weights, two each, less those of one term) are within 2^-19, where the harness has 2^-15 for the 16 bits of bf16."""
    import torch

    c = make(lens, dt, dk=dk, dv=dv, seed=46, decay=lambda n, h: torch.full((n, h), -2.0 ** -10), state_scale=1e-3)
    for x, sign in ((c.q, 1), (c.k, 1), (c.v, -1)):
        x[1:c.n:2] = sign * x[0:c.n // 2 * 2:2]
    out, bound, states, s_bound = c.want()
    if dt == DT_F16:
        bound = bound - (2.0 ** -15 - 2.0 ** -19) * sizes(c)
    for scratch in ("queried", 0):
        c.check(c.call(scratch=scratch), want=(out, bound, states, s_bound))


@pytest.mark.gpu
@LENS
@pytest.mark.parametrize("q_size,k_size,scale", [(40, 40, None), (44, 44, 2.0 ** -20), (-50, -50, 2.0 ** 100), (0, 0, 2.0 ** 90), (30, 30, 2.0 ** -100)])
def test_large_products_and_scales(lens, q_size, k_size, scale):
    """Products of queries and keys, and scales, that times 2^50 are no numbers, under decays that weigh them by factors of that size."""
    import torch

    c = make(lens, DT_BF16, seed=45, decay=lambda n, h: torch.full((n, h), -2.0), state_scale=2.0 ** k_size)
    put(c, "q", c.q[:c.n].float() * 2.0 ** q_size)
    put(c, "k", c.k[:c.n].float() * 2.0 ** k_size)
    c.scale = c.scale if scale is None else scale
    check(c)
