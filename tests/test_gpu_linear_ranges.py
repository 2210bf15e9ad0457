"""Linear attention of numbers of very different sizes beside each other: each within linear_harness's bound of its own terms, whatever its neighbours are."""
import pytest

from oracle import DT_BF16

LENS = pytest.mark.parametrize("lens", [[64], [200, 333], [70, 1, 900]])


def make(*args, **kw):
    from linear_harness import Case

    return Case(*args, **kw)


def put(c, name, x):
    """Rows of q, k or v of a case without gaps, [tokens, heads, channels]."""
    getattr(c, name)[:c.n] = x.reshape(c.n, -1).to(c.q.dtype)


def check(c):
    """By chunks whatever the lengths, with the workspace and without."""
    want = c.want()
    for scratch in ("queried", 0):
        c.check(c.call(scratch=scratch, max_q_len=c.n + 1 if max(c.lens) < 17 else None), want=want)
    c.check(c.call(with_out=False), with_out=False, want=want)


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
