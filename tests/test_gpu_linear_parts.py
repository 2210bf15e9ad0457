"""Linear attention of prompts cut into parts of several chunks: where requests, kept tokens and the parts' borders fall."""
import pytest

from oracle import DT_BF16, DT_F16

BOTH = pytest.mark.parametrize("dt", [DT_F16, DT_BF16])
DIMS = pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])


def make(*args, **kw):
    from linear_harness import Case

    return Case(*args, **kw)


@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("masked", [False, True])
def test_one_prompt_among_many_single_tokens(dk, dv, dt, masked):
    """More than 64 requests, the prompt, masked requests and some without tokens on both sides of the 64th."""
    lens = [1] * 40 + [3000] + [1] * 40
    for r in (3, 38, 62, 63, 64, 65, 80):
        lens[r] = 0
    mask = None
    if masked:
        mask = [1] * len(lens)
        for r in (0, 37, 39, 61, 66, 79):
            mask[r] = 0
    c = make(lens, dt, dk=dk, dv=dv, seed=50, mask=mask)
    want = c.want()
    c.check(c.call(), want=want)
    c.check(c.call(with_out=False), with_out=False, want=want)


@pytest.mark.gpu
@BOTH
@DIMS
def test_prompts_on_both_sides_of_the_64th_request(dk, dv, dt):
    lens = [2] * 62 + [700, 1, 650, 0, 513] + [3] * 62 + [600, 64]
    kept = [max(0, n - 1) for n in lens]
    kept[62], kept[64], kept[66], kept[129] = 333, 192, 513, 0
    c = make(lens, dt, dk=dk, dv=dv, seed=51, kept=kept, mask=[1] * 100 + [0] * 20 + [1] * 11)
    want = c.want()
    c.check(c.call(), want=want)
    c.check(c.call(with_out=False), with_out=False, want=want)


@pytest.mark.gpu
@BOTH
@DIMS
@pytest.mark.parametrize("decay", ["token", "head", None])
def test_kept_tokens_in_parts_of_several_chunks(dk, dv, dt, decay):
    """Workspaces that leave room for parts of 64, 128 and 192 tokens, joined by the rows and by a launch: kept tokens inside of them, at their borders and beside these, on and off the chunks' grid."""
    lens = [700, 450, 513, 400, 0, 384]
    for kept in ([100, 129, 384, 399, 0, 383], [192, 191, 193, 1, 0, 384], [640, 449, 512, 256, 0, 129], [0, 128, 65, 320, 0, 0]):
        c = make(lens, dt, dk=dk, dv=dv, seed=52, kept=kept, decay=decay)
        want = c.want()
        for parts in ("queried", 24, 32):
            scratch = parts if parts == "queried" else 4 * c.hv * (parts + parts * dk * dv) + 16
            c.check(c.call(scratch=scratch), want=want)
            c.check(c.call(scratch=scratch, with_out=False), with_out=False, want=want)
