"""Long walks of the scored decode kernels from inside a page, whose entries of the block table are asked for 64 at a time."""
import numpy as np
import pytest

from cases import make_case
from oracle import DT_BF16, DT_F16, FMT_BF16, FMT_FP8, FMT_Q8_0, FMT_TQ4
from scored_harness import check_scored


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", [0, 8 << 20])
@pytest.mark.parametrize("block,window,seq", [(32, 2048, 2065), (32, 2048, 2070), (32, 2061, 4133), (48, 0, 3120), (48, 3100, 3170),
                                              (64, 4096, 4117), (64, 4112, 4180)])
@pytest.mark.parametrize("fmt,dt", [(FMT_TQ4, DT_BF16), (FMT_BF16, DT_BF16), (FMT_FP8, DT_F16), (FMT_Q8_0, DT_F16)])
def test_windows_that_open_inside_a_page(fmt, dt, block, window, seq, scratch):
    pool, bt, k, v, q, aq, ctx = make_case(fmt, block, [seq, 40], [1, 1], 1300, dt, kv_heads=1, q_heads=8)
    wide = np.zeros((2, bt.shape[1] + 70), dtype=np.int32)
    wide[:, :bt.shape[1]] = bt
    check_scored(pool, wide, [seq, 40], q, dt, aq, ctx, 8, scratch=scratch, window=window, cap=30.0)
