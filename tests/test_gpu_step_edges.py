"""Edges of a decode step's preparation on the GPU: queries whose channels are far apart, against the oracle's exact sums."""
import numpy as np
import pytest
import torch

from tests.test_gpu_step import DIMS, _check_select, _records, _tables

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ block selection
@pytest.mark.parametrize("dims,hq,hkv,n_sel,top", [(DIMS[1], 16, 1, 16, 36), (DIMS[1], 16, 1, 16, 44), (DIMS[0], 1, 1, 40, 44),
                                                   (DIMS[2], 10, 2, 300, 60), (DIMS[0], 256, 1, 7, 100)])
def test_select_of_a_query_with_a_far_channel(dims, hq, hkv, n_sel, top):
    """One channel of 2^top, whose keys are zero, and channels of 1 that decide: its products are 0 exactly, those of the others and
    their sums in fp64 lose 2^-50 of the scores, which are 2^-10 apart and more but for one pair in 10^10."""
    g = torch.Generator().manual_seed(top + hq)
    lens = [65536 if hkv == 1 else 30000, 700, 40]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(top))
    x = torch.randn(count, hkv, 64, dims[0], generator=g)
    x[..., 5] = 0
    q = torch.randn(len(lens), hq, dims[0], generator=g)
    q[:, hq // 2, 5] = 2.0**top
    q[1, 0, 5] = -2.0**top
    _check_select(q.to(torch.bfloat16), _records(x, dims[1]), pages, lens, n_sel)


@pytest.mark.parametrize("dims", DIMS[:3])
def test_select_of_many_rows_with_far_channels(dims):
    """The same where blocks of the second kernel are small; every second row's channels are alike."""
    rng, g = np.random.default_rng(dims[0]), torch.Generator().manual_seed(dims[0])
    lens = rng.integers(1, 1500, 200)
    pages, count = _tables([1500], 32, 16, rng)
    pages = np.stack([np.roll(pages[0], r) for r in range(len(lens))])
    x = torch.randn(count, 4, 64, dims[0], generator=g)
    x[..., 40] = 0
    q = torch.randn(len(lens), 8, dims[0], generator=g)
    q[::2, 1::2, 40] = -2.0**50
    q[::4, 1, 40] = 2.0**-100  # (far below: lost by none of the sums, as its keys are zero)
    _check_select(q.to(torch.bfloat16), _records(x, dims[1]), pages, lens, 9)


def test_select_of_fp16_numbers_from_the_smallest_to_the_largest():
    """256 heads leave the whole numbers 38 bits, of which fp16 has 40."""
    g = torch.Generator().manual_seed(3)
    lens = [5000, 64]
    pages, count = _tables(lens, 32, 16, np.random.default_rng(4))
    x = torch.randn(count, 1, 64, 64, generator=g)
    x[..., 63] = 0
    q = torch.randint(-3, 4, (2, 256, 64), generator=g) * 2.0**-24
    q[:, 17, 63] = 65504.0
    _check_select(q.to(torch.float16), _records(x, 64), pages, lens, 12)
