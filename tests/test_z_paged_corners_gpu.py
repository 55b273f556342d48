"""Corners of the paged cache and of the attention over it: windows without end, infinite keys under the rotation, capped scores beside
hidden keys, what a block loses while its scale grows, batches of single tokens and chunks."""
import math

import pytest
import torch

import paged_ref as R
import test_w_paged_cache_gpu as W

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def _dev(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 30, 2 ** 30])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_window_without_end_where_tokens_have_no_position(window, d):
    """More new tokens than positions, and a window of the largest numbers: positions before the first one see nothing, the others all
    keys up to their own.  Few rows a sequence, and chunks."""
    _, _, _, _, o, lse = W._run_attend(4, 2, d, 16, [5, 3, 1], [2, 3, 40], seed=2, window=window)
    assert (o[:3] == 0).all() and lse[:, :3].isneginf().all() and lse[:, 3:].isfinite().all()
    _, _, _, _, o, lse = W._run_attend(4, 1, d, 16, [40, 70], [17, 90], seed=3, window=window)
    assert (o[:23] == 0).all() and lse[:, :23].isneginf().all() and lse[:, 23:].isfinite().all()
