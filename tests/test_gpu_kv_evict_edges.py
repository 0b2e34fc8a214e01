"""iq_kv_evict where no row has to move."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv_cache import check_evict

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def zeros(rng, w):
    return np.zeros_like(w)


def falling(rng, w):
    return np.broadcast_to(-np.arange(w.shape[2], dtype=np.float32), w.shape).copy()


def last_is_high(rng, w):
    """One free place in the last head of the last sequence, none elsewhere."""
    w = falling(rng, w)
    w[-1, -1, 70] = 1.0
    return w


@pytest.mark.parametrize("sums", [zeros, falling, last_is_high])
@pytest.mark.parametrize("hk,d,page,dtype", [(2, 64, 16, BF), (4, 128, 7, HF), (1, 8, 1, BF), (3, 256, 33, HF)])
def test_the_first_tokens_stay_and_none_is_newest(hk, d, page, dtype, sums):
    """recent = 0 and the largest sums in front: no row moves.  Few rows, which
    one launch moves; the call before leaves other lists behind."""
    check_evict(1, dtype, [300, 170], hk, d, page, 64, 9)
    check_evict(2, dtype, [300, 70, 64, 0, 129, 90], hk, d, page, 64, 0, sums=sums)
    check_evict(3, dtype, [100, 71], hk, d, page, 1, 0, sums=zeros)


@pytest.mark.parametrize("sums", [zeros, falling])
def test_the_first_tokens_stay_in_many_long_rows(sums):
    """The same where one launch moves long lists (many sequences and heads)."""
    check_evict(4, BF, [700] * 40, 8, 16, 16, 400, 0)
    check_evict(5, BF, [700] * 40, 8, 16, 16, 400, 0, sums=sums)


@pytest.mark.parametrize("n", [900, 20011])
def test_the_first_tokens_stay_in_few_long_rows(n):
    """The same where the free places are filled by a launch of their own."""
    check_evict(6, BF, [n, 500], 2, 64, 16, 400, 0, sums=zeros)
    check_evict(7, BF, [n], 2, 64, 16, 400, 0, sums=falling)
