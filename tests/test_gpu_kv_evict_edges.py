"""iq_kv_evict where no row has to move, and evictions one after the other."""
import numpy as np
import pytest
import torch

from infer_amd import ops
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


def test_the_newest_stay_over_several_evictions():
    """`recent` as large as the call before and the tokens added since allow:
    the newest tokens are kept every time, in their order.  A token's key holds
    its age (whole numbers up to 256 are exact in bf16)."""
    rng = np.random.default_rng(8)
    hk, d, page = 3, 16, 7
    cache = ops.alloc_kv(30, page, hk, d)
    table = torch.from_numpy(rng.permutation(30).astype(np.int32)).cuda()[None]
    order = table[0].long()

    def rows(n):
        t = torch.arange(n, device="cuda")
        return order[t // page], t % page

    def write(n0, n1, age):
        p, s = (x[n0:] for x in rows(n1))
        cache.k[p, s] = (age + torch.arange(n1 - n0, device="cuda")).to(BF)[:, None, None]
        cache.v[p, s] = 1.0

    n, age, known = 150, 150, 150
    write(0, n, 0)
    w = torch.from_numpy(rng.random((1, hk, 210)).astype(np.float32)).cuda()
    for budget, recent, added in ((120, 20, 9), (100, 29, 0), (60, 29, 30), (70, 59, 3), (61, 61, 25), (86, 80, 0), (30, 29, 5)):
        assert recent <= known
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        assert ops.kv_evict(cache, table, lens, w, budget, recent).item() == min(n, budget)
        if n > budget:
            n, known = budget, recent
        p, s = rows(n)
        ages = cache.k[p, s, :, 0].float().cpu().numpy()
        for h in range(hk):
            assert np.array_equal(ages[n - recent:, h], np.arange(age - recent, age)), (budget, recent, h)
            assert len(set(ages[:, h])) == n
        write(n, n + added, age)
        n, age, known = n + added, age + added, known + added
        w[:, :, :n] += torch.from_numpy(rng.random((1, hk, n)).astype(np.float32)).cuda()
