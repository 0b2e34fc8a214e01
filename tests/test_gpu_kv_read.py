"""iq_kv_read: cached tokens back as numbers, bit for bit."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import CODES, Pool, decode

pytestmark = pytest.mark.gpu
I8, F8, BF, FP, F32 = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32


def expected(pool, raw, b, tok, out):
    """[n, hk, d] of k and v: a code times its scale in fp32 (exact products
    rounded once), then rounded to the output's type from the fp32 product."""
    p, s = pool.where(b, tok)
    got = []
    for i in range(2):
        if pool.dtype in CODES:
            x = decode(raw[i][p, s], pool.dtype) * raw[2 + i][p, s // pool.block][..., None]
            got.append(torch.from_numpy(x).to(out))
        else:
            got.append(torch.from_numpy(raw[i][p, s]).view(pool.dtype).float().to(out))
    return got


@pytest.mark.parametrize("out", [F32, BF, FP])
@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("page,block,hk,d,order", [(16, 16, 2, 128, "slots"), (24, 3, 4, 64, "heads"), (1, 1, 3, 16, "padded"),
                                                   (100, 50, 1, 80, "slots"), (8, 2, 7, 256, "padded")])
def test_rows(dtype, out, page, block, hk, d, order):
    rng = np.random.default_rng(page + d)
    lens = [0, 1, page, 5 * page + 3, 37]
    width = max(-(-max(lens) // page), 6)
    pool = Pool(rng, len(lens), width, page, hk, d, dtype, block, order)
    pool.fill(rng, lens)
    raw = pool.raw()
    say("read", dtype, out, page, block, hk, d, order)
    for first in (None, [0, 0, page // 2, 7, 36]):
        at = first or [0] * len(lens)
        counts = [n - f for n, f in zip(lens, at)]
        T = sum(counts) + 3
        starts = torch.tensor(np.concatenate([[2], 2 + np.cumsum(counts)]), dtype=torch.int32).cuda()  # two rows before the first
        k, v = (torch.full((T, hk, d), -7.0, dtype=out, device="cuda") for _ in range(2))
        f = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        ops.kv_read(pool.cache, pool.table, starts, first=f, out=(k, v))
        only = ops.kv_read(pool.cache, pool.table, starts, T=T, first=f, dtype=out)
        torch.cuda.synchronize()
        assert torch.all(k[:2] == -7) and torch.all(k[-1:] == -7) and torch.all(v[:2] == -7) and torch.all(v[-1:] == -7)
        t = 2
        for b, m in enumerate(counts):
            ek, ev = expected(pool, raw, b, np.arange(at[b], at[b] + m), out)
            assert torch.equal(k[t:t + m].cpu(), ek) and torch.equal(v[t:t + m].cpu(), ev), b
            t += m
        assert torch.equal(only[0][2:t], k[2:t]) and torch.all(only[1][t:] == 0)
        v2 = torch.full_like(v, 3.0)
        ops.kv_read(pool.cache, pool.table, starts, first=f, out=(None, v2))
        torch.cuda.synchronize()
        assert torch.equal(v2[2:t], v[2:t]) and torch.all(v2[:2] == 3) and torch.all(v2[t:] == 3)


def test_tokens_that_are_not_there():
    rng = np.random.default_rng(4)
    pool = Pool(rng, 3, 2, 8, 2, 32, I8, 4)
    pool.fill(rng, [16, 16, 16])
    pool.table_np[1, 1] = pool.pages
    pool.table.copy_(torch.from_numpy(pool.table_np))
    first = torch.tensor([-2, 0, 12], dtype=torch.int32).cuda()
    starts = torch.tensor([0, 5, 15, 25], dtype=torch.int32).cuda()
    k, v = ops.kv_read(pool.cache, pool.table, starts, T=25, first=first)
    torch.cuda.synchronize()
    nan = torch.isnan(k).all(-1).all(-1).cpu().numpy()
    none = torch.isnan(k).any(-1).any(-1).cpu().numpy()
    want = np.zeros(25, bool)
    want[[0, 1]] = True                 # tokens -2, -1
    want[5 + 8:15] = True               # a page that is none
    want[15 + 4:] = True                # past the table
    assert np.array_equal(nan, want) and np.array_equal(none, want)
    assert np.array_equal(torch.isnan(v).all(-1).all(-1).cpu().numpy(), want)


def test_many_sequences_and_rows():
    """More sequences than lanes, empty ones among them, and rows enough for
    the larger workgroups."""
    rng = np.random.default_rng(6)
    B = 200
    pool = Pool(rng, B, 30, 8, 1, 16, F8, 8)
    lens = rng.integers(0, 240, B) * (rng.random(B) < 0.8)
    lens[:2] = 0
    pool.fill(rng, lens)
    raw = pool.raw()
    starts = np.concatenate([[0], np.cumsum(lens)])
    T = int(starts[-1])
    k, v = ops.kv_read(pool.cache, pool.table, torch.tensor(starts, dtype=torch.int32).cuda(), T=T, dtype=BF)
    want = [expected(pool, raw, b, np.arange(n), BF) for b, n in enumerate(lens)]
    assert T > 16384
    assert torch.equal(k.cpu(), torch.cat([w[0] for w in want])) and torch.equal(v.cpu(), torch.cat([w[1] for w in want]))
