"""Scales of 8-bit caches that are no numbers, in iq_attn_decode_window."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import Pool

pytestmark = pytest.mark.gpu
I8, F8 = torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("n,width,window", [(50, 4, 0), (50, 100, 0), (1500, 94, 0), (700, 94, 90)])
@pytest.mark.parametrize("side", ["k", "v"])
def test_scales_that_are_no_numbers(dtype, bad, n, width, window, side):
    """One block's scale infinite or NaN, keys that point with q and against it:
    the heads that read the block give NaN, the others what they gave.  In one
    workgroup and in chunks, under a window and not."""
    rng = np.random.default_rng(n)
    pool = Pool(rng, 2, width, 16, 2, 64, dtype, 8)
    pool.fill(rng, [n, n])
    q = rng.standard_normal((2, 8, 64)).astype(np.float32)
    raw, t = pool.raw(), pool.table_np
    tok = n - 20  # seen under the window too
    page, slot = t[0, tok // 16], tok % 16
    first = slot // 8 * 8
    codes = raw[0][page, first:first + 8, 1]
    codes[:] = 0
    # key/value head 1's query heads 4..7: the block's products all positive, all negative, of both signs, all zero
    codes[:, 0] = 8 if dtype == I8 else 0x38  # e4m3: 1
    codes[:, 1] = np.where(np.arange(8) % 2, 8, 0xf8) if dtype == I8 else np.where(np.arange(8) % 2, 0x38, 0xb8)
    q[0, 4:8, :] = 0
    q[0, 4, 0], q[0, 5, 0], q[0, 6, 1] = 2.0, -2.0, 2.0
    pool.put(raw)
    lens = torch.tensor([n, n], dtype=torch.int32).cuda()
    qd = torch.from_numpy(q).cuda()
    want = ops.attn_decode(qd, pool.cache, pool.table, lens, window=window).cpu().numpy()
    assert np.isfinite(want).all()
    raw[2 if side == "k" else 3][page, slot // 8, 1] = bad
    pool.put(raw)
    say("attn", dtype, bad, n, width, window, side)
    got = ops.attn_decode(qd, pool.cache, pool.table, lens, window=window).cpu().numpy()
    assert np.isnan(got[0, 4:]).all()
    assert np.array_equal(got[0, :4], want[0, :4]) and np.array_equal(got[1], want[1])
