"""iq_kv_extend: the same tokens in one call and in several, and tokens whose
largest value is the one that made their block's scale."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import LARGEST, Pool

pytestmark = pytest.mark.gpu
I8, F8, BF, FP = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def starts_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()


def rows(rng, T, hk, d, spread=0.8):
    return (rng.standard_normal((T, hk, d)) * np.exp(spread * rng.standard_normal((T, 1, 1)))).astype(np.float32)


def same(got, want, what):
    for i, (g, w) in enumerate(zip(got, want)):
        assert np.array_equal(g, w, equal_nan=True), (what, ("k", "v", "k scales", "v scales")[i])


@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("single", [False, True])
def test_one_sequence_a_call(dtype, single):
    """A batch in one call, and each of its sequences in a call of its own: the
    same bytes, scales and q."""
    rng = np.random.default_rng(31)
    B, page, block, hq, hk, d = 90, 8, 4, 3, 2, 32
    pool = Pool(rng, B, 4, page, hk, d, dtype, block)
    lens = rng.integers(0, 20, B)
    lens[[5, 64]] = -3
    pool.fill(rng, lens)
    before = pool.raw()
    counts = np.ones(B, np.int64) if single else rng.integers(0, 14, B) * (rng.random(B) < 0.6)
    T, at = int(counts.sum()), np.concatenate([[0], np.cumsum(counts)])
    q, k, v = dev(rows(rng, T, hq, d)), dev(rows(rng, T, hk, d)), dev(rows(rng, T, hk, d))
    pos, fr = dev(rng.integers(0, 9000, T)), ops.rope_freqs(d, 1e6)
    w = dev(1 + 0.2 * rng.standard_normal(d), BF)
    n = dev(lens, torch.int32)
    say("extend", dtype, single, counts.tolist())
    got = ops.kv_extend(q, k, v, pos, fr, pool.cache, pool.table, n, starts=None if single else starts_of(counts), q_norm=w,
                        k_norm=w)
    torch.cuda.synchronize()
    want = pool.raw()
    pool.put(before)
    for b in range(B):
        i, j = int(at[b]), int(at[b + 1])
        if i == j:
            continue
        mine = ops.kv_extend(q[i:j], k[i:j], v[i:j], pos[i:j], fr, pool.cache, pool.table[b:b + 1], n[b:b + 1],
                             starts=None if single else starts_of([j - i]), q_norm=w, k_norm=w)
        assert torch.equal(mine, got[i:j]), b
    torch.cuda.synchronize()
    same(pool.raw(), want, "a call each")


@pytest.mark.parametrize("dtype", [I8, F8])
def test_the_largest_value_again(dtype):
    """Tokens of the same largest value one call each.  A scale is that value / Q
    to nearest, so that Q times it may be just below the value: the scale then
    doubles, once; what is stored stays within a step of it (e4m3: half a step of
    each value), and a block filled by one call keeps the first scale."""
    rng = np.random.default_rng(32)
    B, block, hk, d = 400, 8, 1, 32
    Q = LARGEST[dtype]
    x = rng.uniform(-1, 1, (B, block, hk, d)).astype(np.float32)
    x[..., 5] = np.where(rng.random((B, block, hk)) < 0.5, 1, -1)
    x *= np.exp2(rng.uniform(-20, 20, (B, 1, 1, 1))).astype(np.float32)
    x[0], x[1] = x[0] / np.abs(x[0]).max() * np.float32(0.3), x[1] / np.abs(x[1]).max()
    a = np.abs(x).max((2, 3))
    assert np.array_equal(a, np.broadcast_to(a[:, :1], a.shape))
    first = (a[:, 0] / np.float32(Q)).astype(np.float32)
    twice = Q * first.astype(np.float64) < a[:, 0]
    assert 0.2 * B < twice.sum() < 0.8 * B
    pools = [Pool(np.random.default_rng(33), B, 1, block, hk, d, dtype, block) for _ in range(2)]
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    for t in range(block):
        ops.kv_extend(None, dev(x[:, t]), dev(-x[:, t]), None, None, pools[0].cache, pools[0].table, n + t)
        s = pools[0].cache.k_scales.cpu().numpy()[pools[0].table_np[:, 0], 0, 0]
        assert np.array_equal(s, np.where(twice & (t > 0), 2 * first, first)), t
    one = dev(x.reshape(-1, hk, d))
    ops.kv_extend(None, one, -one, None, None, pools[1].cache, pools[1].table, n, starts=starts_of([block] * B))
    torch.cuda.synchronize()
    for i, pool in enumerate(pools):
        s = pool.cache.k_scales.cpu().numpy()[pool.table_np[:, 0], 0, 0].astype(np.float64)
        if i == 1:
            assert np.array_equal(s, first)
        raw = pool.raw()
        pool.raw = lambda: raw
        for b in range(B):
            K, V = pool.values(b, np.arange(block))
            # int8: the newest half a step; the older ones, halved once, a half step of half the scale before.
            # e4m3: half a step of the value, 2^-4, or of the numbers below its normal ones, 2^-10 of a scale, at
            # each of two roundings.  The quotient's own rounding: 2^-24 of at most Q steps.
            y = np.abs(x[b].astype(np.float64))
            half = s[b] * (0.5 + 0.25 * (i == 0)) if dtype == I8 else 2.0 ** -4 * y + 1.5 * 2.0 ** -10 * s[b]
            assert np.all(np.abs(K - x[b]) <= half + 2.0 ** -23 * Q * s[b]), (i, b)
            assert np.array_equal(V, -K)
