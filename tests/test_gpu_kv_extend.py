"""iq_kv_extend: new tokens behind what sequences have cached, in caches of
any type, against a plain form; bit for bit where nothing is normed or
turned."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import CODES, LARGEST, Pool, extend_plain, made_slack, norm_f64
from tests.kv_util import EPS32, HALF_STEP, rope_f64

pytestmark = pytest.mark.gpu
I8, F8, BF, FP = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).cuda()


def starts_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32).cuda()


def same(got, want, what):
    for i, (g, w) in enumerate(zip(got, want)):
        assert np.array_equal(g, w, equal_nan=True), (what, ("k", "v", "k scales", "v scales")[i])


def rows(rng, T, hk, d, spread=0.8):
    return (rng.standard_normal((T, hk, d)) * np.exp(spread * rng.standard_normal((T, 1, 1)))).astype(np.float32)


SHAPES = [  # page, block, hk, d, width, order
    (16, 16, 2, 128, 4, "slots"), (24, 8, 4, 64, 3, "heads"), (1, 1, 3, 16, 40, "slots"), (100, 25, 1, 80, 2, "padded"),
    (64, 64, 2, 256, 2, "slots"), (32, 2, 5, 96, 3, "padded"), (6, 3, 9, 32, 9, "heads"), (16, 1, 16, 48, 3, "slots"),
    (40, 40, 20, 16, 2, "slots"),
]


@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("page,block,hk,d,width,order", SHAPES)
def test_calls_in_a_row(dtype, page, block, hk, d, width, order):
    """Prompts, chunks and single tokens one after the other: every byte of the
    caches and every scale, touched or not."""
    rng = np.random.default_rng(page * 1000 + d)
    B = 5
    pool = Pool(rng, B, width, page, hk, d, dtype, block, order)
    raw = pool.raw()
    lens = np.zeros(B, np.int64)
    for it in range(9):
        single = it % 3 == 2
        counts = np.ones(B, np.int64) if single else rng.integers(0, max(2, pool.cap // 5), B)
        if it == 0:
            counts[:3] = [0, 1, block + 1]
        T = int(counts.sum())
        if T == 0:
            continue
        k, v = rows(rng, T, hk, d), rows(rng, T, hk, d)
        say("extend", dtype, page, block, hk, d, order, it, counts.tolist(), lens.tolist())
        ops.kv_extend(None, dev(k), dev(v), None, None, pool.cache, pool.table, dev(lens, torch.int32),
                      starts=None if single else starts_of(counts))
        torch.cuda.synchronize()
        extend_plain(pool, raw, k, lens, counts, 0)
        extend_plain(pool, raw, v, lens, counts, 1)
        same(pool.raw(), raw, it)
        lens = np.minimum(lens + counts, pool.cap)
    assert lens.max() > block


@pytest.mark.parametrize("dtype", [I8, F8])
def test_every_doubling(dtype):
    """A block whose tokens grow by 1, 2, 4, ... and odd factors: codes and
    scales, and every value within a step of the last scale (an e4m3 value within
    half a step of its own besides)."""
    rng = np.random.default_rng(5)
    pool = Pool(rng, 1, 1, 16, 2, 64, dtype, 16)
    raw, lens = pool.raw(), [0]
    size, xs = 1.0, []
    for t, f in enumerate((1.0, 1.0, 2.0, 4.0, 0.5, 1.0000001, 3.7, 1e3, 2.0, 1.0, 2.0 ** 20, 0.1, 1.5, 2.0, 1.0, 1.0)):
        size *= f
        x = rng.uniform(-1, 1, (1, 2, 64)).astype(np.float32)
        x[:, :, 3] = 1.0
        x *= np.float32(size)
        xs.append(x[0])
        ops.kv_extend(None, dev(x), dev(-x), None, None, pool.cache, pool.table, dev(np.array(lens), torch.int32))
        torch.cuda.synchronize()
        extend_plain(pool, raw, x, lens, [1], 0)
        extend_plain(pool, raw, -x, lens, [1], 1)
        same(pool.raw(), raw, t)
        lens[0] += 1
        K, V = pool.values(0, np.arange(lens[0]))
        s = pool.cache.k_scales[pool.table_np[0, 0], 0].cpu().numpy()[None, :, None].astype(np.float64)
        true = np.array(xs, np.float64)
        # int8: 1/2 + 1/4 + 1/8 ...; e4m3: half a step is 2^-4 of a value at each rounding, or 2^-10 of the
        # scale below its normal numbers (2^-6), halved with every doubling
        most = s if dtype == I8 else 2.0 ** -4 * np.abs(true) + 2 * 2.0 ** -10 * s
        assert np.all(np.abs(K - true) <= most * (1 + 1e-6))
        assert np.array_equal(V, -K)


def turned(x, w, eps, pos, freqs, rot):
    """Exact rows, and how far they may be off."""
    y = x.astype(np.float64)
    if w is not None:
        y = norm_f64(y, w, eps)
    slack = made_slack(y, w, rot // 2)
    return (rope_f64(y, pos, freqs, rot) if rot else y), slack


@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("hq,hk,d,rot,norms", [(28, 4, 128, 128, "qk"), (12, 2, 64, 64, ""), (5, 5, 96, 32, "k"),
                                               (40, 8, 16, 16, "q"), (6, 2, 256, 128, "qk"), (3, 1, 80, 80, "qk"),
                                               (17, 1, 32, 0, "qk")])
def test_norms_and_rotation(dtype, hq, hk, d, rot, norms):
    rng = np.random.default_rng(d + hq)
    B, page, block = 4, 16, 8
    pool = Pool(rng, B, 5, page, hk, d, dtype, block)
    lens = np.array([0, 13, 31, 70])
    pool.fill(rng, lens)
    for counts in ([1, 1, 1, 1], [19, 0, 7, 9]):
        T = sum(counts)
        q, k, v = rows(rng, T, hq, d), rows(rng, T, hk, d) * 3, rows(rng, T, hk, d)
        pos = rng.integers(0, 131072, T)
        freqs = 1e6 ** (-2.0 * np.arange(rot // 2) / max(rot, 1))
        w = {n: torch.from_numpy(1 + 0.3 * rng.standard_normal(d)).to(BF) for n in "qk"}
        eps = 1e-6
        got = ops.kv_extend(dev(q), dev(k), dev(v), dev(pos) if rot else None, dev(freqs) if rot else None, pool.cache,
                            pool.table, dev(lens, torch.int32), starts=starts_of(counts) if T != B else None,
                            q_norm=w["q"].cuda() if "q" in norms else None, k_norm=w["k"].cuda() if "k" in norms else None,
                            eps=eps)
        torch.cuda.synchronize()
        wf = {n: w[n].double().numpy() if n in norms else None for n in "qk"}
        ref, slack = turned(q, wf["q"], eps, pos, freqs, rot)
        assert np.all(np.abs(got.cpu().double().numpy() - ref) <= slack)
        ref, slack = turned(k, wf["k"], eps, pos, freqs, rot)
        t = 0
        for b, m in enumerate(counts):
            if m == 0:
                continue
            tok = np.arange(lens[b], lens[b] + m)
            K, V = pool.values(b, tok)
            for x, y, sl, sc in ((K, ref[t:t + m], slack[t:t + m], pool.cache.k_scales),
                                 (V, v[t:t + m].astype(np.float64), 0.0, pool.cache.v_scales)):
                if dtype in CODES:
                    p, s = pool.where(b, tok)
                    step = sc.cpu().double().numpy()[p, s // block][..., None]
                    # half a step (of the scale; of the value, or of e4m3's subnormals), the division's rounding
                    # and the largest value's own when it makes the scale
                    half = 0.5 * step if dtype == I8 else np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * step)
                    most = half + sl + 4 * EPS32 * (np.abs(y) + step * (LARGEST[dtype] if dtype == I8 else 0))
                    if dtype == F8:
                        most = most * (1 + 2.0 ** -3)  # (a value next to a power of two may round with the larger step)
                else:
                    most = HALF_STEP[dtype] * (np.abs(y) + sl) + sl + (2.0 ** -25 if dtype == FP else 0)
                assert np.all(np.abs(x - y) <= most), (b, np.abs(x - y).max())
            t += m
        lens = lens + np.array(counts)


@pytest.mark.parametrize("dtype", [I8, F8, BF])
def test_rows_without_a_place(dtype):
    """Idle sequences, full ones, pages that are not there, rows of no
    sequence, tokens past the table: nothing else changes, and q is made."""
    rng = np.random.default_rng(8)
    B, page, block, hk, d = 7, 16, 4, 2, 32
    pool = Pool(rng, B, 3, page, hk, d, dtype, block)
    lens = np.array([-1, 48, 49, 30, 10, -2 ** 31, 2 ** 31 - 1])
    pool.table_np[3, 2], pool.table_np[4, 0], pool.table_np[4, 1] = -1, pool.pages, -2 ** 31
    pool.table.copy_(torch.from_numpy(pool.table_np))
    raw = pool.raw()
    counts = [3, 2, 2, 9, 12, 1, 4]
    T = sum(counts) + 5  # five rows behind the last sequence
    k, v, q = rows(rng, T, hk, d), rows(rng, T, hk, d), rows(rng, T, 3, d)
    for c, n in ((counts, T), ([1] * B, B)):
        got = ops.kv_extend(dev(q[:n]), dev(k[:n]), dev(v[:n]), None, None, pool.cache, pool.table, dev(lens, torch.int32),
                            starts=starts_of(c) if n == T else None)
        torch.cuda.synchronize()
        assert np.array_equal(got.cpu().numpy(), q[:n])
        extend_plain(pool, raw, k, lens, c, 0)
        extend_plain(pool, raw, v, lens, c, 1)
        same(pool.raw(), raw, n)


@pytest.mark.parametrize("dtype", [I8, F8])
def test_values_at_the_edges(dtype):
    """Zeros, subnormals, fp32's largest, infinities and NaN, and a block that
    starts anew after them."""
    rng = np.random.default_rng(9)
    hk, d, block = 2, 16, 4
    pool = Pool(rng, 1, 4, 8, hk, d, dtype, block)
    raw, n = pool.raw(), 0
    big = np.float32(3.4028235e38)
    for x in (0.0, 1e-45, 1e-40, 1e-38, 1e-30, 1.0, big, big, 0.0, 0.0, float("nan"), 1.0, 1.0, float("inf"), 2.0, -0.0,
              0.0, -float("inf"), 5.0, 6.0):
        row = np.zeros((1, hk, d), np.float32)
        row[:, 0, 5], row[:, 1, 7] = x, 1.0
        row[:, :, 2] = np.float32(x) * np.float32(0.3) if np.isfinite(x) else 0.3
        ops.kv_extend(None, dev(row), dev(-row), None, None, pool.cache, pool.table, dev(np.array([n]), torch.int32))
        torch.cuda.synchronize()
        extend_plain(pool, raw, row, [n], [1], 0)
        extend_plain(pool, raw, -row, [n], [1], 1)
        same(pool.raw(), raw, (n, x))
        n += 1
    K, _ = pool.values(0, np.arange(n))
    assert np.all(np.isnan(K[8:12, 0])) and np.all(np.isfinite(K[8:12, 1])) and np.all(np.isfinite(K[:8]))
    # the second block again from its first token, as after a shorter length: finite once more
    row = rows(rng, 2, hk, d)
    ops.kv_extend(None, dev(row), dev(row), None, None, pool.cache, pool.table, dev(np.array([8]), torch.int32),
                  starts=starts_of([2]))
    torch.cuda.synchronize()
    assert np.all(np.isfinite(pool.values(0, np.arange(8, 10))[0]))


def test_norm_of_extreme_rows():
    """Squares past fp32's range on either side."""
    d = 64
    pool = Pool(np.random.default_rng(1), 4, 1, 16, 1, d, BF)
    x = np.random.default_rng(2).standard_normal((4, 1, d)).astype(np.float32)
    x *= np.array([1e30, 1e-30, 1.0, 1e37], np.float32)[:, None, None]
    w = torch.ones(d, dtype=BF).cuda()
    for eps in (0.0, 1e-6):
        q = ops.kv_extend(dev(x), dev(x), dev(x), None, None, pool.cache, pool.table, dev(np.zeros(4), torch.int32),
                          q_norm=w, eps=eps).cpu().double().numpy()
        ref = norm_f64(x.astype(np.float64), 1.0, eps)
        assert np.all(np.abs(q - ref) <= 2 * EPS32 * np.abs(ref) + 1e-45)


@pytest.mark.parametrize("dtype", [I8, BF])
def test_many_sequences(dtype):
    """More sequences than a wave has lanes, with gaps, in one call; and the
    same tokens one sequence a call."""
    rng = np.random.default_rng(10)
    B, page, block, hk, d = 300, 8, 4, 2, 32
    pool = Pool(rng, B, 4, page, hk, d, dtype, block)
    lens = rng.integers(0, 20, B)
    lens[[5, 64, 299]] = -3
    pool.fill(rng, lens)
    raw = pool.raw()
    counts = rng.integers(0, 14, B) * (rng.random(B) < 0.6)
    T = int(counts.sum())
    k, v = rows(rng, T, hk, d), rows(rng, T, hk, d)
    ops.kv_extend(None, dev(k), dev(v), None, None, pool.cache, pool.table, dev(lens, torch.int32), starts=starts_of(counts))
    torch.cuda.synchronize()
    extend_plain(pool, raw, k, lens, counts, 0)
    extend_plain(pool, raw, v, lens, counts, 1)
    same(pool.raw(), raw, "many")


def test_in_place_and_on_another_stream():
    rng = np.random.default_rng(11)
    pool = Pool(rng, 3, 2, 16, 2, 64, I8, 8)
    lens = dev(np.array([3, 9, 20]), torch.int32)
    q, k = dev(rows(rng, 3, 4, 64)), dev(rows(rng, 3, 2, 64))
    fr, pos = ops.rope_freqs(64, 1e6), dev(np.array([3, 9, 20]))
    pool.fill(rng, [3, 9, 20])
    before = pool.raw()
    want = ops.kv_extend(q, k, k, pos, fr, pool.cache, pool.table, lens)
    torch.cuda.synchronize()
    raw = pool.raw()
    pool.put(before)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ops.kv_extend(q, k, k, pos, fr, pool.cache, pool.table, lens, q_out=q, stream=s)
    torch.cuda.synchronize()
    assert got is q and torch.equal(got, want)
    same(pool.raw(), raw, "stream")


@pytest.mark.parametrize("dtype", [F8, BF])
def test_most_sequences_and_a_part_of_a_table(dtype):
    """1024 sequences, a token each; the table is a slice of a wider one."""
    rng = np.random.default_rng(12)
    B, page, block, hk, d = 1024, 4, 2, 1, 16
    pool = Pool(rng, B, 3, page, hk, d, dtype, block)
    lens = rng.integers(-1, 13, B)
    pool.fill(rng, np.minimum(lens, 12))
    raw = pool.raw()
    wide = torch.full((B, 7), -9, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = pool.table
    k, v = rows(rng, B, hk, d), rows(rng, B, hk, d)
    q = rows(rng, B, 3, d)
    got = ops.kv_extend(dev(q), dev(k), dev(v), None, None, pool.cache, wide[:, 2:5], dev(lens, torch.int32))
    torch.cuda.synchronize()
    extend_plain(pool, raw, k, lens, [1] * B, 0)
    extend_plain(pool, raw, v, lens, [1] * B, 1)
    same(pool.raw(), raw, "most")
    assert np.array_equal(got.cpu().numpy(), q)


def test_unaligned_inputs():
    """q, k, v, norms and q_out at any multiple of their own size."""
    rng = np.random.default_rng(13)
    B, hq, hk, d = 3, 6, 2, 64
    fr, pos = ops.rope_freqs(d, 1e6), dev(np.array([5, 6, 7]))
    got = []
    for off in (0, 1, 3):
        for starts in (None, torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda()):
            rng = np.random.default_rng(13)
            pool = Pool(rng, B, 2, 16, hk, d, I8, 8)
            pool.fill(rng, [5, 6, 7])

            def at(shape):
                x = torch.empty(int(np.prod(shape)) + off, device="cuda")[off:].view(shape)
                return x.copy_(dev(rows(rng, *shape)))
            q, k, v = at((B, hq, d)), at((B, hk, d)), at((B, hk, d))
            w = torch.empty(d + off, dtype=BF, device="cuda")[off:].copy_(dev(1 + 0.1 * rng.standard_normal(d)))
            out = torch.empty(B * hq * d + off, device="cuda")[off:].view(B, hq, d)
            ops.kv_extend(q, k, v, pos, fr, pool.cache, pool.table, dev(np.array([5, 6, 7]), torch.int32), starts=starts,
                          q_norm=w, k_norm=w, q_out=out)
            torch.cuda.synchronize()
            got.append([out.cpu().numpy(), *pool.raw()])
    for g in got[1:]:
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(g, got[0]))


@pytest.mark.parametrize("dtype", [I8, BF])
def test_more_workgroups_than_a_launch_has(dtype):
    """2^24 tokens and more, in one call of several launches (the last of the
    cache's part and the first of the queries' in one)."""
    T, d, page = 2 ** 24 + 1001, 16, 1024
    pages = -(-T // page)
    cache = ops.alloc_kv(pages, page, 1, d, dtype, block=1 if dtype == I8 else None)
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda").view(1, pages)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, 1, d, device="cuda", generator=gen)
    starts, zero = torch.tensor([0, T], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    say("extend", dtype, T)
    got = ops.kv_extend(x, x, x, None, None, cache, table, zero, starts=starts)
    assert torch.equal(got, x)
    del got
    k, v = ops.kv_read(cache, table, starts, T=T)
    assert torch.equal(k, v)
    if dtype == I8:
        # half a step, and the roundings of the scale, the quotient and the product (each of at most 127 steps)
        step = x.abs().amax((1, 2), keepdim=True) / 127
        assert torch.all((k - x).abs() <= (0.5 + 4 * 127 * EPS32) * step)
    else:
        assert torch.equal(k, x.to(BF).float())
