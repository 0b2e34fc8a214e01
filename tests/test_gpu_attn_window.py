"""iq_attn_decode_window: attention over 8-bit caches, and under a window with
first tokens that stay visible over caches of any type, against 64 bits."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import CODES, Pool
from tests.kv_util import EPS32, attn_f64, attn_rel

pytestmark = pytest.mark.gpu
I8, F8, BF, FP = torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16


def rel(d, ck):
    """attn_rel, and three more roundings of a score (a key's scale times the
    call's, the product with it) and two of a weight (a value's scale), each
    half a step."""
    return attn_rel(d, ck) + 6 * EPS32 * ck + 4 * EPS32


def seen(n, window, sinks):
    t = np.arange(n)
    return t if window == 0 else t[(t >= n - window) | (t < sinks)]


def check(pool, q, lens, got, window=0, sinks=0, scale=None):
    d = pool.d
    K, V = [np.zeros((0,))] * 2
    for b, n in enumerate(lens):
        t = seen(max(n, 0), window, sinks)
        K, V = pool.values(b, t) if n > 0 else (np.zeros((0, pool.hk, d)),) * 2
        ref, _, ck, cv = attn_f64(q[b].astype(np.float64), K, V, d ** -0.5 if scale is None else scale)
        # (a weight below fp32's normal numbers, 2^-126, may become 0: it is then off by itself, which
        # moves the sum over tokens of p |v| by at most 2^-126 times the sum of |v|)
        g = q.shape[1] // pool.hk
        lost = 2.0 ** -126 * np.repeat(np.abs(V).sum(0), g, 0)
        err, most = np.abs(got[b].astype(np.float64) - ref), rel(d, ck)[:, None] * cv + lost
        assert np.all(err <= most), (b, n, float((err / np.maximum(most, 1e-300)).max()))


def run(rng, lens, hq, hk, d, page, block, dtype, order="slots", window=0, sinks=0, sd=1.0, width=None):
    width = max(1, -(-max(lens) // page)) if width is None else width
    pool = Pool(rng, len(lens), width, page, hk, d, dtype, block, order)
    pool.fill(rng, lens)
    q = (rng.standard_normal((len(lens), hq, d)) * sd).astype(np.float32)
    out = torch.full((len(lens), hq, d), -5.0, device="cuda")
    say("attn", dtype, lens[:8], hq, hk, d, page, block, order, window, sinks)
    ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, torch.tensor(lens, dtype=torch.int32).cuda(),
                    out=out, window=window, sinks=sinks)
    torch.cuda.synchronize()
    check(pool, q, lens, out.cpu().numpy(), window, sinks)
    return pool, q, out


HEADS = [(28, 4, 128), (12, 2, 128), (16, 16, 64), (3, 3, 32), (2, 1, 16), (5, 1, 80), (40, 2, 96), (8, 4, 256),
         (24, 1, 48), (34, 2, 240)]


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_heads(dtype, hq, hk, d):
    rng = np.random.default_rng(hq * d)
    run(rng, [1, 0, 17, 32, 33, 200, 129, 2], hq, hk, d, 16, 16, dtype)


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("page,block,order", [(16, 16, "heads"), (24, 8, "padded"), (1, 1, "slots"), (100, 25, "slots"),
                                              (7, 7, "heads"), (64, 32, "padded"), (64, 64, "slots"), (33, 3, "slots"),
                                              (5, 1, "heads")])
def test_pages_blocks_and_orders(dtype, page, block, order):
    rng = np.random.default_rng(page)
    run(rng, [300, 31, 1, 64, 99], 6, 3, 64, page, block, dtype, order)


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("B,n,hq,hk,d", [(1, 9001, 14, 2, 128), (3, 4099, 8, 8, 64), (40, 700, 4, 2, 32), (2, 5000, 6, 1, 256)])
def test_long_and_many(dtype, B, n, hq, hk, d):
    rng = np.random.default_rng(n)
    lens = [n] + rng.integers(0, n + 1, B - 1).tolist()
    run(rng, lens, hq, hk, d, 16, 8, dtype)


@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 17), (100, 0), (64, 64), (299, 1), (300, 1),
                                          (1000, 5), (5, 1000), (2 ** 40, 2 ** 40), (1, 298)])
def test_windows(dtype, window, sinks):
    rng = np.random.default_rng(window % 1000 + sinks % 1000)
    run(rng, [300, 0, 1, 33, 150, 34, 299, 18], 6, 2, 64, 16, 16, dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [I8, F8, BF, FP])
@pytest.mark.parametrize("hq,hk,d", [(28, 4, 128), (16, 16, 32), (20, 1, 96), (4, 2, 256)])
def test_long_windows(dtype, hq, hk, d):
    rng = np.random.default_rng(d)
    run(rng, [6001, 2, 1500, 6000, 3333], hq, hk, d, 24, 24, dtype, window=1501, sinks=9)


@pytest.mark.parametrize("dtype", [I8, BF])
def test_pages_outside_the_window_may_go(dtype):
    """Freed pages, with ids that are none, and tokens of NaN outside the
    window: the same answer."""
    rng = np.random.default_rng(3)
    window, sinks, page = 40, 5, 16
    lens = [200, 55, 130]
    pool, q, out = run(rng, lens, 4, 2, 64, page, 16, dtype, window=window, sinks=sinks)
    raw = pool.raw()
    for b, n in enumerate(lens):
        keep = set((seen(n, window, sinks) // page).tolist())
        for p in range(pool.table_np.shape[1]):
            if p not in keep:
                for a in raw:  # 8 bits: scales of NaN; 16: values of NaN
                    a[pool.table_np[b, p]] = np.nan if a.dtype == np.float32 else -1 if a.dtype == np.int16 else 255
                pool.table_np[b, p] = (-1, pool.pages, 2 ** 31 - 1)[p % 3]
    pool.put(raw)
    table = torch.from_numpy(pool.table_np).cuda()
    again = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, table, torch.tensor(lens, dtype=torch.int32).cuda(),
                            window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [I8, F8])
def test_what_is_not_a_number(dtype):
    """NaN scales of keys and values, pages that are not there, lengths that
    are none; other heads and sequences keep their answers."""
    rng = np.random.default_rng(4)
    lens = [50, 50, 50, 50, -1, 65, -2 ** 31, 40]
    pool = Pool(rng, 8, 4, 16, 2, 64, dtype, 8)
    pool.fill(rng, [max(0, min(n, 64)) for n in lens])
    q = rng.standard_normal((8, 6, 64)).astype(np.float32)
    q[7, 1, 3] = np.nan
    t = pool.table_np
    raw = pool.raw()
    raw[2][t[0, 1], 1, 0] = np.nan       # a key's block of sequence 0, head 0
    raw[3][t[1, 2], 0, 1] = np.nan       # a value's of sequence 1, head 1
    raw[3][t[2, 3], 0, 1] = np.inf       # the block of tokens 48, 49
    pool.put(raw)
    t[3, 2] = -1
    out = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, torch.from_numpy(t).cuda(),
                          torch.tensor(lens, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.isnan(got[0, :3]).all() and np.isfinite(got[0, 3:]).all()
    assert np.isnan(got[1, 3:]).all() and np.isfinite(got[1, :3]).all()
    assert not np.isfinite(got[2, 3:]).any() and np.isfinite(got[2, :3]).all()
    assert np.isnan(got[3:7]).all()
    assert np.isnan(got[7, 1]).all() and np.isfinite(got[7, [0, 2, 3, 4, 5]]).all()


@pytest.mark.parametrize("dtype", [I8, F8])
def test_scales_of_any_size(dtype):
    """Values of 1e-24 to 1e33 (a value's scale of 2^-86 or more: the third bf16
    term of a weight of 2^-24 times it is a normal number), keys large enough that one token
    takes all, and blocks of zeros."""
    rng = np.random.default_rng(12)
    lens = [90, 90, 90, 70]
    pool = Pool(rng, 4, 6, 16, 1, 32, dtype, 4)
    pool.fill(rng, lens)
    raw = pool.raw()
    t = pool.table_np
    raw[3][t[0]] *= np.float32(1e-24)
    raw[3][t[1]] *= np.float32(1e33)
    raw[2][t[2]] *= np.float32(300.0)
    raw[3][t[3, :2]] = 0.0
    raw[2][t[3, 1:3]] = 0.0
    pool.put(raw)
    q = rng.standard_normal((4, 3, 32)).astype(np.float32)
    out = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, torch.tensor(lens, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    check(pool, q, lens, out.cpu().numpy())


def test_window_as_the_whole():
    """A window that covers every token gives what no window gives, over 16
    bits bit for bit what iq_attn_decode gives."""
    rng = np.random.default_rng(2)
    for dtype in (BF, FP, I8, F8):
        pool, q, out = run(rng, [700, 33, 5], 12, 2, 128, 16, 16, dtype)
        lens = torch.tensor([700, 33, 5], dtype=torch.int32).cuda()
        for window, sinks in ((704, 0), (700, 4), (2 ** 62, 3), (1, 703), (2 ** 70, 2 ** 64)):
            again = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, lens, window=window, sinks=sinks)
            torch.cuda.synchronize()
            assert torch.equal(again, out), (dtype, window, sinks)


def test_long_rows_past_32_bits():
    """A pool whose last pages lie past 2^32 bytes (8-bit codes)."""
    page, hk, d = 64, 4, 128
    pages = (2 ** 32 + 2 ** 28) // (page * hk * d)
    k = torch.zeros(pages, page, hk, d, dtype=I8, device="cuda")
    cache = ops.KvCache(k, k, *[torch.zeros(pages, 1, hk, device="cuda") for _ in range(2)])
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32).cuda()
    x = torch.randn(3 * page, hk, d, device="cuda")
    zero, starts = torch.zeros(1, dtype=torch.int32).cuda(), torch.tensor([0, 3 * page], dtype=torch.int32).cuda()
    ops.kv_extend(None, x, x, None, None, cache, table, zero, starts=starts)
    rk, rv = ops.kv_read(cache, table, starts, T=3 * page)
    torch.cuda.synchronize()
    assert torch.equal(rk, rv)
    s = cache.k_scales[table[0].long()].repeat_interleave(page, 1).view(-1, hk, 1)
    assert torch.all((rk - x).abs() <= 0.5 * s * 1.0001)
    q = torch.randn(1, 8, d, device="cuda")
    out = ops.attn_decode(q, cache, table, torch.tensor([3 * page], dtype=torch.int32).cuda())
    got, K = out.cpu().numpy(), rk.double().cpu().numpy()
    ref, _, ck, cv = attn_f64(q[0].double().cpu().numpy(), K, K, d ** -0.5)
    assert np.all(np.abs(got[0] - ref) <= rel(d, ck)[:, None] * cv)


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2)])
@pytest.mark.parametrize("dtype", [I8, F8, FP])
def test_most_sequences(dtype, window, sinks):
    """1024 sequences of a few tokens, in a slice of a wider table."""
    rng = np.random.default_rng(21)
    B, hq, hk, d, page = 1024, 3, 1, 16, 8
    lens = rng.integers(0, 41, B)
    pool = Pool(rng, B, 5, page, hk, d, dtype, 4)
    pool.fill(rng, lens)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    wide = torch.full((B, 9), -3, dtype=torch.int32, device="cuda")
    wide[:, 1:6] = pool.table
    out = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, wide[:, 1:6], torch.from_numpy(lens).int().cuda(),
                          window=window, sinks=sinks)
    torch.cuda.synchronize()
    got, raw = out.cpu().numpy(), pool.raw()
    pool.raw = lambda: raw
    check(pool, q, lens, got, window, sinks)


@pytest.mark.parametrize("dtype", [I8, F8])
def test_scores_past_fp32(dtype):
    """Keys whose scores lie below fp32's range weigh nothing, a head with no
    others gives zeros; scores above it give NaN."""
    B, d, n = 4, 32, 70
    pool = Pool(np.random.default_rng(5), B, 5, 16, 1, d, dtype, 2)
    pool.fill(np.random.default_rng(6), [n] * B)
    raw, t = pool.raw(), pool.table_np
    q = np.zeros((B, 2, d), np.float32)
    q[:, :, 0], q[:, 1, 0] = 4.0, -4.0
    ones = 127 if dtype == I8 else 0x7e  # the largest code
    raw[0][:] = 0
    raw[0][..., 0] = ones
    raw[2][:] = 0.01
    raw[2][t[0, :4]] = 3e38      # sequence 0: 64 huge keys, then 6 of its own size
    raw[2][t[1]] = 3e38          # 1: all huge
    raw[2][t[2, 2], 3] = 3e38    # 2: two tokens
    pool.put(raw)
    out = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, torch.tensor([n] * B, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert np.isnan(got[:3, 0]).all() and np.isfinite(got[3]).all()  # +inf
    V = [pool.values(b, np.arange(n))[1][:, 0] for b in range(B)]
    keep = [np.arange(n) >= 64, np.zeros(n, bool), ~((np.arange(n) >= 38) & (np.arange(n) < 40)), np.ones(n, bool)]
    for b in range(B):
        w = V[b][keep[b]]
        want = w.mean(0) if len(w) else np.zeros(d)  # (equal keys)
        most = (64 * EPS32 + 4 * EPS32) * np.abs(w).mean(0) if len(w) else 0.0
        assert np.all(np.abs(got[b, 1] - want) <= most), b


def test_two_streams_at_once():
    """Calls on two streams that overlap: each its own workspace, each the
    answer that it has alone."""
    rng = np.random.default_rng(7)
    jobs = []
    for dtype in (I8, F8):
        lens = [3000, 1, 700, 2500]
        pool = Pool(rng, 4, 188, 16, 2, 128, dtype, 16)
        pool.fill(rng, lens)
        q = torch.from_numpy(rng.standard_normal((4, 12, 128)).astype(np.float32)).cuda()
        n = torch.tensor(lens, dtype=torch.int32).cuda()
        jobs.append((pool, q, n, ops.attn_decode(q, pool.cache, pool.table, n).clone(),
                     [torch.empty_like(q) for _ in range(20)], torch.cuda.Stream()))
    for j in jobs:
        ops.init(0, j[5])
    torch.cuda.synchronize()
    for i in range(20):
        for pool, q, n, _, outs, s in jobs:
            ops.attn_decode(q, pool.cache, pool.table, n, out=outs[i], stream=s)
    torch.cuda.synchronize()
    for _, _, _, want, outs, _ in jobs:
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype,B,hq,hk,d,window", [(I8, 150, 3, 1, 128, 0), (F8, 97, 4, 2, 64, 0), (BF, 200, 2, 1, 128, 500),
                                                    (FP, 130, 4, 1, 64, 0), (I8, 300, 2, 2, 32, 77)])
def test_long_rows_of_more_sequences_than_lanes(dtype, B, hq, hk, d, window):
    """Over 64 sequences, some of several chunks."""
    rng = np.random.default_rng(B)
    lens = (np.exp(rng.uniform(0, np.log(900), B))).astype(np.int64)
    lens[[0, 70, B - 1]] = [900, 871, 899]
    lens[[3, 66]] = 0
    pool = Pool(rng, B, 57, 16, hk, d, dtype, 16)
    pool.fill(rng, lens)
    q = rng.standard_normal((B, hq, d)).astype(np.float32)
    out = ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, torch.from_numpy(lens).int().cuda(),
                          window=window, sinks=5)
    torch.cuda.synchronize()
    got, raw = out.cpu().numpy(), pool.raw()
    pool.raw = lambda: raw
    check(pool, q, lens, got, window, 5)


@pytest.mark.parametrize("dtype,B,hq,hk,d,tiles", [(I8, 1, 6, 1, 128, 12), (I8, 1, 6, 1, 128, 13), (F8, 2, 4, 2, 256, 8),
                                                   (F8, 2, 4, 2, 256, 9), (I8, 43, 6, 3, 128, 16), (I8, 43, 6, 3, 128, 17),
                                                   (F8, 300, 2, 1, 64, 32), (F8, 300, 2, 1, 64, 33), (I8, 70, 4, 4, 256, 32),
                                                   (BF, 3, 4, 2, 64, 12), (FP, 2, 4, 1, 128, 8), (BF, 65, 8, 2, 80, 16),
                                                   (BF, 70, 4, 4, 256, 32), (FP, 70, 4, 4, 256, 33), (F8, 9, 80, 2, 32, 12)])
def test_sequences_whole_and_split(dtype, B, hq, hk, d, tiles):
    """Tables of as many tiles of 32 tokens as one workgroup takes in a row, and
    of one more; of 16-bit caches, windows of them in longer tables."""
    rng = np.random.default_rng(B + tiles)
    n = tiles * 32
    if dtype in CODES:
        lens = [n, 0, 1, n - 1, 33][:B] + rng.integers(0, n + 1, max(0, B - 5)).tolist()
        run(rng, lens, hq, hk, d, 32, 32, dtype)
    else:
        lens = [n + 70, 0, n, n + 1, 5][:B] + rng.integers(0, n + 71, max(0, B - 5)).tolist()
        run(rng, lens, hq, hk, d, 32, None, dtype, window=n - 3, sinks=3)


@pytest.mark.parametrize("dtype,window", [(I8, 0), (BF, 300)])
def test_lengths_out_of_range_of_whole_sequences(dtype, window):
    rng = np.random.default_rng(8)
    lens = [40, 0, 200, 320, 7]
    pool, q, out = run(rng, lens, 4, 2, 64, 16, 16, dtype, window=window, width=21)
    bad = [40, -1, 200, 337, 2 ** 31 - 1]
    got = torch.empty_like(out)
    ops.attn_decode(torch.from_numpy(q).cuda(), pool.cache, pool.table, torch.tensor(bad, dtype=torch.int32).cuda(), out=got, window=window)
    for b in range(5):
        if bad[b] == lens[b]:
            assert torch.equal(got[b], out[b])
        else:
            assert torch.isnan(got[b]).all()
