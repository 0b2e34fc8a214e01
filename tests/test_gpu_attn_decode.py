"""iq_attn_decode against a plain 64-bit form: types, grouped heads, page
sizes and memory orders, lengths around every tile and split border, rows
that are empty or refused, and the weights it accumulates."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv_util import EPS32, Paged, attn_f64, attn_rel

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def run_case(seed, dtype, hq, hk, d, page, lens, order="slots", weights=False, scale=None, qsd=1.0, wide=0):
    rng = np.random.default_rng(seed)
    say("attn", seed, dtype, hq, hk, d, page, lens[:6], len(lens), order, weights)
    pg = Paged(rng, lens, hk, d, page, dtype, order)
    B = len(lens)
    q = (rng.standard_normal((B, hq, d)) * qsd).astype(np.float32)
    qd = torch.from_numpy(q).cuda()
    table = pg.table
    if wide:  # a table of more columns, the ones past a sequence's pages holding anything
        table = torch.full((B, pg.width + wide), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
        table[:, :pg.width] = pg.table
    cap = table.shape[1] * page
    w = w0 = None
    if weights:
        w0 = rng.standard_normal((B, hk, cap + 3)).astype(np.float32)
        w = torch.from_numpy(w0).cuda()
    out = torch.full_like(qd, 777.0)
    ops.attn_decode(qd, pg.cache, table, pg.lens_t, out=out, weights=w, scale=scale)
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    gw = None if w is None else w.cpu().numpy()
    sc = d ** -0.5 if scale is None else scale
    worst = 0.0
    for b, n in enumerate(lens):
        ref, p, ck, cv = attn_f64(q[b].astype(np.float64), pg.K[b].double().numpy(), pg.V[b].double().numpy(), sc)
        if n == 0:
            assert np.all(got[b] == 0.0), b
        else:
            rel = attn_rel(d, ck)[:, None]
            bound = rel * cv + 1e-30
            r = np.abs(got[b] - ref) / bound
            worst = max(worst, float(r.max()))
            assert np.all(r <= 1.0), (b, n, float(r.max()))
        if weights:
            g = hq // hk
            ref_w = p.reshape(hk, g, n).sum(1)
            bound = (attn_rel(d, ck).reshape(hk, g, 1) * p.reshape(hk, g, n)).sum(1)
            bound = bound + EPS32 * np.abs(w0[b, :, :n] + ref_w) + g * EPS32 * ref_w + 1e-30
            err = np.abs(gw[b, :, :n].astype(np.float64) - w0[b, :, :n] - ref_w)
            assert np.all(err <= bound), (b, n, float((err / bound).max()))
            assert np.array_equal(gw[b, :, n:], w0[b, :, n:]), b
    say("   worst share of the bound", worst)
    return out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,d,page", [(28, 4, 128, 16), (12, 2, 128, 24), (2, 1, 64, 7), (16, 16, 64, 100)])
def test_lengths_around_borders(dtype, hq, hk, d, page):
    run_case(1, dtype, hq, hk, d, page, EDGES, weights=True)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 72, 80, 96, 120, 136, 192, 248, 256])
def test_head_sizes(dtype, d):
    run_case(2 + d, dtype, 6, 2, d, 16, [1, 45, 130, 700], weights=True)


@pytest.mark.parametrize("hq,hk", [(1, 1), (5, 1), (16, 1), (17, 1), (33, 1), (71, 1), (40, 8), (64, 4)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_head_groups(dtype, hq, hk):
    run_case(40 + hq, dtype, hq, hk, 64, 16, [300, 0, 77], weights=True)


@pytest.mark.parametrize("page", [1, 3, 16, 33, 64, 1000])
@pytest.mark.parametrize("order", ["slots", "heads", "padded"])
def test_pages_and_memory_orders(page, order):
    run_case(80 + page, BF, 7, 1, 128, page, [5, 260, 1023], order)
    run_case(81 + page, HF, 12, 4, 80, page, [5, 260, 1023], order)


def test_one_long_sequence():
    run_case(100, BF, 28, 4, 128, 64, [40007], weights=True)
    run_case(101, HF, 12, 2, 128, 16, [65536])


def test_very_different_lengths():
    rng = np.random.default_rng(5)
    run_case(102, BF, 12, 2, 128, 16, [30000, 1, 0, 17, 5000] + rng.integers(1, 200, 90).tolist(), weights=True)


def test_many_sequences():
    rng = np.random.default_rng(6)
    run_case(103, HF, 4, 2, 32, 8, rng.integers(0, 60, 1024).tolist(), weights=True)


def test_wide_table():
    """Columns that no sequence reaches: the split goes by the lengths."""
    run_case(104, BF, 28, 4, 128, 16, [2000, 3, 400], wide=4000, weights=True)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scales_and_large_scores(dtype):
    run_case(105, dtype, 7, 1, 128, 16, [400, 33], scale=1.0, qsd=3.0, weights=True)  # scores of some hundreds
    run_case(106, dtype, 7, 1, 128, 16, [400, 33], scale=0.0)
    run_case(107, dtype, 7, 1, 128, 16, [400, 33], scale=-0.3)
    run_case(108, dtype, 7, 1, 128, 16, [400, 33], qsd=1e-4)
    run_case(109, dtype, 7, 1, 128, 16, [400, 33], scale=1e-5, qsd=1e4)


@pytest.mark.parametrize("dtype,big", [(BF, 1e10), (HF, 6e4)])
def test_scores_below_the_range(dtype, big):
    """Products past fp32's range: those tokens' weight is 0, whole tiles and
    chunks of them included."""
    rng = np.random.default_rng(15)
    pg = Paged(rng, [3000, 700], 2, 64, 16, dtype)
    for b, n in enumerate(pg.lens):
        skip = np.arange(n) % 977 != 650
        K = torch.zeros(n, 2, 64, dtype=dtype)
        K[torch.from_numpy(skip)] = -big
        K[torch.from_numpy(~skip)] = 0.0
        p, s = pg.where(b, np.arange(n))
        pg.cache.k[p.cuda(), s.cuda()] = K.cuda()
        pg.K[b] = K
    q = torch.full((2, 6, 64), 3e38 if dtype == HF else 1e32, device="cuda")
    w = torch.zeros(2, 2, pg.width * 16, device="cuda")
    out = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t, weights=w)
    for b, n in enumerate(pg.lens):
        live = np.flatnonzero(np.arange(n) % 977 == 650)
        V = pg.V[b].double().numpy()[live]
        for h in range(6):
            assert np.allclose(out[b, h].cpu().numpy(), V[:, h // 3].mean(0), rtol=0, atol=64 * EPS32 * np.abs(V).max())
        want = np.zeros((2, n))
        want[:, live] = 3.0 / len(live)
        assert np.allclose(w[b, :, :n].cpu().numpy(), want, rtol=64 * EPS32, atol=0)


def small(rng, lens=(40, 70, 100), dtype=BF):
    pg = Paged(rng, lens, 2, 64, 16, dtype)
    q = torch.from_numpy(rng.standard_normal((len(lens), 6, 64)).astype(np.float32)).cuda()
    return pg, q


def test_refused_rows_are_nan_and_alone():
    """A length below 0 or past the table gives NaN, a page id outside the
    pool too; the other sequences keep their values."""
    rng = np.random.default_rng(7)
    pg, q = small(rng, (40, 70, 100, 64))
    good = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)
    for lens, bad in (([40, -1, 100, 64], [1]), ([40, 70, 7 * 16 + 1, 64], [2]), ([2 ** 31 - 1, 70, 100, -2 ** 31], [0, 3])):
        w = torch.ones(4, 2, 7 * 16, device="cuda")
        out = ops.attn_decode(q, pg.cache, pg.table, torch.tensor(lens, dtype=torch.int32, device="cuda"), weights=w)
        for b in range(4):
            if b in bad:
                assert torch.isnan(out[b]).all() and torch.all(w[b] == 1), (lens, b)
            else:
                assert torch.equal(out[b], good[b]), (lens, b)
    for page in (-1, pg.cache.pages, 2 ** 31 - 1, -2 ** 31):
        t = pg.table.clone()
        t[2, 3] = page
        out = ops.attn_decode(q, pg.cache, t, pg.lens_t)
        assert torch.isnan(out[2]).all()
        assert torch.equal(out[[0, 1, 3]], good[[0, 1, 3]])


def test_non_finite_values_stay_with_their_heads():
    rng = np.random.default_rng(8)
    pg, q = small(rng)
    good = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)
    p, s = pg.where(1, [33])
    for t, x in ((pg.cache.k, float("nan")), (pg.cache.v, float("nan")), (pg.cache.v, float("inf"))):
        keep = t[p[0], s[0], 1].clone()
        t[p[0], s[0], 1] = x
        out = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)
        t[p[0], s[0], 1] = keep
        assert not torch.isfinite(out[1, 3:]).any()
        assert torch.equal(out[1, :3], good[1, :3]) and torch.equal(out[[0, 2]], good[[0, 2]])
    q2 = q.clone()
    q2[1, 4, 7] = float("inf")
    out = ops.attn_decode(q2, pg.cache, pg.table, pg.lens_t)
    assert torch.isnan(out[1, 4]).all()
    rest = [0, 1, 2, 3, 5]
    assert torch.equal(out[1, rest], good[1, rest]) and torch.equal(out[[0, 2]], good[[0, 2]])


def test_same_bits_every_time():
    rng = np.random.default_rng(9)
    pg = Paged(rng, [5000, 30, 900], 4, 128, 16, BF)
    q = torch.from_numpy(rng.standard_normal((3, 28, 128)).astype(np.float32)).cuda()
    a = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)
    for _ in range(5):
        assert torch.equal(a, ops.attn_decode(q, pg.cache, pg.table, pg.lens_t))


def test_two_streams_at_once():
    rng = np.random.default_rng(10)
    cases = []
    for i in range(2):
        pg = Paged(rng, [6000 + i, 50, 700], 4, 128, 16, BF)
        q = torch.from_numpy(rng.standard_normal((3, 28, 128)).astype(np.float32)).cuda()
        cases.append((pg, q, ops.attn_decode(q, pg.cache, pg.table, pg.lens_t), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (pg, q, _, s) in enumerate(cases):
            outs[i].append(ops.attn_decode(q, pg.cache, pg.table, pg.lens_t, stream=s))
    torch.cuda.synchronize()
    for i, (_, _, ref, _) in enumerate(cases):
        assert all(torch.equal(o, ref) for o in outs[i])


def test_pool_past_32_bits():
    """Pages whose byte offsets pass 2^32: the same values as in a small pool."""
    rng = np.random.default_rng(11)
    pg = Paged(rng, [100], 2, 128, 16, BF)
    q = torch.from_numpy(rng.standard_normal((1, 14, 128)).astype(np.float32)).cuda()
    ref = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)
    n = pg.cache.pages
    big = 2 ** 32 // (16 * 2 * 128 * 2) + 3 * n
    k = torch.empty(big, 16, 2, 128, dtype=BF, device="cuda")
    v = torch.empty(big, 16, 2, 128, dtype=BF, device="cuda")
    k[-n:], v[-n:] = pg.cache.k, pg.cache.v
    out = ops.attn_decode(q, ops.KvCache(k, v), pg.table + (big - n), pg.lens_t)
    assert torch.equal(out, ref)


def test_any_alignment_and_table_stride():
    """q, out and weights 4 bytes past a 16-byte border, table rows inside a
    wider tensor, the cache a slice of a larger pool: the same bits."""
    rng = np.random.default_rng(13)
    pg = Paged(rng, [700, 45, 2100], 2, 96, 24, HF)
    q = torch.from_numpy(rng.standard_normal((3, 10, 96)).astype(np.float32)).cuda()
    cap = pg.width * 24
    w = torch.rand(3, 2, cap, device="cuda")
    w1 = torch.empty(w.numel() + 1, device="cuda")[1:].view_as(w).copy_(w)
    ref = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t, weights=w)
    q1 = torch.empty(q.numel() + 1, device="cuda")[1:].view_as(q).copy_(q)
    out = torch.empty(q.numel() + 3, device="cuda")[3:].view_as(q)
    table = torch.full((3, pg.width + 9), -1, dtype=torch.int32, device="cuda")
    table[:, 5:5 + pg.width] = pg.table + 2
    n = pg.cache.pages
    pool = [torch.empty(n + 5, 24, 2, 96, dtype=HF, device="cuda") for _ in range(2)]
    pool[0][2:2 + n], pool[1][2:2 + n] = pg.cache.k, pg.cache.v
    ops.attn_decode(q1, ops.KvCache(*pool), table[:, 5:5 + pg.width], pg.lens_t, out=out, weights=w1)
    assert torch.equal(out, ref) and torch.equal(w1, w)


def test_shared_pages():
    """Two sequences with a common prefix in the same pages."""
    rng = np.random.default_rng(14)
    pg = Paged(rng, [640, 800], 2, 64, 16, BF)
    table = pg.table.clone()
    table[0, :40] = pg.table[1, :40]
    q = torch.from_numpy(rng.standard_normal((2, 6, 64)).astype(np.float32)).cuda()
    q[0] = q[1]
    lens = torch.tensor([640, 640], dtype=torch.int32, device="cuda")
    out = ops.attn_decode(q, pg.cache, table, lens)
    assert torch.equal(out[0], out[1])


def test_longest_sequence():
    """2^31 - 65536 tokens, the most that a table can hold, in one page of
    65536 slots that every table entry names: the softmax over equal runs is
    the softmax over one of them.  Every lane adds up to 2^31 / (512 * 4 * 32) *
    8 = 2^18 rounded terms, each off by at most half a step of the sum."""
    rng = np.random.default_rng(12)
    n, runs = 65536, 32767
    k, v = (torch.from_numpy(rng.standard_normal((1, n, 1, 8)).astype(np.float32)).to(BF).cuda() for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((1, 2, 8)).astype(np.float32)).cuda()
    table = torch.zeros(1, runs, dtype=torch.int32, device="cuda")
    out = ops.attn_decode(q, ops.KvCache(k, v), table, torch.tensor([runs * n], dtype=torch.int32, device="cuda"))
    ref, _, ck, cv = attn_f64(q[0].cpu().double().numpy(), k[0].cpu().double().numpy(), v[0].cpu().double().numpy(), 8 ** -0.5)
    assert np.all(np.abs(out[0].cpu().numpy() - ref) <= (attn_rel(8, ck)[:, None] + 2 ** 18 * EPS32) * cv)
