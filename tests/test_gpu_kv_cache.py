"""iq_kv_append and iq_kv_evict against plain 64-bit forms."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv_util import EPS32, HALF_STEP, Paged, evict_moves, rope_f64

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def check_append(seed, dtype, T, hq, hk, d, rot, page, far, order="slots", in_place=False):
    rng = np.random.default_rng(seed)
    say("append", seed, dtype, T, hq, hk, d, rot, page, far, order)
    pages = -(-T // page) + 3
    kv = [Paged(rng, [1], hk, d, page, dtype).memory(pages, order, 5.0, "cuda") for _ in range(2)]
    cache = ops.KvCache(*kv)
    q = rng.standard_normal((T, hq, d)).astype(np.float32)
    k, v = (rng.standard_normal((T, hk, d)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, far, T)
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    skip = rng.random(T) < 0.2
    slots[skip] = rng.choice([-1, pages * page, 2 ** 62, -2 ** 62], int(skip.sum()))
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    freqs = ops.rope_freqs(rot, 1e6) if rot else None
    qd = dev(q)
    out = ops.kv_append(qd if hq else None, dev(k), dev(v), dev(pos) if rot else None, dev(slots), freqs, cache,
                        q_out=qd if in_place else None)
    torch.cuda.synchronize()
    f = np.array([1e6 ** (-2.0 * i / rot) for i in range(rot // 2)]) if rot else np.zeros(0)
    # two products and a sum of fp32 roundings, cos and sin to 2 steps each
    def near(got, x, slack):
        ref = rope_f64(x.astype(np.float64), pos, f, rot)
        h = rot // 2
        c = np.abs(x).astype(np.float64)
        c[..., :h] += np.abs(x[..., h:rot])
        c[..., h:rot] += np.abs(x[..., :h])
        err = np.abs(got - ref)
        b32 = 8 * EPS32 * c
        assert np.all(err <= b32 + slack(np.abs(ref) + b32)), float((err / (b32 + slack(np.abs(ref)) + 1e-30)).max())
    if hq:
        assert (out.data_ptr() == qd.data_ptr()) == in_place
        near(out.cpu().numpy().reshape(T, hq, d), q, lambda r: 0 * r)
    live = ~skip
    p, s = slots[live] // page, slots[live] % page
    kc, vc = cache.k.cpu(), cache.v.cpu()
    half = HALF_STEP[dtype]
    tiny = 2.0 ** -25 if dtype == HF else 0.0  # half a step of fp16's subnormal values
    pos = pos[live]
    near(kc[p, s].double().numpy(), k[live], lambda r: half * r + tiny)
    assert torch.equal(vc[p, s], torch.from_numpy(v[live]).to(dtype))
    rest = np.ones((pages, page), bool)
    rest[p, s] = False
    assert torch.all(kc[rest] == 5) and torch.all(vc[rest] == 5)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T", [1, 2, 17, 300])
@pytest.mark.parametrize("hq,hk,d", [(28, 4, 128), (12, 2, 128), (2, 1, 64), (3, 3, 80), (16, 1, 256), (1, 1, 8)])
def test_append(dtype, T, hq, hk, d):
    check_append(T + d, dtype, T, hq, hk, d, d, 16, 131072)


@pytest.mark.parametrize("rot", [0, 8, 64, 120])
@pytest.mark.parametrize("order", ["slots", "heads", "padded"])
def test_append_part_rotary_and_orders(rot, order):
    check_append(rot, BF, 33, 6, 2, 128, rot, 7, 4096, order, in_place=rot == 64)


def test_append_far_positions():
    """10^9 positions on: the angle keeps its precision."""
    check_append(5, BF, 50, 4, 2, 64, 64, 16, 10 ** 9)


def test_append_cache_only():
    check_append(6, HF, 9, 0, 2, 64, 64, 16, 500)


def test_append_any_alignment_of_the_inputs():
    rng = np.random.default_rng(9)
    T, hq, hk, d = 37, 6, 2, 64
    dev = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    q, k, v = dev(T, hq, d), dev(T, hk, d), dev(T, hk, d)
    pos, slots = torch.arange(T, device="cuda") * 1000, torch.randperm(64, device="cuda")[:T]
    fr = ops.rope_freqs(d, 1e4)
    odd = lambda t: torch.empty(t.numel() + 1, device="cuda")[1:].view_as(t).copy_(t)  # noqa: E731
    a, b = (ops.alloc_kv(4, 16, hk, d) for _ in range(2))
    qa = ops.kv_append(q, k, v, pos, slots, fr, a)
    qb = ops.kv_append(odd(q), odd(k), odd(v), pos, slots, fr, b, q_out=odd(q))
    assert torch.equal(qa, qb) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_append_rounds_and_keeps_specials():
    cache = ops.alloc_kv(1, 4, 1, 8, HF)
    x = torch.tensor([65519.0, 65520.0, float("nan"), float("-inf"), -0.0, 2.0 ** -25, 2.0 ** -24, 1 + 2.0 ** -11],
                     device="cuda").view(1, 1, 8)
    ops.kv_append(None, x, x, None, torch.zeros(1, dtype=torch.int64, device="cuda"), None, cache)
    got, ref = cache.v[0, 0, 0].cpu(), x.view(8).cpu().half()
    assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0)) and torch.isnan(got[2])
    cache = ops.alloc_kv(1, 4, 1, 8, BF)
    ops.kv_append(None, x, x, None, torch.zeros(1, dtype=torch.int64, device="cuda"), None, cache)
    got, ref = cache.k[0, 0, 0].cpu(), x.view(8).cpu().bfloat16()
    assert torch.equal(got.nan_to_num(7.0), ref.nan_to_num(7.0)) and torch.isnan(got[2])


def check_evict(seed, dtype, lens, hk, d, page, budget, recent, order="slots", sums=None, pad=5):
    rng = np.random.default_rng(seed)
    say("evict", seed, dtype, lens[:6], len(lens), hk, d, page, budget, recent, order)
    pg = Paged(rng, lens, hk, d, page, dtype, order)
    B, cap = len(lens), pg.width * page
    w = np.exp(2 * rng.standard_normal((B, hk, cap + pad))).astype(np.float32)
    if sums is not None:
        w = sums(rng, w).astype(np.float32)
    wd = torch.from_numpy(w).cuda()
    before = [t.cpu().clone() for t in (pg.cache.k, pg.cache.v)]
    new = ops.kv_evict(pg.cache, pg.table, pg.lens_t, wd, budget, recent)
    torch.cuda.synchronize()
    got_w, after = wd.cpu().numpy(), [pg.cache.k.cpu(), pg.cache.v.cpu()]
    assert new.cpu().tolist() == [min(n, budget) for n in lens]
    want_w = w.copy()
    bits = [t.view(torch.int16).clone() for t in before]
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        for h in range(hk):
            src = evict_moves(w[b, h, :n], budget, recent)
            want_w[b, h, :budget] = w[b, h, src]
            want_w[b, h, budget:n] = 0
            (p0, s0), (p1, s1) = pg.where(b, src), pg.where(b, np.arange(budget))
            for t, o in zip(bits, before):
                t[p1, s1, h] = o.view(torch.int16)[p0, s0, h]
    assert np.array_equal(got_w.view(np.int32), want_w.view(np.int32))
    for t, a in zip(bits, after):
        assert torch.equal(a.contiguous().view(torch.int16), t), "rows"


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (64, 0), (64, 64), (100, 7), (299, 50), (300, 10)])
def test_evict(dtype, budget, recent):
    check_evict(budget + recent, dtype, [300, 0, 1, 64, 65, 101, 128, 299], 2, 64, 16, budget, recent)


@pytest.mark.parametrize("hk,d,page,order", [(4, 128, 16, "slots"), (1, 8, 1, "slots"), (3, 80, 7, "heads"),
                                             (2, 256, 33, "padded"), (8, 96, 100, "slots")])
def test_evict_layouts(hk, d, page, order):
    check_evict(d, BF, [500, 77, 1300], hk, d, page, 300, 64, order)


@pytest.mark.parametrize("n,budget,recent", [(20011, 5000, 700), (20011, 20010, 9000), (20011, 15000, 0),
                                             (70000, 1000, 999), (20011, 19000, 18000), (20011, 13000, 12900),
                                             (9000, 8743, 8000), (9000, 8745, 8000)])
def test_evict_long(n, budget, recent):
    check_evict(n + budget, BF, [n, 40], 2, 64, 16, budget, recent)


def test_evict_one_by_one():
    """A full window whose rows all move down by one."""
    check_evict(1, BF, [1025, 1025], 2, 128, 16, 1024, 1024)
    check_evict(2, BF, [1025, 1025], 2, 128, 16, 1024, 512)


def test_evict_uses_only_the_batch_table_columns():
    """Table rows inside a wider tensor, sums 4 bytes past a 16-byte border:
    the same result."""
    rng = np.random.default_rng(12)
    pg = Paged(rng, [300, 80], 2, 64, 16, BF)
    k0, v0 = pg.cache.k.clone(), pg.cache.v.clone()
    w = torch.rand(2, 2, pg.width * 16, device="cuda")
    w1 = torch.empty(w.numel() + 1, device="cuda")[1:].view_as(w).copy_(w)
    ops.kv_evict(pg.cache, pg.table, pg.lens_t, w, 60, 13)
    k1, v1 = pg.cache.k.clone(), pg.cache.v.clone()
    pg.cache.k.copy_(k0)
    pg.cache.v.copy_(v0)
    table = torch.full((2, pg.width + 6), -1, dtype=torch.int32, device="cuda")
    table[:, 2:2 + pg.width] = pg.table
    ops.kv_evict(pg.cache, table[:, 2:2 + pg.width], pg.lens_t, w1, 60, 13)
    bits = lambda t: t.view(torch.int16)  # noqa: E731
    assert torch.equal(w, w1)
    assert torch.equal(bits(pg.cache.k), bits(k1)) and torch.equal(bits(pg.cache.v), bits(v1))


def test_evict_many_sequences():
    rng = np.random.default_rng(3)
    check_evict(3, HF, rng.integers(0, 120, 1024).tolist(), 1, 8, 8, 60, 20)


def test_evict_ties_and_specials():
    check_evict(4, BF, [900, 333], 2, 64, 16, 200, 30, sums=lambda r, w: np.zeros_like(w))
    check_evict(5, BF, [900, 333], 2, 64, 16, 200, 30, sums=lambda r, w: r.integers(0, 3, w.shape) * 0.5)
    odd = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3.0, -3.0, 3e38, -np.nan], np.float32)
    check_evict(6, BF, [900, 333], 2, 64, 16, 200, 30, sums=lambda r, w: odd[r.integers(0, len(odd), w.shape)])
    check_evict(7, BF, [900, 333], 2, 64, 16, 700, 30, sums=lambda r, w: np.full_like(w, np.nan))


def test_evict_ties_in_long_rows():
    """More sums than a workgroup holds at once, most of them equal."""
    check_evict(8, BF, [70001, 33000], 1, 8, 64, 40000, 100, sums=lambda r, w: r.integers(0, 3, w.shape) * 0.5)
    check_evict(9, BF, [70001, 33000], 1, 8, 64, 20000, 0, sums=lambda r, w: np.zeros_like(w))
    check_evict(10, BF, [98304], 1, 8, 64, 65536, 1, sums=lambda r, w: r.standard_normal(w.shape))


def test_evict_refused_rows_are_left():
    rng = np.random.default_rng(8)
    pg = Paged(rng, [90, 90, 90, 90], 2, 64, 16, BF)
    w = torch.rand(4, 2, 96, device="cuda")
    table, lens = pg.table.clone(), pg.lens_t.clone()
    lens[0] = -3
    lens[1] = 97
    table[2, 5] = pg.cache.pages
    before = [t.clone() for t in (pg.cache.k, pg.cache.v, w)]
    new = ops.kv_evict(pg.cache, table, lens, w, 50, 10)
    assert new.cpu().tolist() == [-3, 97, 90, 50]
    assert torch.equal(w[:3], before[2][:3]) and not torch.equal(w[3], before[2][3])
    for b in range(3):
        p, s = pg.where(b, np.arange(90))
        for t, o in zip((pg.cache.k, pg.cache.v), before):
            assert torch.equal(t[p, s], o[p, s])
