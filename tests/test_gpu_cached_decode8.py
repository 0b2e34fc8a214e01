"""CachedDecodeStep over 8-bit caches, with norms of the heads and under a
window: tokens added, attended to and read back as one program, eager and as a
replayed graph."""
import numpy as np
import pytest
import torch

from infer_amd import chain as C
from infer_amd import ops
from tests.gpu_util import say
from tests.kv8_util import CODES, LARGEST, decode, made_slack, norm_f64
from tests.kv_util import EPS32, HALF_STEP, attn_f64, rope_f64
from tests.test_gpu_attn_window import rel, seen
from tests.test_gpu_chain import check_gemv, f64, make_model

pytestmark = pytest.mark.gpu
I8, F8, BF = torch.int8, torch.float8_e4m3fn, torch.bfloat16
THETA = 1e6


def build(seed, B, dtypes, block=8, heads=4, kv=2, hd=64, pages=4, page=16, norms=True, window=0, sinks=0):
    """One layer for each of dtypes."""
    rng = np.random.default_rng(seed)
    L = len(dtypes)
    host, dev = make_model(rng, heads * hd, 512, heads, kv, hd, 300, L, 1, 0)
    dev["cfg"]["theta"] = THETA
    for hl, dl in zip(host["layers"], dev["layers"]):
        for n in ("q_norm", "k_norm") if norms else ():
            w = torch.from_numpy(1 + 0.3 * rng.standard_normal(hd)).to(BF)
            hl[n], dl[n] = w.double().numpy(), w.cuda()
    need = B * pages
    table = rng.permutation(need + 3)[:need].reshape(B, pages).astype(np.int32)
    caches = [ops.alloc_kv(need + 3, page, kv, hd, t, block=block if t in CODES else None) for t in dtypes]
    for c in caches:  # whatever lies where no token was added has no influence
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(255)
        if c.block:
            c.k_scales.fill_(float("nan"))
            c.v_scales.fill_(float("nan"))
    step = C.CachedDecodeStep(dev, caches, torch.from_numpy(table).cuda(), window=window, sinks=sinks)
    return rng, host, step, table


def cached(step, li, table, b, t):
    """K, V of tokens t, and their scales."""
    c = step.caches[li]
    p, s = table[b, t // step.page].astype(np.int64), t % step.page
    got = []
    for x, sc in ((c.k, c.k_scales), (c.v, c.v_scales)):
        if c.block:
            y = sc.cpu().double().numpy()[p, s // c.block][..., None]
            got += [decode(x.view(torch.uint8).cpu().numpy()[p, s], c.k.dtype).astype(np.float64) * y, y]
        else:
            got += [x[torch.from_numpy(p).cuda(), torch.from_numpy(s).cuda()].double().cpu().numpy(), None]
    return got


def check_layers(step, host, table, lens, pos):
    c = host["cfg"]
    nh, nkv, hd, H = c["heads"], c["kv_heads"], c["head_dim"], c["hidden"]
    freqs = THETA ** (-2.0 * np.arange(hd // 2) / hd)
    for li, b in enumerate(step.per_layer):
        dtype, hl = step.caches[li].k.dtype, host["layers"][li]
        for r in range(step.rows):
            n, at = lens[r], np.array([pos[r]])
            q, k, v = (f64(b[x]).reshape(step.rows, -1, hd)[r] for x in ("q", "k", "v"))

            def made(x, name):
                y = norm_f64(x, hl[name], c["eps"]) if name in hl else x
                return rope_f64(y[None], at, freqs, hd)[0], made_slack(y, hl.get(name), hd // 2)
            ref, slack = made(q, "q_norm")
            q_rot = f64(b["q_rot"]).reshape(step.rows, nh, hd)[r]
            assert np.all(np.abs(q_rot - ref) <= slack)
            t = seen(n, step.window, step.sinks)
            K, ks, V, vs = cached(step, li, table, r, t)
            kr, slack = made(k, "k_norm")
            for x, y, sl, s in ((K[-1], kr, slack, ks), (V[-1], v, 0.0, vs)):
                if dtype in CODES:
                    # half a step, and the roundings of the division and of the scale
                    half = 0.5 * s[-1] if dtype == I8 else np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * s[-1]) * (1 + 2.0 ** -3)
                    most = half + 2 * sl + 4 * EPS32 * (np.abs(y) + s[-1] * LARGEST[dtype])
                else:
                    most = HALF_STEP[dtype] * (np.abs(y) + sl) + sl
                assert np.all(np.abs(x - y) <= most), (li, r, n)
            ref, _, ck, cv = attn_f64(q_rot, K, V, hd ** -0.5)
            got = f64(b["attn"]).reshape(step.rows, nh, hd)[r]
            assert np.all(np.abs(got - ref) <= rel(hd, ck)[:, None] * cv), (li, r, n)
            h, h1 = f64(b["h"]).reshape(step.rows, H)[r], f64(b["h1"]).reshape(step.rows, H)[r]
            check_gemv(h1 - h, hl["o"], got.reshape(-1), np.arange(H), f"L{li}.o+res", slack=np.abs(h1) * 2.0 ** -24)


@pytest.mark.parametrize("B,dtypes,norms,window,sinks", [(1, (I8, F8), False, 0, 0), (3, (F8, BF, I8), True, 20, 3),
                                                         (2, (BF, BF), True, 0, 0), (2, (BF, I8), False, 7, 0)])
def test_steps(B, dtypes, norms, window, sinks):
    rng, host, step, table = build(B, B, dtypes, norms=norms, window=window, sinks=sinks)
    lens = np.zeros(B, np.int64)
    for it in range(50):
        step.step(rng.integers(0, host["cfg"]["vocab"], B).tolist())
        torch.cuda.synchronize()
        lens += 1
        assert step.lens.cpu().tolist() == lens.tolist() == step.held.cpu().tolist()
        if it < 20 or it % 7 == 0:
            check_layers(step, host, table, lens, lens - 1)
        assert torch.isfinite(step.logits).all()
    # the whole sequences as numbers
    starts = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32).cuda()
    for li, c in enumerate(step.caches):
        k, v = ops.kv_read(c, step.table, starts, T=int(lens.sum()))
        for b in range(B):
            K, _, V, _ = cached(step, li, table, b, np.arange(lens[b]))
            n = slice(int(starts[b]), int(starts[b + 1]))
            # (a product rounded once to fp32)
            assert np.all(np.abs(k[n].cpu().double().numpy() - K) <= EPS32 * np.abs(K))
            assert np.all(np.abs(v[n].cpu().double().numpy() - V) <= EPS32 * np.abs(V))
    say("cached decode", B, dtypes, norms, window, sinks)


def test_rows_without_a_place():
    """A missing page, then a full table, beside a row that goes on; idle rows;
    a row that starts anew in used pages."""
    rng, host, step, table = build(5, 3, (I8, F8), pages=2)
    twin = build(5, 3, (I8, F8), pages=2)[2]
    step.table[1, 1] = step.caches[0].pages
    for it in range(18):
        step.step(it)
        twin.step(it)
    assert torch.isnan(step.logits[1]).all() and torch.equal(step.logits[[0, 2]], twin.logits[[0, 2]])
    assert step.held.cpu().tolist() == [18, 16, 18]
    step.table[1, 1] = int(table[1, 1])
    step.lens[2] = -1
    step.step(3)
    assert step.held.cpu().tolist()[:2] == [19, 17] and torch.isnan(step.logits[2]).all()
    torch.cuda.synchronize()
    for li in range(2):  # the row's first token of its second page
        K, _, V, _ = cached(step, li, table, 1, np.arange(17))
        assert np.isfinite(K).all() and np.isfinite(V).all()
    # the third row from its beginning: the same steps as a fresh one, whatever its pages held
    step.lens[2], step.positions[2] = 0, 0
    fresh = build(5, 3, (I8, F8), pages=2)[2]
    for it in range(9):
        step.step([0, 0, 40 + it])
        fresh.step([0, 0, 40 + it])
    assert torch.equal(step.logits[2], fresh.logits[2]) and torch.isfinite(step.logits[2]).all()
    for it in range(20):
        step.step(1)
    assert torch.isnan(step.logits[:2]).all() and torch.isfinite(step.logits[2]).all()


def test_graph_replays_like_eager():
    runs = []
    for graph in (False, True):
        rng, host, step, table = build(11, 2, (I8, F8, BF), window=9, sinks=2)
        ids = rng.integers(0, host["cfg"]["vocab"], (14, 2))
        got, g, s = [], None, torch.cuda.Stream()
        ops.init(0, s)
        torch.cuda.synchronize()
        for it in range(14):
            step.ids.copy_(torch.from_numpy(ids[it]))
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                if not graph or it == 0:
                    step.step()
                else:
                    if g is None:
                        g = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(g, stream=s):
                            step.step()
                    g.replay()
            torch.cuda.synchronize()
            got.append([step.logits.clone(), *(c.k.view(torch.uint8).clone() for c in step.caches),
                        *(c.k_scales.nan_to_num(7.0) for c in step.caches if c.block)])
            with torch.cuda.stream(s):  # other work on the same workspace
                x = torch.randn(3, 9000, device="cuda")
                ops.logprobs(x, top=9)
                ops.linear(x[:, :512].contiguous(), step.model["layers"][0]["down"])
            torch.cuda.synchronize()
        runs.append(got)
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_what_goes_together():
    with pytest.raises(ValueError, match="weights"):
        C.CachedDecodeStep(*parts(I8), weights=True)
    with pytest.raises(ValueError, match="weights"):
        C.CachedDecodeStep(*parts(BF), weights=True, window=5)
    with pytest.raises(ValueError, match="negative"):
        C.CachedDecodeStep(*parts(BF), window=-5)


def parts(dtype):
    rng = np.random.default_rng(0)
    _, dev = make_model(rng, 128, 256, 2, 1, 64, 50, 1, 1, 0)
    dev["cfg"]["theta"] = THETA
    return dev, [ops.alloc_kv(2, 16, 1, 64, dtype)], torch.zeros(1, 2, dtype=torch.int32).cuda()


def test_no_allocation_in_the_operators():
    """Once a stream has its workspace, every operator can be captured the
    first time it is called; every replay gives what the eager calls give."""
    rng = np.random.default_rng(3)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    for dtype in (I8, F8, BF):
        cache = ops.alloc_kv(40, 16, 2, 128, dtype, block=16 if dtype in CODES else None)
        table = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
        zero, lens = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([203, 251], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, 200, 450], dtype=torch.int32, device="cuda")
        x = f(450, 2, 128)
        ops.kv_extend(None, x, x, None, None, cache, table, zero, starts=starts)
        few = torch.tensor([0, 3, 4], dtype=torch.int32, device="cuda")
        at = torch.tensor([200, 250], dtype=torch.int32, device="cuda")
        q, k, v, q1 = f(4, 12, 128), 4 * f(4, 2, 128), 4 * f(4, 2, 128), f(2, 12, 128)
        pos, fr = torch.tensor([200, 201, 202, 250], device="cuda"), ops.rope_freqs(128, THETA)
        w = torch.ones(128, dtype=BF, device="cuda")
        qo, out, rows = torch.empty_like(q), torch.empty_like(q1), [torch.zeros(454, 2, 128, dtype=BF, device="cuda") for _ in range(2)]
        all_, saved = torch.tensor([0, 203, 454], dtype=torch.int32, device="cuda"), [t.clone() for t in (cache.k, cache.v)]
        scales = [t.clone() for t in (cache.k_scales, cache.v_scales)] if cache.block else []

        def run(s):
            for t, u in zip((cache.k, cache.v, *((cache.k_scales, cache.v_scales) if cache.block else ())), saved + scales):
                t.view(torch.uint8).copy_(u.view(torch.uint8))
            ops.kv_extend(q, k, v, pos, fr, cache, table, at, starts=few, q_norm=w, k_norm=w, q_out=qo, stream=s)
            ops.attn_decode(q1, cache, table, lens, out=out, window=100, sinks=4, stream=s)
            ops.kv_read(cache, table, all_, out=rows, stream=s)
            return [qo, out, *rows, cache.k.view(torch.uint8), cache.v.view(torch.uint8)]
        s = torch.cuda.Stream()
        ops.init(0, s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got = run(s)
        want = [t.clone() for t in run(None)]
        torch.cuda.synchronize()
        for _ in range(4):
            for t in (qo, out, *rows):
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            run(None)
            torch.cuda.synchronize()


def test_capture_without_workspace_is_refused():
    cache = ops.alloc_kv(2, 16, 1, 64, I8)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q, x = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(9, device="cuda")
    s = torch.cuda.Stream()  # no iq_init_stream
    torch.cuda.synchronize()
    out, g = torch.empty_like(q), torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="iq_"):
        with torch.cuda.graph(g, stream=s):
            x.add_(0.0)  # (a non-empty capture)
            ops.attn_decode(q, cache, table, lens, out=out, stream=s)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtypes", [(I8, F8), (BF, I8)])
def test_a_ring_of_pages_under_a_window(dtypes):
    """A window of 20 and 3 first tokens need the first page and the last three:
    the table names the same few pages over and over, with the answers of a table
    that names new ones."""
    got = []
    for ring in (False, True):
        rng, host, step, table = build(6, 2, dtypes, window=20, sinks=3, pages=8)
        if ring:
            for b in range(2):
                for p in range(4, 8):
                    table[b, p] = table[b, p - 3]
            step.table.copy_(torch.from_numpy(table))
        for it in range(120):
            step.step([it, 299 - it])
            got.append(step.logits.clone())
    assert all(torch.equal(a, b) for a, b in zip(got[:120], got[120:]))
    assert torch.isfinite(got[-1]).all()


def test_norms_with_kept_weights_and_evictions():
    """Layers with norms over 16-bit caches whose rows are evicted: tokens go
    behind what is left, at positions that go on; the weights of what was cached
    add up to one per head and step."""
    B = 3
    rng, host, step, table = build(31, B, (BF, BF))
    step = C.CachedDecodeStep(step.model, step.caches, step.table, weights=True)
    c = host["cfg"]
    group = c["heads"] // c["kv_heads"]
    lens, pos = np.zeros(B, np.int64), np.zeros(B, np.int64)
    for it in range(45):
        before = [w.double().sum(-1).cpu().numpy() for w in step.weights]
        step.step(rng.integers(0, c["vocab"], B).tolist())
        torch.cuda.synchronize()
        lens, pos = lens + 1, pos + 1
        assert step.lens.cpu().tolist() == lens.tolist() == step.held.cpu().tolist()
        assert step.positions.cpu().tolist() == pos.tolist()
        check_layers(step, host, table, lens, pos - 1)
        for w, old in zip(step.weights, before):
            # a weight is 2^x / l with |x| below 64 (rows of norm 8 * 2.2 at most): two roundings of x and
            # 64 half steps more (exp, sums, division), in it and in l; and the additions' own rounding
            new = w.double().sum(-1).cpu().numpy()
            assert np.all(np.abs(new - old - group) <= 2 * (2 * 64 + 64) * EPS32 * group + (group + 1) * EPS32 * new)
        if it in (19, 33):
            step.evict(9, 4)
            lens = np.minimum(lens, 9)
