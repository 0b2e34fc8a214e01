"""The decode step over paged caches (infer_amd/chain.py, CachedDecodeStep):
append, attention, eviction and log probabilities as one program, eager and
as a replayed graph."""
import numpy as np
import pytest
import torch

from infer_amd import chain as C
from infer_amd import ops
from oracle import oracle as O
from tests.gpu_util import say
from tests.kv_util import EPS32, HALF_STEP, attn_f64, attn_rel, evict_moves, logprobs_f64, rope_f64, top_order
from tests.test_gpu_chain import check_gemv, f64, make_model

pytestmark = pytest.mark.gpu

THETA = 1e6


def build(seed, B, heads=4, kv=2, hd=64, L=2, pages=4, page=16, dtype=torch.bfloat16, weights=True):
    rng = np.random.default_rng(seed)
    host, dev = make_model(rng, heads * hd, 512, heads, kv, hd, 300, L, 1, 0)
    dev["cfg"]["theta"] = THETA
    need = B * pages
    table = rng.permutation(need + 3)[:need].reshape(B, pages).astype(np.int32)
    caches = [ops.alloc_kv(need + 3, page, kv, hd, dtype) for _ in range(L)]
    for c in caches:  # whatever lies where no token was added has no influence
        c.k.fill_(float("nan"))
        c.v.fill_(float("nan"))
    return rng, host, C.CachedDecodeStep(dev, caches, torch.from_numpy(table).cuda(), weights), table


def cached(step, li, table, b, n):
    t = np.arange(n)
    p, s = torch.from_numpy(table[b, t // step.page].astype(np.int64)), torch.from_numpy(t % step.page)
    return [x[p.cuda(), s.cuda()].double().cpu().numpy() for x in (step.caches[li].k, step.caches[li].v)]


def check_layers(step, host, table, lens, pos, sums):
    """Every layer's append, attention and o projection on the step's own
    vectors; sums: the weights so far (float64), updated."""
    c = host["cfg"]
    nh, nkv, hd, H = c["heads"], c["kv_heads"], c["head_dim"], c["hidden"]
    freqs = THETA ** (-2.0 * np.arange(hd // 2) / hd)
    half = HALF_STEP[step.caches[0].k.dtype]
    # below 2^-14 fp16's steps are 2^-24 whatever the value: half a step is 2^-25
    tiny = 2.0 ** -25 if step.caches[0].k.dtype == torch.float16 else 0.0
    for li, b in enumerate(step.per_layer):
        for r in range(step.rows):
            n = lens[r]
            q, k, v = (f64(b[x]).reshape(step.rows, -1, hd)[r] for x in ("q", "k", "v"))
            at = np.array([pos[r]])
            q_rot = f64(b["q_rot"]).reshape(step.rows, nh, hd)[r]
            cond = np.abs(q) + np.abs(np.roll(q, hd // 2, 1))
            assert np.all(np.abs(q_rot - rope_f64(q[None], at, freqs, hd)[0]) <= 8 * EPS32 * cond)
            K, V = cached(step, li, table, r, n)
            kr = rope_f64(k[None], at, freqs, hd)[0]
            slack = 8 * EPS32 * (np.abs(k) + np.abs(np.roll(k, hd // 2, 1)))
            assert np.all(np.abs(K[-1] - kr) <= half * (np.abs(kr) + slack) + slack + tiny)
            assert np.all(np.abs(V[-1] - v) <= half * np.abs(v) + tiny)
            ref, p, ck, cv = attn_f64(q_rot, K, V, hd ** -0.5)
            got = f64(b["attn"]).reshape(step.rows, nh, hd)[r]
            assert np.all(np.abs(got - ref) <= attn_rel(hd, ck)[:, None] * cv), (li, r, n)
            if step.weights:
                sums[li][r][:, :n] += p.reshape(nkv, -1, n).sum(1)
            h, h1 = f64(b["h"]).reshape(step.rows, H)[r], f64(b["h1"]).reshape(step.rows, H)[r]
            check_gemv(h1 - h, host["layers"][li]["o"], got.reshape(-1), np.arange(H), f"L{li}.o+res",
                       slack=np.abs(h1) * 2.0 ** -24)


@pytest.mark.parametrize("B,dtype", [(1, torch.bfloat16), (3, torch.float16)])
def test_steps_evictions_and_answers(B, dtype):
    rng, host, step, table = build(B, B, dtype=dtype)
    V, L, nkv = host["cfg"]["vocab"], host["cfg"]["layers"], host["cfg"]["kv_heads"]
    lens = np.zeros(B, np.int64)
    pos = np.zeros(B, np.int64)
    sums = [np.zeros((B, nkv, step.capacity)) for _ in range(L)]
    for it in range(50):
        ids = rng.integers(0, V, B).tolist()
        step.step(ids)
        torch.cuda.synchronize()
        lens += 1
        assert step.lens.cpu().tolist() == lens.tolist()
        check_layers(step, host, table, lens, pos, sums)
        pos += 1
        if it % 12 == 0:
            tokens = torch.from_numpy(rng.integers(0, V, B)).cuda()
            r = step.logprobs(tokens, top=7)
            x = step.logits.cpu().numpy()
            for b in range(B):
                lp, h = logprobs_f64(x[b])
                ids7 = top_order(x[b], 7)
                assert np.array_equal(r.top_ids[b].cpu().numpy(), ids7)
                bound = 2 * EPS32 * (np.abs(lp).max() + 20) + 80 * EPS32
                assert abs(float(r.logprob[b]) - lp[int(tokens[b])]) <= bound
                assert np.all(np.abs(r.top_logprobs[b].cpu().numpy() - lp[ids7]) <= bound)
                assert abs(float(r.entropy[b]) - h) <= 200 * EPS32 * (1 + np.abs(lp).max())
        if it in (20, 33, 41):
            w = [x.cpu().numpy() for x in step.weights]
            for li in range(L):  # the sums: every step's rounding, half a step of at most `it`
                assert np.allclose(w[li], sums[li], rtol=1e-4, atol=0)
            before = [[cached(step, li, table, b, lens[b]) for b in range(B)] for li in range(L)]
            budget, recent = 17, 6
            step.evict(budget, recent)
            torch.cuda.synchronize()
            for li in range(L):
                for b in range(B):
                    n = lens[b]
                    now = cached(step, li, table, b, budget)
                    for h in range(nkv):
                        src = evict_moves(w[li][b, h, :n], budget, recent)
                        for o, t in zip(before[li][b], now):
                            assert np.array_equal(o[src, h], t[:, h]), (li, b, h)
                        sums[li][b, h, :budget] = sums[li][b, h, src]
                        sums[li][b, h, budget:] = 0
                assert np.array_equal(step.weights[li].cpu().numpy()[:, :, budget:], 0 * w[li][:, :, budget:])
            lens[:] = budget
            assert step.lens.cpu().tolist() == lens.tolist()
    say("cached decode", B, lens, pos)


def test_full_and_missing_pages():
    rng, host, step, table = build(7, 3, pages=2, weights=False)
    step.table[2, 1] = -1
    for it in range(34):
        step.step(it)
        if it == 15:
            ref = step.logits.clone()
    torch.cuda.synchronize()
    assert torch.isfinite(ref).all()
    assert torch.isnan(step.logits).all()  # 33 tokens do not fit 32 places, the third row's second page is none
    assert step.lens.cpu().tolist() == [34] * 3
    with pytest.raises(ValueError):
        step.evict(5, 1)


def test_graph_replays_like_eager():
    """One captured step, replayed: the state moves on by itself.  Eager work
    on the same stream's workspace runs between the replays."""
    B = 2
    runs = []
    for graph in (False, True):
        rng, host, step, table = build(11, B)
        ids = rng.integers(0, host["cfg"]["vocab"], (12, B))
        top = ops.alloc_logprobs(B, 5)
        got = []
        g, s = None, torch.cuda.Stream()
        ops.init(0, s)
        torch.cuda.synchronize()
        for it in range(12):
            step.ids.copy_(torch.from_numpy(ids[it]))
            torch.cuda.synchronize()
            if not graph or it == 0:
                with torch.cuda.stream(s):
                    step.step()
                    step.logprobs(step.ids, 5, top)
            else:
                if g is None:
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=s):
                        step.step()
                        step.logprobs(step.ids, 5, top)
                with torch.cuda.stream(s):
                    g.replay()
            if it == 7:
                with torch.cuda.stream(s):
                    step.evict(5, 2)
            torch.cuda.synchronize()
            got.append([step.logits.clone(), *(x.clone() for x in top), *(w.clone() for w in step.weights)])
            with torch.cuda.stream(s):  # other work on the same workspace
                x = torch.randn(3, 9000, device="cuda")
                ops.logprobs(x, top=9)
                ops.linear(x[:, :512].contiguous(), step.model["layers"][0]["down"])
            torch.cuda.synchronize()
        runs.append(got)
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_no_allocation_in_the_operators():
    """Once a stream has its workspace, every operator can be captured the
    first time it is called."""
    rng = np.random.default_rng(3)
    cache = ops.alloc_kv(40, 16, 2, 128)
    table = torch.arange(32, dtype=torch.int32, device="cuda").view(2, 16)
    lens = torch.tensor([200, 256], dtype=torch.int32, device="cuda")
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    cache.k.copy_(f(*cache.k.shape))
    cache.v.copy_(f(*cache.v.shape))
    q, k, v, x = f(2, 12, 128), f(2, 2, 128), f(2, 2, 128), f(2, 40000)
    pos, slots = torch.tensor([199, 255], device="cuda"), torch.tensor([12 * 16 + 7, 31 * 16 + 15], device="cuda")
    fr, w = ops.rope_freqs(128, THETA), torch.rand(2, 2, 256, device="cuda")
    w0, k0, v0 = w.clone(), cache.k.clone(), cache.v.clone()
    out, qo, lp = torch.empty_like(q), torch.empty_like(q), ops.alloc_logprobs(2, 20)
    new = torch.empty_like(lens)

    def run(s):
        w.copy_(w0)
        cache.k.copy_(k0)
        cache.v.copy_(v0)
        ops.kv_append(q, k, v, pos, slots, fr, cache, q_out=qo, stream=s)
        ops.attn_decode(qo, cache, table, lens, out=out, weights=w, stream=s)
        ops.kv_evict(cache, table, lens, w, 100, 30, new_lens=new, stream=s)
        ops.logprobs(x, pos, 20, lp, stream=s)
        return [out, qo, w, new, cache.k, cache.v, *lp]
    s = torch.cuda.Stream()
    ops.init(0, s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = run(s)
    want = [t.clone() for t in run(None)]
    torch.cuda.synchronize()
    for _ in range(4):
        for t in (out, qo, new, *lp):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        run(None)
        torch.cuda.synchronize()


def test_capture_without_workspace_is_refused():
    cache = ops.alloc_kv(2, 16, 1, 64)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q, w, x = torch.zeros(1, 4, 64, device="cuda"), torch.zeros(1, 1, 32, device="cuda"), torch.zeros(1, 9000, device="cuda")
    out, new, lp = torch.empty_like(q), torch.empty_like(lens), ops.alloc_logprobs(1, 3)
    for call in (lambda s: ops.attn_decode(q, cache, table, lens, out=out, stream=s),
                 lambda s: ops.kv_evict(cache, table, lens, w, 1, 1, new_lens=new, stream=s),
                 lambda s: ops.logprobs(x, top=3, out=lp, stream=s)):
        s = torch.cuda.Stream()  # no iq_init_stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="iq_"):
            with torch.cuda.graph(g, stream=s):
                x.add_(0.0)  # (a non-empty capture)
                call(s)
        torch.cuda.synchronize()
