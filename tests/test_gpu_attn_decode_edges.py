"""iq_attn_decode where its scores are extreme and where its sizes are: scores
of 2^22 to 2^33, rows none of whose scores lies in fp32's range, and more heads
in a batch than one launch has room for."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv_util import EPS32, Paged, attn_rel

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def set_keys(pg, b, K):
    """Sequence b's keys, one number a token for all heads and values."""
    p, s = pg.where(b, np.arange(len(K)))
    pg.cache.k[p.cuda(), s.cuda()] = torch.from_numpy(np.asarray(K, np.float32)).to(pg.dtype).cuda()[:, None, None]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens", [[90, 17], [3000]])
def test_large_equal_scores(dtype, lens):
    """Every third key gives the same large score, the others 0: the weight is
    1 / (number of large ones) there and 0 elsewhere.  All p are equal powers of
    two, so the values' sum has n roundings at most, and the division one."""
    rng = np.random.default_rng(21)
    pg = Paged(rng, lens, 1, 8, 16, dtype)
    n = max(lens)
    for b, m in enumerate(lens):
        set_keys(pg, b, 0.5 * (np.arange(m) % 3 == 0))
    for e in np.arange(22, 34, 0.25):
        # 8 products of 2^e / 4 and 1/2: a score of 2^e (in powers of e)
        q = torch.full((len(lens), 3, 8), float(2.0 ** e / 4), device="cuda")
        w = torch.zeros(len(lens), 1, pg.width * 16, device="cuda")
        out = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t, weights=w, scale=1.0)
        for b, m in enumerate(lens):
            live = np.arange(m) % 3 == 0
            V = pg.V[b].double().numpy()[live, 0]
            err = np.abs(out[b].cpu().double().numpy() - V.mean(0))
            assert np.all(err <= (n + 4) * EPS32 * np.abs(V).mean(0)), (e, b, float(np.nanmax(err)))
            want = np.where(live, 3.0 / live.sum(), 0.0)
            # exp and 1 / sum to a step each, three additions
            assert np.all(np.abs(w[b, 0, :m].cpu().double().numpy() - want) <= 8 * EPS32 * want), (e, b)


@pytest.mark.parametrize("dtype,big,qbig", [(BF, 1e10, 1e32), (HF, 6e4, 3e38)])
@pytest.mark.parametrize("lens", [[1, 33, 100, 127], [3000, 700], [20000]])
def test_no_score_in_range(dtype, big, qbig, lens):
    """Heads all of whose scores lie below fp32's range: zeros, and nothing
    added to the weights, in one chunk and in several.  The third head of each
    three has equal scores and is the mean of the values."""
    rng = np.random.default_rng(22)
    pg = Paged(rng, lens, 2, 64, 16, dtype)
    for b, n in enumerate(lens):
        set_keys(pg, b, np.full(n, -big))
    q = torch.full((len(lens), 6, 64), qbig, device="cuda")
    q[:, 2::3] = 0.0
    w0 = torch.rand(len(lens), 2, pg.width * 16, device="cuda")
    w = w0.clone()
    for weights in (None, w):
        out = ops.attn_decode(q, pg.cache, pg.table, pg.lens_t, weights=weights).cpu()
        for b, n in enumerate(lens):
            V = pg.V[b].double().numpy()
            for h in range(6):
                if h % 3 < 2:
                    assert torch.all(out[b, h] == 0), (b, h, out[b, h, :3])
                else:
                    err = np.abs(out[b, h].double().numpy() - V[:, h // 3].mean(0))
                    assert np.all(err <= (n + 4) * EPS32 * np.abs(V[:, h // 3]).mean(0))
    for b, n in enumerate(lens):
        want = w0[b, :, :n].double() + 1.0 / n
        assert torch.all((w[b, :, :n].double() - want).abs() <= EPS32 * want + 4 * EPS32 / n)
        assert torch.equal(w[b, :, n:], w0[b, :, n:])


def test_no_score_in_range_keeps_nan():
    """A page that is none still gives NaN to such a head and to its weights,
    a value that is NaN to the head."""
    rng = np.random.default_rng(23)
    pg = Paged(rng, [300, 300], 1, 64, 16, BF)
    for b in range(2):
        set_keys(pg, b, np.full(300, -1e10))
    q = torch.full((2, 2, 64), 1e32, device="cuda")
    table = pg.table.clone()
    table[1, 7] = -1
    w = torch.zeros(2, 1, pg.width * 16, device="cuda")
    out = ops.attn_decode(q, pg.cache, table, pg.lens_t, weights=w)
    assert torch.all(out[0] == 0) and torch.isnan(out[1]).all()
    assert torch.all(w[0] == 0) and torch.isnan(w[1, 0, :300]).all()
    p, s = pg.where(0, [200])
    pg.cache.v[p[0], s[0]] = float("nan")
    assert torch.isnan(ops.attn_decode(q, pg.cache, pg.table, pg.lens_t)[0]).all()


@pytest.mark.parametrize("B,hq,hk,d", [(1024, 8192, 16, 8), (900, 16384, 64, 8)])
def test_many_heads_in_a_batch(B, hq, hk, d):
    """More (sequence, head) pairs than one launch keeps maxima and sums of."""
    say("attn", B, hq, hk, d)
    gen = torch.Generator(device="cuda").manual_seed(B)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    K, V = f(B, 16, hk, d).to(BF), f(B, 16, hk, d).to(BF)
    q = f(B, hq, d)
    lens = torch.randint(0, 17, (B,), generator=gen, device="cuda", dtype=torch.int32)
    order = torch.randperm(B, generator=gen, device="cuda")
    cache = ops.KvCache(K[order].contiguous(), V[order].contiguous())
    table = torch.empty(B, dtype=torch.int32, device="cuda")
    table[order] = torch.arange(B, dtype=torch.int32, device="cuda")
    out = ops.attn_decode(q, cache, table[:, None], lens).view(B, hk, hq // hk, d)
    step = 50
    for b in range(0, B, step):
        qd = q[b:b + step].view(-1, hk, hq // hk, d).double() * d ** -0.5
        Kd, Vd = K[b:b + step].double(), V[b:b + step].double()
        live = torch.arange(16, device="cuda")[None, :] < lens[b:b + step, None]
        s = torch.stack([(qd * Kd[:, t, :, None]).sum(-1) for t in range(16)], -1)
        ck = torch.stack([(qd * Kd[:, t, :, None]).abs().sum(-1) for t in range(16)], -1)
        s = s.masked_fill(~live[:, None, None], float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        ref = sum(p[..., t, None] * Vd[:, t, :, None] for t in range(16))
        cv = sum(p[..., t, None] * Vd[:, t, :, None].abs() for t in range(16))
        rel = attn_rel(d, ck.masked_fill(~live[:, None, None], 0).amax(-1))[..., None]
        assert torch.all((out[b:b + step].double() - ref).abs() <= rel * cv), b
