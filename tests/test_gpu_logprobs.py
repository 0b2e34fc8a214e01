"""iq_logprobs against a plain 64-bit form."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.gpu_util import say
from tests.kv_util import EPS32, logprobs_f64, top_order

pytestmark = pytest.mark.gpu


def check(x, tokens, top, pad=0, ent=True, offset=0):
    T, V = x.shape
    say("logprobs", T, V, top, pad)
    buf = np.full(T * (V + pad) + offset, 1e30, np.float32)
    rows = buf[offset:].reshape(T, V + pad)
    rows[:, :V] = x
    xd = torch.from_numpy(buf).cuda()[offset:].view(T, V + pad)[:, :V]
    tk = None if tokens is None else torch.from_numpy(np.asarray(tokens, np.int64)).cuda()
    out = ops.alloc_logprobs(T, top)
    if not ent:
        out = out._replace(entropy=None)
    r = ops.logprobs(xd, tk, top=top, out=out)
    torch.cuda.synchronize()
    for t in range(T):
        lp, h = logprobs_f64(x[t])
        ids = top_order(x[t], top)
        if top:
            assert np.array_equal(r.top_ids[t].cpu().numpy(), ids), (t, r.top_ids[t].cpu().numpy()[:8], ids[:8])
        want = [] if tokens is None else [(r.logprob[t], tokens[t])]
        want += [(r.top_logprobs[t, i], ids[i]) for i in range(top)]
        for got, id_ in want:
            got = float(got)
            if lp is None or not 0 <= id_ < V:
                assert np.isnan(got), (t, id_, got)
            elif lp[id_] < -np.finfo(np.float32).max:
                assert got == -np.inf  # -inf itself, and what an fp32 cannot hold (-6e38 rounds to -inf)
            else:
                # the differences to the maximum and to the log of the sum, each rounded; the sum of
                # rounded exponentials (2 steps each, half a step for each of ~64 levels of addition)
                assert abs(got - lp[id_]) <= 2 * EPS32 * (abs(lp[id_]) + 2 * np.log(V) + 1) + 80 * EPS32, (t, got, lp[id_])
        if ent:
            got = float(r.entropy[t])
            if lp is None:
                assert np.isnan(got)
            else:
                p = np.exp(lp)
                cond = (p * np.abs(np.where(p > 0, x[t].astype(np.float64) - x[t].max(), 0))).sum()
                assert abs(got - h) <= 160 * EPS32 * (cond + 1) + 2 * EPS32 * np.log(V), (t, got, h)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 160, 255, 1000, 4095, 4097, 9999, 33000])
@pytest.mark.parametrize("T", [1, 5])
def test_sizes(T, V):
    rng = np.random.default_rng(V + T)
    x = (rng.standard_normal((T, V)) * 3).astype(np.float32)
    for top in sorted({0, 1, min(V, 20), min(V, 64)}):
        check(x, rng.integers(0, V, T), top, pad=top % 7, offset=top % 3)


@pytest.mark.parametrize("T,top", [(1, 5), (3, 20), (32, 20), (70, 64), (300, 1), (600, 0)])
def test_vocabulary(T, top):
    rng = np.random.default_rng(T)
    V = 152064 if T < 100 else 20011
    x = (rng.standard_normal((T, V)) * 2).astype(np.float32)
    x[np.arange(T), rng.integers(0, V, T)] += 14
    check(x, rng.integers(0, V, T), top)


@pytest.mark.parametrize("V", [100, 5000, 152064])
def test_ties_and_orders(V):
    rng = np.random.default_rng(V)
    x = np.zeros((8, V), np.float32)
    x[1] = rng.integers(0, 3, V)
    x[2] = np.arange(V) / 16.0               # ascending: every value is a new maximum
    x[3] = -np.arange(V) / 16.0
    x[4] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    x[5, V // 2:] = 1.0                      # a border inside
    x[6] = -1e30
    x[7] = np.round(rng.standard_normal(V) * 4) / 4
    check(x, rng.integers(0, V, 8), 64)


@pytest.mark.parametrize("V", [70, 9000, 152064])
def test_masked_and_non_finite(V):
    rng = np.random.default_rng(V + 1)
    x = rng.standard_normal((9, V)).astype(np.float32)
    x[0, rng.random(V) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, V - 1] = -5.0                       # one token left
    x[2] = -np.inf                           # none
    x[3, V // 3] = np.inf
    x[4, V // 2] = np.nan
    x[4, V - 2] = -np.nan
    x[5] = np.finfo(np.float32).min          # masked by the type's lowest value
    x[6] = np.finfo(np.float32).min
    x[6, 3] = 2.0
    x[7] = 3e38
    x[7, 5] = -3e38
    x[8] *= 1e-30
    check(x, [0, V - 1, 1, 2, 3, 4, 3, 5, 8], 64)


def test_tokens_outside_and_optional_outputs():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((6, 3000)).astype(np.float32)
    check(x, [-1, 3000, 0, 2999, 2 ** 62, -2 ** 62], 3)
    check(x, None, 3, ent=False)
    check(x, None, 0)
    check(x, [1, 2, 3, 4, 5, 6], 0, ent=False)


def test_peaked_and_flat():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((4, 152064)).astype(np.float32)
    x[0, 77] = 60.0    # entropy near 0
    x[1] = 0.25        # log V
    x[2] *= 30
    x[3] += 1000
    check(x, [77, 0, 1, 2], 20)


def test_long_rows_with_many_alternatives():
    """More parts of a row than one step of the join holds."""
    rng = np.random.default_rng(9)
    x = (rng.standard_normal((2, 700001)) * 2).astype(np.float32)
    x[1] = np.round(x[1] * 4) / 4
    check(x, [5, 700000], 64)
    x[0, 300000] = np.nan
    check(x, [5, 700000], 64)


def test_more_elements_than_32_bits():
    """Rows past 2^31 floats from the first."""
    V, T = 160, 3
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((T, V)) * 3).astype(np.float32)
    ld = 2 ** 30 + 8
    big = torch.zeros(2 * ld + V, device="cuda")
    rows = torch.as_strided(big, (T, V), (ld, 1))
    rows.copy_(torch.from_numpy(x))
    tk = torch.tensor([1, 2, 3], device="cuda")
    a, b = ops.logprobs(rows, tk, top=7), ops.logprobs(rows.contiguous(), tk, top=7)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_same_bits_every_time():
    rng = np.random.default_rng(6)
    x = torch.from_numpy((rng.standard_normal((9, 152064)) * 3).astype(np.float32)).cuda()
    tk = torch.arange(9, device="cuda")
    a = ops.logprobs(x, tk, top=20)
    for _ in range(5):
        b = ops.logprobs(x, tk, top=20)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
