"""iq_attn_decode where its scores are extreme."""
import numpy as np
import pytest
import torch

from infer_amd import ops
from tests.kv_util import EPS32, Paged

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
