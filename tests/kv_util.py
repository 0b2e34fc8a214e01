"""A paged cache for tests of the decode-step operators (random pages, NaN
wherever no token lies) and plain 64-bit forms of the operators."""
import numpy as np
import torch

from infer_amd import ops

EPS32 = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Paged:
    """Sequences of lengths `lens` in pages of a pool.  order "slots": memory
    [pages, page_size, heads, dim]; "heads": [pages, heads, page_size, dim];
    "padded": rows of heads * dim + 24 values inside a larger tensor."""

    def __init__(self, rng, lens, hk, d, page, dtype, order="slots", spare=2, room=0, fill=float("nan"), device="cuda"):
        self.lens, self.hk, self.d, self.page, self.dtype = list(lens), hk, d, page, dtype
        B = len(lens)
        need = [-(-(max(0, n) + room) // page) for n in lens]
        self.width = max(1, max(need))
        pages = sum(need) + spare
        ids = rng.permutation(pages)
        self.table_np = np.full((B, self.width), -7, np.int32)
        at = 0
        for b, m in enumerate(need):
            self.table_np[b, :m] = ids[at:at + m]
            at += m
        kv = [self.memory(pages, order, fill, device) for _ in range(2)]
        self.cache = ops.KvCache(*kv)
        self.K, self.V = [], []  # per sequence [n, hk, d], the values as stored
        for b, n in enumerate(lens):
            for store, t, sd in ((self.K, kv[0], 1.0), (self.V, kv[1], 1.0)):
                x = torch.from_numpy((rng.standard_normal((max(0, n), hk, d)) * sd).astype(np.float32)).to(dtype)
                store.append(x)
                if n > 0:
                    p, s = self.where(b, np.arange(n))
                    t[p.to(device), s.to(device)] = x.to(device)
        self.table = torch.from_numpy(self.table_np).to(device)
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device=device)

    def memory(self, pages, order, fill, device):
        hk, d, page = self.hk, self.d, self.page
        if order == "heads":
            return torch.full((pages, hk, page, d), fill, dtype=self.dtype, device=device).transpose(1, 2)
        if order == "padded":
            t = torch.full((pages, page, hk * d + 24), fill, dtype=self.dtype, device=device)
            return t[:, :, 8:8 + hk * d].view(pages, page, hk, d)
        return torch.full((pages, page, hk, d), fill, dtype=self.dtype, device=device)

    def where(self, b, tok):
        tok = np.asarray(tok)
        return (torch.from_numpy(self.table_np[b, tok // self.page].astype(np.int64)),
                torch.from_numpy((tok % self.page).astype(np.int64)))

    def read(self, b, n):
        """The first n tokens' K and V as they lie in memory now."""
        p, s = self.where(b, np.arange(n))
        return [t[p.to(t.device), s.to(t.device)].cpu() for t in (self.cache.k, self.cache.v)]


def attn_f64(q, K, V, scale):
    """q [heads, d], K, V [n, hk, d] (float64 numpy): out, p [heads, n], the
    conditioning sums sum |q k| (largest over tokens, per head) and sum p |v|."""
    hq, d = q.shape
    n, hk, _ = K.shape
    g = hq // hk
    out, cv = np.zeros((hq, d)), np.zeros((hq, d))
    p, ck = np.zeros((hq, n)), np.zeros(hq)
    if n == 0:
        return out, p, ck, cv
    for h in range(hq):
        k, v = K[:, h // g], V[:, h // g]
        s = scale * (k @ q[h])
        e = np.exp(s - s.max())
        p[h] = e / e.sum()
        out[h], cv[h] = p[h] @ v, p[h] @ np.abs(v)
        ck[h] = (abs(scale) * (np.abs(k) @ np.abs(q[h]))).max()
    return out, p, ck, cv


def attn_rel(d, ck):
    """Relative error of a softmax weight: a score is a sum of d products in
    fp32 (d roundings that add up like sqrt(d), each half a step of the running
    sum, at most the conditioning sum; factor 4 for the largest of many) and
    one more of the scaling, exp moves by the score's absolute error, in
    numerator and sum; 64 half steps for exp, the sums over tokens in blocks
    and the division."""
    return 2 * (4 * np.sqrt(d) + 2) * EPS32 * ck + 64 * EPS32


def sum_order(w):
    """Positions by sum descending, ties and NaN (lowest) by position."""
    key = np.where(np.isnan(w), -np.inf, w.astype(np.float64))
    nan_last = np.isnan(w).astype(np.int64)
    return np.lexsort((np.arange(len(w)), -key, nan_last))


def evict_moves(w, budget, recent):
    """Source slot of every slot below budget."""
    n = len(w)
    old, cut = n - recent, budget - recent
    keep = np.sort(sum_order(w[:old])[:cut])
    src = np.full(budget, -1, np.int64)
    low = keep[keep < cut]
    src[low] = low
    free = np.flatnonzero(src[:cut] < 0)
    src[free] = keep[keep >= cut]
    src[cut:] = np.arange(old, n)
    return src


def rope_f64(x, pos, freqs, rot):
    """x [T, heads, d] float64."""
    y = x.copy()
    h = rot // 2
    a = pos[:, None, None].astype(np.float64) * freqs
    c, s = np.cos(a), np.sin(a)
    y[..., :h] = x[..., :h] * c - x[..., h:rot] * s
    y[..., h:rot] = x[..., h:rot] * c + x[..., :h] * s
    return y


def logprobs_f64(x):
    """x [V] float32: log probabilities and entropy in 64 bits; None without a
    distribution."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
        return None, None
    e = np.exp(x - x.max())
    lp = x - x.max() - np.log(e.sum())
    p = e / e.sum()
    return lp, -(p[p > 0] * lp[p > 0]).sum()


def top_order(x, k):
    """Ids by value descending, NaN first, ties by id."""
    nan = np.isnan(x)
    key = np.where(nan, np.inf, x.astype(np.float64))
    return np.lexsort((np.arange(len(x)), -key, ~nan))[:k]
