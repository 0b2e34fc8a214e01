"""A paged cache of any type for tests (random pages, the worst bytes wherever
no token lies) and plain forms of iq_kv_extend and iq_kv_read."""
import numpy as np
import torch

from infer_amd import ops
from tests.kv_util import EPS32

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CODES = (torch.int8, torch.float8_e4m3fn)


def encode(y, dtype):
    """float32 numpy values to codes (uint8 numpy), to nearest even."""
    y = np.clip(y, -LARGEST[dtype], LARGEST[dtype]).astype(np.float32)
    if dtype == torch.int8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    return torch.from_numpy(y).to(dtype).view(torch.uint8).numpy()


def decode(c, dtype):
    """Codes (uint8 numpy) to float32."""
    return torch.from_numpy(np.ascontiguousarray(c)).view(dtype).float().numpy()


class Pool:
    """B block-table rows of `width` pages each over a pool, in random order."""

    def __init__(self, rng, B, width, page, hk, d, dtype, block=None, order="slots", spare=2, device="cuda"):
        self.page, self.hk, self.d, self.dtype, self.block = page, hk, d, dtype, block
        self.pages = B * width + spare
        self.table_np = rng.permutation(self.pages)[:B * width].reshape(B, width).astype(np.int32)
        self.cap = width * page
        kv = [self.memory(order, device) for _ in range(2)]
        scales = (None, None)
        if dtype in CODES:
            nb = page // block
            scales = [torch.full((self.pages, nb, hk + 3), float("nan"), device=device)[:, :, 1:1 + hk] if order == "padded"
                      else torch.full((hk, self.pages, nb), float("nan"), device=device).permute(1, 2, 0) if order == "heads"
                      else torch.full((self.pages, nb, hk), float("nan"), device=device) for _ in range(2)]
        self.cache = ops.KvCache(*kv, *scales)
        self.table = torch.from_numpy(self.table_np).to(device)

    def memory(self, order, device):
        hk, d, page, pages = self.hk, self.d, self.page, self.pages
        bytes_ = torch.empty(0, dtype=self.dtype).element_size()
        shape = {"slots": (pages, page, hk, d), "heads": (pages, hk, page, d), "padded": (pages, page, hk * d + 48)}[order]
        # all ones: NaN in every floating type, -1 in int8
        t = torch.full((*shape[:-1], shape[-1] * bytes_), 255, dtype=torch.uint8, device=device).view(self.dtype)
        if order == "heads":
            return t.transpose(1, 2)
        if order == "padded":
            return t[:, :, 16:16 + hk * d].view(pages, page, hk, d)
        return t

    def where(self, b, tok):
        tok = np.asarray(tok)
        return self.table_np[b, tok // self.page].astype(np.int64), tok % self.page

    def raw(self):
        """Codes (or 16-bit values' bits) and scales of k and v, as numpy."""
        bits = torch.uint8 if self.dtype in CODES else torch.int16
        got = [t.view(bits).cpu().numpy().copy() for t in (self.cache.k, self.cache.v)]
        if self.dtype in CODES:
            got += [t.cpu().numpy().copy() for t in (self.cache.k_scales, self.cache.v_scales)]
        return got

    def values(self, b, tok):
        """K, V of these tokens as they lie in memory now, float64."""
        p, s = self.where(b, tok)
        raw = self.raw()
        if self.dtype in CODES:
            return [decode(c[p, s], self.dtype).astype(np.float64) * sc[p, s // self.block][..., None].astype(np.float64)
                    for c, sc in ((raw[0], raw[2]), (raw[1], raw[3]))]
        return [torch.from_numpy(c[p, s]).view(self.dtype).double().numpy() for c in raw]

    def fill(self, rng, lens, sd=1.0, spread=0.5):
        """Random tokens in the first lens[b] places (by the plain form)."""
        raw = self.raw()
        for x in range(2):
            for b, n in enumerate(lens):
                if n <= 0:
                    continue
                v = rng.standard_normal((n, self.hk, self.d)) * sd * np.exp(spread * rng.standard_normal((n, self.hk, 1)))
                v = v.astype(np.float32)
                p, s = self.where(b, np.arange(n))
                if self.dtype not in CODES:
                    raw[x][p, s] = torch.from_numpy(v).to(self.dtype).view(torch.int16).numpy()
                    continue
                for j in range(0, n, self.block):
                    extend_block(raw[x], raw[2 + x], self, b, j, v[j:j + self.block])
        self.put(raw)

    def put(self, raw):
        for t, a in zip((self.cache.k, self.cache.v), raw):
            t.view(torch.uint8 if self.dtype in CODES else torch.int16).copy_(torch.from_numpy(a))
        if self.dtype in CODES:
            for t, a in zip((self.cache.k_scales, self.cache.v_scales), raw[2:]):
                t.copy_(torch.from_numpy(a))


def new_scale(old, a, dtype):
    """The scale of a block with scale `old` (0: a new one) that receives values
    up to a, and how often it doubled; in fp32, as documented."""
    Q = LARGEST[dtype]
    if not np.isfinite(a) or not np.isfinite(old):
        return np.float32(np.nan), 0
    if old == 0:
        return (np.float32(0) if a == 0 else max(np.float32(a) / np.float32(Q), np.float32(2.0 ** -126))), 0
    up = 0
    while float(a) > Q * float(old) * 2.0 ** up:
        up += 1
    return np.float32(float(old) * 2.0 ** up), up


def extend_block(codes, scales, pool, b, tok, x):
    """x [n, hk, d] float32 to the tokens tok.. of one block, in place."""
    begin = tok // pool.block * pool.block
    p, s0 = (int(t) for t in pool.where(b, begin))
    j = s0 // pool.block
    for h in range(pool.hk):
        old = np.float32(0) if tok == begin else scales[p, j, h]
        a = np.abs(x[:, h]).max()
        s, up = new_scale(old, a, pool.dtype)
        if up:
            rows = slice(s0, s0 + tok - begin)
            codes[p, rows, h] = encode(np.ldexp(decode(codes[p, rows, h], pool.dtype), -up), pool.dtype)
        scales[p, j, h] = s
        at = s0 + tok - begin
        with np.errstate(all="ignore"):
            y = x[:, h] / s if s > 0 else np.zeros_like(x[:, h])
        codes[p, at:at + len(x), h] = encode(y, pool.dtype)


def extend_plain(pool, raw, x, lens, counts, which):
    """The plain form on raw (k: which 0, v: 1), x [T, hk, d] float32 as it is
    stored (normed and turned)."""
    t = 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        mine = x[t:t + m]
        t += m
        if n < 0 or n > pool.cap:
            continue
        mine = mine[:max(0, pool.cap - n)]
        span = pool.block if pool.dtype in CODES else 1
        i = 0
        while i < len(mine):
            tok = n + i
            k = min(len(mine) - i, (tok // span + 1) * span - tok)
            if 0 <= pool.table_np[b, tok // pool.page] < pool.pages:
                if pool.dtype in CODES:
                    extend_block(raw[which], raw[2 + which], pool, b, tok, mine[i:i + k])
                else:
                    p, s = pool.where(b, [tok])
                    raw[which][p, s] = torch.from_numpy(mine[i:i + 1]).to(pool.dtype).view(torch.int16).numpy()
            i += k


def norm_f64(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def made_slack(x, w, half):
    """How far a normed and turned value may be off, from the exact normed row
    x [.., d]: the squares are summed in 64 bits, so a norm is 2 roundings (the
    root's product, the norm's), and a turn 2 products of values with cosines
    that are off by 2 half steps of 1 (their argument, a fraction of a turn up
    to pi, to 2^-23 of pi; 4 half steps with the function's own), and a sum."""
    mate = np.concatenate([x[..., half:2 * half], x[..., :half], x[..., 2 * half:]], -1)
    turned = np.arange(x.shape[-1]) < 2 * half
    return ((2 if w is not None else 0) + np.where(turned, 12, 0)) * EPS32 * (np.abs(x) + np.where(turned, np.abs(mate), 0))
