"""The operators around a decode step's cache in its smaller and shorter
forms: caches of 8 bits, and attention that sees only some of the tokens.

    extend  new tokens behind what each sequence has cached: optional norms of
            q and k for each head and the rotary embedding in the same pass,
            k and v rounded into their pages; an 8-bit cache has a scale for
            each block of tokens and key/value head
    read    cached tokens back as rows of numbers
    attn8   attention of one token a sequence over an 8-bit cache
    window  the same over the newest tokens and a few first ones, any cache

Each case is one eager call (extend with "read" is two: a chunk of a prompt,
and the cache read back for the chunk's own attention) at sizes of the models
that bench.py and the tests run (Qwen2.5-1.5B / 7B heads), or of generic size;
`draw` gives further cases of the same ranges.  With `own` false, `run` is
plain torch in 32 bits; with `own` true it makes the library's calls.

    listed()             the cases
    draw(rng)            one more case of their ranges
    prepare(case, seed)  inputs on the device, from the seed alone
    run(state)           one pass; its outputs
    work(case)           bytes and operations that the call cannot do without
    exact(case, seed)    the outputs in 64 bits
"""
import math
import random

import numpy as np
import torch

own = False

# query heads, key/value heads, head size (bench.py)
MODELS = {
    "1.5b": dict(heads=12, kv_heads=2, dim=128),
    "7b": dict(heads=28, kv_heads=4, dim=128),
}
THETA, EPS = 1e6, 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}  # of the codes
OUTS = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# the most that a drawn case reads
MOST_CACHED = 131072 * 4 * 128
MOST_READ = 8 * 8192 * 4 * 128
MOST_ROWS = 2048


def listed():
    m7, m1 = MODELS["7b"], MODELS["1.5b"]
    return [
        # Every layer of a decode step for a batch of users: launch cost.
        dict(name="extend-7b-e4m3-16x1", op="extend", type="e4m3", page=16, block=16, B=16, new=1, len=700, norm=False,
             read="", far=32768, **m7),
        # The same with norms of the heads, over 16 bits.
        dict(name="extend-norm-7b-bf16-32x1", op="extend", type="bf16", page=16, block=0, B=32, new=1, len=300,
             norm=True, read="", far=32768, **m7),
        # Three prompts' chunks, of odd lengths, pages that no tile divides.
        dict(name="extend-norm-1.5b-e4m3-3x681", op="extend", type="e4m3", page=24, block=8, B=3, new=681, len=900,
             norm=True, read="", far=131072, **m1),
        # A prompt's chunk, and everything so far read back for its attention.
        dict(name="extend-read-7b-int8-4x509", op="extend", type="int8", page=64, block=32, B=4, new=509, len=1500,
             norm=False, read="bf16", far=32768, **m7),
        # One short sequence taken out of the cache.
        dict(name="read-1.5b-int8-1x777-fp32", op="read", type="int8", page=16, block=16, B=1, len=777, read="fp32",
             **m1),
        # A batch of long ones.
        dict(name="read-7b-e4m3-8x8192-bf16", op="read", type="e4m3", page=64, block=64, B=8, len=8192, read="bf16",
             **m7),
        # The first tokens of an answer to a short prompt: launch cost.
        dict(name="attn8-7b-int8-1x17", op="attn8", type="int8", page=16, block=16, B=1, len=17, ragged=False, **m7),
        # One user with a very long context: the length has to be split.
        dict(name="attn8-7b-int8-1x131072", op="attn8", type="int8", page=64, block=32, B=1, len=131072, ragged=False,
             **m7),
        # A full decode batch of sequences of very different ages.
        dict(name="attn8-1.5b-e4m3-32x8192-ragged", op="attn8", type="e4m3", page=16, block=16, B=32, len=8192,
             ragged=True, **m1),
        # A key/value head for every query head, short rows, odd pages, a scale a token.
        dict(name="attn8-16h64-int8-24x2047", op="attn8", type="int8", page=24, block=1, B=24, len=2047, ragged=True,
             heads=16, kv_heads=16, dim=64),
        # A batch of long sequences of which each sees its newest part.
        dict(name="window-7b-bf16-16x16384", op="window", type="bf16", page=16, block=0, B=16, len=16384, ragged=True,
             window=4096, sinks=4, **m7),
        # One user's very long chat under a short window: launch cost.
        dict(name="window-1.5b-int8-1x131072", op="window", type="int8", page=64, block=16, B=1, len=131072,
             ragged=False, window=1000, sinks=17, **m1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn_heads(rng):
    r = rng.random()
    if r < 0.6:
        return MODELS["7b" if r < 0.3 else "1.5b"]
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv, dim=rng.choice([32, 64, 80, 96, 128]))


def draw(rng):
    op = rng.choice(["extend", "extend", "read", "attn8", "attn8", "window"])
    t = rng.choice(["int8", "e4m3"] if op == "attn8" else ["int8", "e4m3", "int8", "e4m3", "bf16", "fp16"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 100])
    block = rng.choice([n for n in (1, 2, 4, 8, 16, 24, 25, 32, 50, 64, 100) if page % n == 0]) if t in LARGEST else 0
    base = dict(op=op, type=t, page=page, block=block, **_drawn_heads(rng))
    row = base["kv_heads"] * base["dim"]
    if op == "extend":
        B = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, MOST_ROWS // B)
        return dict(B=B, new=new, len=_log_int(rng, 1, min(4000, max(2, MOST_READ // 4 // row // B))),
                    norm=rng.random() < 0.5, read=rng.choice(["", "", "bf16"]) if t != "int8" else "bf16",
                    far=_log_int(rng, 4096, 131072), **base)
    if op == "read":
        n = _log_int(rng, 1, 16384)
        return dict(B=_log_int(rng, 1, max(1, min(64, MOST_READ // row // n))), len=n, read=rng.choice(sorted(OUTS)),
                    **base)
    most = MOST_CACHED // row
    n = _log_int(rng, 1, min(131072, most))
    c = dict(B=_log_int(rng, 1, max(1, min(64, most // n))), len=n, ragged=rng.random() < 0.5, **base)
    if op == "window":
        c.update(window=_log_int(rng, 1, 2 * n), sinks=rng.choice([0, 0, 1, 4, rng.randrange(1, 100)]))
    return c


def _spread(case, n, least=1):
    """B whole numbers up to n, one of them n and (of several) one the least."""
    B = case["B"]
    rng = random.Random(1000003 * B + n)
    got = [_log_int(rng, max(1, least), n) if rng.random() < 0.5 else rng.randrange(least, n + 1) for _ in range(B)]
    got[rng.randrange(B)] = n
    if B > 1:
        got[(got.index(n) + 1) % B] = least
    return got


def lengths(case):
    """The sequences' cached tokens before the call."""
    if case["op"] in ("extend", "read"):
        return _spread(case, case["len"], 0 if case["op"] == "extend" else 1)
    return _spread(case, case["len"]) if case["ragged"] else [case["len"]] * case["B"]


def added(case):
    """The tokens that an extend adds to each sequence."""
    return [1] * case["B"] if case["new"] == 1 else _spread(case, case["new"])


def seen(case):
    """How many tokens each sequence's attention sees."""
    if case["op"] != "window":
        return lengths(case)
    return [min(n, case["window"] + case["sinks"]) for n in lengths(case)]


def _rand(gen, *shape, sd=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * sd


class State:
    pass


def _codes(x, scale, t):
    """x / scale to the nearest code of type t."""
    y = (x / torch.where(scale > 0, scale, 1.0)).clamp(-LARGEST[t], LARGEST[t])
    return y.round().to(torch.int8) if t == "int8" else y.to(torch.float8_e4m3fn)


def _pool(case, gen, pages):
    """A pool of random values, and its scales (a block's largest value / the
    largest code)."""
    x = _rand(gen, pages, case["page"], case["kv_heads"], case["dim"])
    t = case["type"]
    if t not in LARGEST:
        return x.to(TYPES[t]), None
    blocks = x.view(pages, case["page"] // case["block"], case["block"], case["kv_heads"], case["dim"])
    scale = blocks.abs().amax((2, 4)) / LARGEST[t]
    return _codes(blocks, scale[:, :, None, :, None], t).view(x.shape), scale


def _cache(s, case, gen, tokens):
    """Pages for sequences of this many tokens, in random order, with a few
    spare ones; table entries past a sequence's pages are -1."""
    page = case["page"]
    need = [max(1, -(-n // page)) for n in tokens]
    pages = sum(need) + 3
    (s.k, s.ks), (s.v, s.vs) = _pool(case, gen, pages), _pool(case, gen, pages)
    order = torch.randperm(pages, generator=gen, device="cuda")[: sum(need)].to(torch.int32)
    at = np.concatenate([i * max(need) + np.arange(m) for i, m in enumerate(need)])
    table = torch.full((len(tokens) * max(need),), -1, dtype=torch.int32, device="cuda")
    table[torch.from_numpy(at).cuda()] = order
    s.table = table.view(len(tokens), max(need))


def _starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.case = case
    op, hk, hq, d = case["op"], case["kv_heads"], case["heads"], case["dim"]
    lens = lengths(case)
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if op == "extend":
        new = added(case)
        T = s.T = sum(new)
        _cache(s, case, gen, [a + b for a, b in zip(lens, new)])
        s.starts = None if case["new"] == 1 else _starts(new)
        # tokens differ in size: some exceed what their block has held so far
        s.q, s.vn = _rand(gen, T, hq, d), _rand(gen, T, hk, d) * torch.exp(_rand(gen, T, 1, 1, sd=0.5))
        s.kn = _rand(gen, T, hk, d, sd=2.0) * torch.exp(_rand(gen, T, 1, 1, sd=0.5))
        s.positions = torch.randint(0, case["far"], (T,), generator=gen, device="cuda")
        s.freqs = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
        s.q_norm = s.k_norm = None
        if case["norm"]:
            s.q_norm = (1 + _rand(gen, d, sd=0.2)).to(torch.bfloat16)
            s.k_norm = (1 + _rand(gen, d, sd=0.2)).to(torch.bfloat16)
        s.q_out = torch.empty_like(s.q)
        if case["read"]:  # everything that each sequence then has
            s.all, s.rows = _starts([a + b for a, b in zip(lens, new)]), sum(lens) + T
    elif op == "read":
        _cache(s, case, gen, lens)
        s.all, s.rows = _starts(lens), sum(lens)
    else:
        _cache(s, case, gen, lens)
        s.q = _rand(gen, case["B"], hq, d, sd=1.5)
        s.out = torch.empty_like(s.q)
    if case.get("read"):
        s.out = tuple(torch.empty(s.rows, hk, d, dtype=OUTS[case["read"]], device="cuda") for _ in range(2))
    if own:
        from infer_amd import ops
        s.cache = ops.KvCache(s.k, s.v, s.ks, s.vs)
    return s


def run(s):
    c = s.case
    if c["op"] == "extend":
        r = {"q": _extend_own(s) if own else _extend(s)}
        if s.ks is not None:
            r.update(ks=s.ks, vs=s.vs)
        if c["read"]:
            r["k"], r["v"] = _read_own(s) if own else _read(s)
        else:
            r.update(k=s.k, v=s.v)
        return r
    if c["op"] == "read":
        k, v = _read_own(s) if own else _read(s)
        return {"k": k, "v": v}
    return _attn_own(s) if own else _attn(s)


# ------------------------------------------------------- the library's calls
def _extend_own(s):
    from infer_amd import ops
    return ops.kv_extend(s.q, s.kn, s.vn, s.positions, s.freqs, s.cache, s.table, s.lens, starts=s.starts,
                         q_norm=s.q_norm, k_norm=s.k_norm, eps=EPS, q_out=s.q_out)


def _read_own(s):
    from infer_amd import ops
    return ops.kv_read(s.cache, s.table, s.all, out=s.out)


def _attn_own(s):
    from infer_amd import ops
    c = s.case
    return ops.attn_decode(s.q, s.cache, s.table, s.lens, out=s.out, window=c.get("window", 0), sinks=c.get("sinks", 0))


# ------------------------------------------------------------- plain forms
def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, cos, sin):
    """Pairs (i, i + d/2) of every head turned by the row's angles."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _owners(starts, B, T):
    """Each row's sequence, and its place among that sequence's rows."""
    if starts is None:
        b = torch.arange(B, device="cuda")
        return b, torch.zeros_like(b)
    b = torch.repeat_interleave(torch.arange(B, device="cuda"), (starts[1:] - starts[:-1]).long(), output_size=T)
    return b, torch.arange(T, device="cuda") - starts[b]


def _extend(s):
    c = s.case
    page, block, t = c["page"], c["block"], c["type"]
    ang = s.positions[:, None].double() * s.freqs  # far positions lose their angle in 32 bits
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    q, k = _rotate(_normed(s.q, s.q_norm), cos, sin), _rotate(_normed(s.kn, s.k_norm), cos, sin)
    b, i = _owners(s.starts, c["B"], s.T)
    tok = s.lens[b].long() + i
    pg, slot = s.table[b, tok // page].long(), tok % page
    if t not in LARGEST:
        s.k[pg, slot], s.v[pg, slot] = k.to(s.k.dtype), s.vn.to(s.v.dtype)
        return q
    # the block that each sequence's first new token falls into may hold older ones
    n0 = s.lens.long()
    pg0, blk0 = s.table.gather(1, (n0 // page)[:, None])[:, 0].long(), n0 % page // block
    older = n0 % block
    slots0 = blk0[:, None] * block + torch.arange(block, device="cuda")
    stays = torch.arange(block, device="cuda") < older[:, None]
    for x, codes, scales in ((k, s.k, s.ks), (s.vn, s.v, s.vs)):
        nb = page // block
        most = torch.zeros(scales.shape[0] * nb, c["kv_heads"], device="cuda")
        at = pg * nb + slot // block
        most.scatter_reduce_(0, at[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
        # a new block's scale comes from its values; an older one's doubles until they fit
        had = torch.zeros_like(most)
        had[pg0 * nb + blk0] = torch.where(older[:, None] > 0, scales[pg0, blk0], 0.0)
        need = most.double() / (LARGEST[t] * had.double().clamp(min=1e-300))
        mant, e = torch.frexp(need)
        up = torch.where((had > 0) & (need > 1), e - (mant == 0.5).int(), 0)
        scale = torch.where(had > 0, torch.ldexp(had, up), (most / LARGEST[t]).clamp(min=2.0 ** -126) * (most > 0))
        moved = torch.ldexp(codes.view(torch.uint8)[pg0[:, None], slots0].view(codes.dtype).float(),
                            -up[pg0 * nb + blk0][:, None, :, None])
        moved = moved.round().to(torch.int8) if t == "int8" else moved.to(torch.float8_e4m3fn)
        raw = codes.view(torch.uint8)
        raw[pg0[:, None], slots0] = torch.where(stays[:, :, None, None], moved.view(torch.uint8),
                                                raw[pg0[:, None], slots0])
        scales[pg, slot // block] = scale[at]
        raw[pg, slot] = _codes(x, scale[at][..., None], t).view(torch.uint8)
    return q


def _values(s, codes, scales, pg, slot):
    """The numbers that lie at these places, in 32 bits."""
    if scales is None:
        return codes[pg, slot].float()
    x = codes.view(torch.uint8)[pg, slot].view(codes.dtype).float()
    return x * scales[pg, slot // s.case["block"]][..., None]


def _read(s):
    page = s.case["page"]
    b, tok = _owners(s.all, s.case["B"], s.rows)
    pg, slot = s.table[b, tok // page].long(), tok % page
    for to, codes, scales in zip(s.out, (s.k, s.v), (s.ks, s.vs)):
        to.copy_(_values(s, codes, scales, pg, slot))
    return s.out


def _attn(s):
    c = s.case
    B, hk, g, d, page = s.q.shape[0], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["page"]
    cap = s.table.shape[1] * page
    n = s.lens.long()[:, None]
    tok = torch.arange(cap, device="cuda").expand(B, cap)
    live = tok < n
    if c["op"] == "window" and c["window"] + c["sinks"] < cap:
        # the first `sinks` tokens and the newest `window`
        i = torch.arange(c["window"] + c["sinks"], device="cuda").expand(B, -1)
        gap = (n - c["window"] - c["sinks"]).clamp(min=0)
        tok = torch.where(i < c["sinks"], i, i + gap)
        live = tok < n
    pg, slot = s.table.gather(1, (tok // page).clamp(max=s.table.shape[1] - 1)).long().clamp(min=0), tok % page
    zero = torch.zeros((), device="cuda")
    K = _values(s, s.k, s.ks, pg, slot).permute(0, 2, 3, 1).contiguous()
    V = torch.where(live[:, :, None, None], _values(s, s.v, s.vs, pg, slot), zero).transpose(1, 2).contiguous()
    sc = torch.matmul(s.q.view(B, hk, g, d), K) * d ** -0.5
    sc = torch.where(live[:, None, None], sc, torch.full((), -math.inf, device="cuda"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, V).view(B, c["heads"], d)


# ---------------------------------------------------------------- 64 bits
def _decoded(codes, scales, block):
    x = codes.float().double()
    if scales is None:
        return x
    return x * scales.double().repeat_interleave(block, 1)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    op, hk, d, page, block, t = (case[x] for x in ("op", "kv_heads", "dim", "page", "block", "type"))
    lens = lengths(case)
    if op == "read":
        K, V = _decoded(s.k, s.ks, block), _decoded(s.v, s.vs, block)
        out = {"k": [], "v": []}
        for b, n in enumerate(lens):
            i = torch.arange(n, device="cuda")
            for name, x in (("k", K), ("v", V)):
                out[name].append(x[s.table[b].long()[i // page], i % page])
        return {name: torch.cat(x) for name, x in out.items()}
    if op == "extend":
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s.positions[:, None, None] * s.freqs)

        def made(x, w):
            x = x.double()
            if w is not None:
                x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
            z = torch.complex(x[..., : d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        r = {"q": made(s.q, s.q_norm)}
        first = np.concatenate([[0], np.cumsum(added(case))])
        for name, x, codes, scales in (("k", made(s.kn, s.k_norm), s.k, s.ks), ("v", s.vn.double(), s.v, s.vs)):
            codes, got = codes.float().double(), None if scales is None else scales.double()
            for b, n in enumerate(lens):
                m = added(case)[b]
                i = torch.arange(n, n + m, device="cuda")
                pg, slot = s.table[b].long()[i // page], i % page
                mine = x[first[b]:first[b] + m]
                if got is None:
                    codes[pg, slot] = mine
                    continue
                # blocks of the sequence that the new tokens touch, padded with nothing to whole ones
                j0, j1 = n // block, (n + m - 1) // block
                whole = torch.zeros((j1 - j0 + 1) * block, hk, d, dtype=torch.float64, device="cuda")
                whole[n - j0 * block: n - j0 * block + m] = mine
                scale = whole.view(-1, block, hk, d).abs().amax((1, 3)) / LARGEST[t]
                at = torch.arange(j0, j1 + 1, device="cuda") * block
                apg, ablk = s.table[b].long()[at // page], at % page // block
                if n % block:
                    had = got[apg[0], ablk[0]]
                    up = torch.log2(scale[0] / had).ceil().clamp(min=0)
                    scale[0] = had * 2 ** up
                    o = torch.arange(j0 * block, n, device="cuda") % page
                    y = codes[apg[0], o] / 2 ** up[:, None]
                    codes[apg[0], o] = y.round() if t == "int8" else y.float().to(TYPES[t]).double()
                got[apg, ablk] = scale
                y = mine / scale[(i // block - j0)][..., None]
                codes[pg, slot] = y.round() if t == "int8" else y.float().clamp(-448, 448).to(TYPES[t]).double()
            if got is not None:
                r[name + "s"] = got
            if case["read"]:
                vals = codes if got is None else codes * got.repeat_interleave(block, 1)[..., None]
                rows = []
                for b, n in enumerate(lens):
                    i = torch.arange(n + added(case)[b], device="cuda")
                    rows.append(vals[s.table[b].long()[i // page], i % page])
                codes = torch.cat(rows)
            r[name] = codes
        return r
    g = case["heads"] // hk
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        i = torch.arange(n, device="cuda")
        if op == "window":
            i = i[(i < case["sinks"]) | (i >= n - case["window"])]
        pg, slot = s.table[b].long()[i // page], i % page
        K, V = s.k.view(torch.uint8 if block else s.k.dtype)[pg, slot], s.v.view(torch.uint8 if block else s.v.dtype)[pg, slot]
        K, V = K.view(s.k.dtype).float().double(), V.view(s.v.dtype).float().double()
        if block:
            K, V = K * s.ks[pg, slot // block].double()[..., None], V * s.vs[pg, slot // block].double()[..., None]
        for h in range(hk):
            p = torch.softmax(s.q[b, h * g:(h + 1) * g].double() @ K[:, h].t() / math.sqrt(d), 1)
            out[b, h * g:(h + 1) * g] = p @ V[:, h]
    return out


def work(case):
    op, hq, hk, d, block = case["op"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    size = 1 if block else 2
    # codes and scales of one token's k and v
    token = 2 * hk * (d * size + (4 / block if block else 0))
    if op == "extend":
        T, n = sum(added(case)), sum(lengths(case))
        b, f = T * (4 * d * (2 * hq + 2 * hk) + 8) + T * token, T * d * (3 * hq + 6 * hk + 4 * (hq + hk) * case["norm"])
        if case["read"]:
            rows = T + n
            b, f = b + rows * (token + 2 * hk * d * 2), f + 2 * rows * hk * d
        return dict(bytes=b, flops=f)
    if op == "read":
        rows = sum(lengths(case))
        return dict(bytes=rows * (token + 2 * hk * d * (4 if case["read"] == "fp32" else 2)), flops=2 * rows * hk * d)
    total = sum(seen(case))
    return dict(bytes=total * token + 8 * case["B"] * hq * d + 4 * (total // case["page"] + case["B"]),
                flops=4 * total * hq * d)
