"""The operators of a decode step around the quantised linears: the paged
key/value cache, the attention of one new token over it, eviction from it by
accumulated attention weight, and the log probabilities of the answer.

    append    rotary embedding of q and k, k and v rounded into their pages
    attn      attention of one token a sequence over its pages (grouped
              heads), optionally adding each cached token's weight to a sum
    evict     the cache of every key/value head cut to a budget: the newest
              tokens and those of the largest accumulated weight stay
    logprobs  log probability of given tokens, entropy, the top alternatives

Each case is one eager call at sizes of the models that bench.py and the
tests run (Qwen2.5-1.5B / 7B heads and vocabularies), or of generic size;
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

# query heads, key/value heads, head size, vocabulary (bench.py)
MODELS = {
    "1.5b": dict(heads=12, kv_heads=2, dim=128, vocab=151936),
    "7b": dict(heads=28, kv_heads=4, dim=128, vocab=152064),
}
THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# the most that a drawn case reads: cached values, logits, appended rows
MOST_CACHED = 131072 * 4 * 128
MOST_LOGITS = 999 * 152064
MOST_ROWS = 1021


def _heads(model):
    m = MODELS[model]
    return dict(heads=m["heads"], kv_heads=m["kv_heads"], dim=m["dim"])


def listed():
    return [
        # Every layer of a decode step for a full batch of users: launch cost.
        dict(name="append-7b-bf16-16tok", op="append", type="bf16", page=16, T=16, far=32768, **_heads("7b")),
        # One chunk of a prompt, of an odd length, pages that no tile divides.
        dict(name="append-1.5b-fp16-1021tok", op="append", type="fp16", page=24, T=1021, far=131072,
             **_heads("1.5b")),
        # The first tokens of an answer to a short prompt: launch cost.
        dict(name="attn-7b-bf16-1x17", op="attn", type="bf16", page=16, B=1, len=17, ragged=False, weights=False,
             **_heads("7b")),
        # One user with a very long context: the length has to be split.
        dict(name="attn-7b-bf16-1x131072", op="attn", type="bf16", page=64, B=1, len=131072, ragged=False,
             weights=False, **_heads("7b")),
        # A full decode batch of sequences of very different ages.
        dict(name="attn-1.5b-bf16-32x8192-ragged", op="attn", type="bf16", page=16, B=32, len=8192, ragged=True,
             weights=False, **_heads("1.5b")),
        # A key/value head for every query head, short rows, an odd page size.
        dict(name="attn-16h64-fp16-24x2047", op="attn", type="fp16", page=24, B=24, len=2047, ragged=True,
             weights=False, heads=16, kv_heads=16, dim=64),
        # Attention that also accumulates what an eviction goes by.
        dict(name="attn-weights-7b-bf16-8x4113", op="attn", type="bf16", page=16, B=8, len=4113, ragged=False,
             weights=True, **_heads("7b")),
        # A running batch cut back by a few pages.
        dict(name="evict-7b-bf16-16x2112", op="evict", type="bf16", page=16, B=16, len=2112, budget=2048, recent=256,
             **_heads("7b")),
        # One long prompt cut to a quarter.
        dict(name="evict-1.5b-fp16-1x32768", op="evict", type="fp16", page=64, B=1, len=32768, budget=8192,
             recent=1000, **_heads("1.5b")),
        # One user's next token with a few alternatives: launch cost.
        dict(name="logprobs-151936-1row-top5", op="logprobs", T=1, V=151936, top=5),
        # A decode batch with the most alternatives that clients ask for.
        dict(name="logprobs-152064-32rows-top20", op="logprobs", T=32, V=152064, top=20),
        # Scoring a prompt: every position's logits, no alternatives.
        dict(name="logprobs-152064-999rows", op="logprobs", T=999, V=152064, top=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn_heads(rng):
    r = rng.random()
    if r < 0.35:
        return _heads("7b")
    if r < 0.7:
        return _heads("1.5b")
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), kv_heads=kv, dim=rng.choice([32, 64, 80, 96, 128]))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "evict", "logprobs"])
    if op == "logprobs":
        V = rng.choice([151936, 152064, rng.randrange(160, 60000)])
        T = _log_int(rng, 1, min(2048, max(1, MOST_LOGITS // V)))
        return dict(op=op, T=T, V=V, top=rng.choice([0, 1, 5, rng.randrange(2, 21)]))
    base = dict(type=rng.choice(["bf16", "fp16"]), page=rng.choice([1, 8, 16, 24, 32, 64, 100]), **_drawn_heads(rng))
    if op == "append":
        return dict(op=op, T=_log_int(rng, 1, MOST_ROWS), far=_log_int(rng, 64, 131072), **base)
    most = MOST_CACHED // (base["kv_heads"] * base["dim"])
    if op == "attn":
        n = _log_int(rng, 1, min(131072, most))
        B = _log_int(rng, 1, max(1, min(64, most // n)))
        return dict(op=op, B=B, len=n, ragged=rng.random() < 0.5, weights=rng.random() < 0.3, **base)
    n = _log_int(rng, 64, 32768)
    B = _log_int(rng, 1, max(1, min(64, most // 4 // n)))
    budget = rng.randrange(max(1, n // 8), n)
    return dict(op=op, B=B, len=n, budget=budget, recent=rng.randrange(0, budget + 1), **base)


def lengths(case):
    """The sequences' lengths: all equal, or of very different ages (the
    longest `len`, one of a single token)."""
    B, n = case["B"], case["len"]
    if not case.get("ragged"):
        return [n] * B
    rng = random.Random(1000003 * B + n)
    got = [_log_int(rng, 1, n) if rng.random() < 0.5 else rng.randrange(1, n + 1) for _ in range(B)]
    got[rng.randrange(B)] = n
    if B > 1:
        got[(got.index(n) + 1) % B] = 1
    return got


def _rand(gen, *shape, sd=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * sd


class State:
    pass


def _cache(s, case, gen, lens):
    """Pages for sequences of these lengths, in random order, with a few
    spare ones; table entries past a sequence's pages are -1."""
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + 3
    dt = TYPES[case["type"]]
    s.k = _rand(gen, pages, page, hk, d).to(dt)
    s.v = _rand(gen, pages, page, hk, d).to(dt)
    order = torch.randperm(pages, generator=gen, device="cuda")[: sum(need)].to(torch.int32)
    at = np.concatenate([i * max(need) + np.arange(m) for i, m in enumerate(need)])
    table = torch.full((len(lens) * max(need),), -1, dtype=torch.int32, device="cuda")
    table[torch.from_numpy(at).cuda()] = order
    s.table = table.view(len(lens), max(need))
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.case = case
    op = case["op"]
    if op == "logprobs":
        T, V, k = case["T"], case["V"], case["top"]
        # a model's logits: a broad bulk and, in every row, a few likely tokens
        s.logits = _rand(gen, T, V, sd=2.0)
        likely = (torch.randint(0, V, (T, 1), generator=gen, device="cuda")
                  + torch.arange(24, device="cuda") * (V // 24)) % V
        s.logits.scatter_add_(1, likely, _rand(gen, T, 24, sd=3.0) + 8.0)
        pick = torch.rand(T, generator=gen, device="cuda") < 0.7
        s.tokens = torch.where(pick, likely[:, 0], torch.randint(0, V, (T,), generator=gen, device="cuda"))
    else:
        hk, hq, d = case["kv_heads"], case["heads"], case["dim"]
        if op == "append":
            T, page = case["T"], case["page"]
            s.freqs = torch.tensor([THETA ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device="cuda")
            s.q, s.kn, s.vn = _rand(gen, T, hq, d), _rand(gen, T, hk, d, sd=2.0), _rand(gen, T, hk, d)
            _cache(s, case, gen, [T + 2 * page])
            slot = torch.randperm((T + 2 * page) // page * page, generator=gen, device="cuda")[:T]
            s.slots = s.table.view(-1).long()[slot // page] * page + slot % page
            s.positions = torch.randint(0, case["far"], (T,), generator=gen, device="cuda")
            s.q_out = torch.empty_like(s.q)
        else:
            lens = lengths(case)
            _cache(s, case, gen, lens)
            B, cap = len(lens), s.table.shape[1] * case["page"]
            # what earlier steps have accumulated: a few tokens hold most of it
            s.sums = torch.exp(_rand(gen, B, hk, cap, sd=1.5))
            if op == "attn":
                s.q = _rand(gen, B, hq, d, sd=1.5)
                s.out = torch.empty_like(s.q)
                s.weights = s.sums.clone() if case["weights"] else None
            else:
                s.weights = s.sums.clone()
                s.new_lens = torch.empty_like(s.lens)
    if own:
        from infer_amd import ops
        if op == "logprobs":
            s.answer = ops.alloc_logprobs(case["T"], case["top"])
        else:
            s.cache = ops.KvCache(s.k, s.v)
    return s


def run(s):
    op = s.case["op"]
    if op == "append":
        q = _append_own(s) if own else _append(s)
        return {"q": q, "k": s.k, "v": s.v}
    if op == "attn":
        out = _attn_own(s) if own else _attn(s)
        return {"out": out, "weights": s.weights} if s.weights is not None else {"out": out}
    if op == "evict":
        # the attention steps since the last eviction have filled the sums
        s.weights.copy_(s.sums)
        lens = _evict_own(s) if own else _evict(s)
        return {"lens": lens, "weights": s.weights, "k": s.k, "v": s.v}
    lp, ent, ids, top = _logprobs_own(s) if own else _logprobs(s)
    return {"logprob": lp, "entropy": ent, "ids": ids, "top": top} if s.case["top"] else {"logprob": lp, "entropy": ent}


# ------------------------------------------------------- the library's calls
def _append_own(s):
    from infer_amd import ops
    return ops.kv_append(s.q, s.kn, s.vn, s.positions, s.slots, s.freqs, s.cache, q_out=s.q_out)


def _attn_own(s):
    from infer_amd import ops
    return ops.attn_decode(s.q, s.cache, s.table, s.lens, out=s.out, weights=s.weights)


def _evict_own(s):
    from infer_amd import ops
    return ops.kv_evict(s.cache, s.table, s.lens, s.weights, s.case["budget"], s.case["recent"], new_lens=s.new_lens)


def _logprobs_own(s):
    from infer_amd import ops
    r = ops.logprobs(s.logits, s.tokens, top=s.case["top"], out=s.answer)
    return r.logprob, r.entropy, r.top_ids, r.top_logprobs


# ------------------------------------------------------------- plain forms
def _rotate(x, cos, sin):
    """Pairs (i, i + d/2) of every head turned by the row's angles."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    ang = s.positions[:, None].double() * s.freqs  # far positions lose their angle in 32 bits
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    page = s.case["page"]
    s.k[s.slots // page, s.slots % page] = _rotate(s.kn, cos, sin).to(s.k.dtype)
    s.v[s.slots // page, s.slots % page] = s.vn.to(s.v.dtype)
    return _rotate(s.q, cos, sin)


def _attn(s):
    c = s.case
    B, hk, g, d = s.q.shape[0], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    pages = s.table.long().clamp(min=0)
    cap = pages.shape[1] * c["page"]
    live = torch.arange(cap, device="cuda")[None, :] < s.lens[:, None]  # [B, cap]
    K = s.k[pages].view(B, cap, hk, d).transpose(1, 2).float()
    V = s.v[pages].view(B, cap, hk, d).transpose(1, 2).float()
    V = torch.where(live[:, None, :, None], V, torch.zeros((), device="cuda")).contiguous()
    sc = torch.matmul(s.q.view(B, hk, g, d), K.transpose(2, 3).contiguous()) * d ** -0.5
    sc = torch.where(live[:, None, None], sc, torch.full((), -math.inf, device="cuda"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    if s.weights is not None:
        s.weights += p.sum(2)
    return torch.matmul(p, V).view(B, c["heads"], d)


def _evict(s):
    """Stable order: the kept tokens below the cut stay, holes among them are
    filled in ascending order by the kept ones above it, then the newest
    tokens follow in their order."""
    c = s.case
    n, budget, recent, page = c["len"], c["budget"], c["recent"], c["page"]
    B, hk = s.table.shape[0], c["kv_heads"]
    s.new_lens.copy_(s.lens.clamp(max=budget))
    if n <= budget:
        return s.new_lens
    old, cut = n - recent, budget - recent  # older tokens now, and how many of them stay
    w = s.weights[:, :, :n]
    rank = torch.sort(w[:, :, :old], dim=-1, descending=True, stable=True).indices
    keep = torch.zeros(B, hk, old, dtype=torch.bool, device="cuda").scatter_(2, rank[:, :, :cut], True)
    at = torch.arange(old, device="cuda").expand(B, hk, old)
    # kept ones first, those below the cut before those above it; the i-th hole takes the i-th kept one above
    hole = (~keep & (at < cut)).long()
    high = (keep & (at >= cut)).long()
    nth_high = torch.sort(torch.where(high > 0, at, at + n), dim=-1).values
    src = torch.where(hole[:, :, :cut] > 0, nth_high.gather(2, (hole.cumsum(2) - 1).clamp(min=0)[:, :, :cut]),
                      at[:, :, :cut])
    src = torch.cat([src, torch.arange(old, n, device="cuda").expand(B, hk, recent)], 2)  # [B, hk, budget]
    b, h = torch.arange(B, device="cuda")[:, None, None], torch.arange(hk, device="cuda")[None, :, None]
    dst = torch.arange(budget, device="cuda").expand(B, hk, budget)
    tb = s.table.long()
    from_page, to_page = tb[b, src // page], tb[b, dst // page]
    s.k[to_page, dst % page, h] = s.k[from_page, src % page, h]
    s.v[to_page, dst % page, h] = s.v[from_page, src % page, h]
    s.weights[:, :, :budget] = w.gather(2, src)
    s.weights[:, :, budget:n] = 0
    return s.new_lens


def _logprobs(s):
    x = s.logits
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + z.log()
    lp = (x.gather(1, s.tokens[:, None]) - lse)[:, 0]
    ent = (z.log() - (e * (x - m)).sum(1, keepdim=True) / z)[:, 0]
    if not s.case["top"]:
        return lp, ent, None, None
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : s.case["top"]]
    return lp, ent, ids, x.gather(1, ids) - lse


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        lp = torch.log_softmax(s.logits.double(), 1)
        r = {"logprob": lp[torch.arange(case["T"], device="cuda"), s.tokens], "entropy": -(lp.exp() * lp).sum(1)}
        if case["top"]:
            # the ids are whole numbers: held to the plain form's
            r.update(ids=None, top=lp.topk(case["top"], 1).values)
        return r
    if op == "append":
        d = case["dim"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s.positions[:, None, None] * s.freqs)

        def turned(x):
            x = x.double()
            z = torch.complex(x[..., : d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        k, v = s.k.double(), s.v.double()
        k.view(-1, case["kv_heads"], d)[s.slots] = turned(s.kn)
        v.view(-1, case["kv_heads"], d)[s.slots] = s.vn.double()
        return {"q": turned(s.q), "k": k, "v": v}
    if op == "evict":
        return None  # values only move
    g, d = case["heads"] // case["kv_heads"], case["dim"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    sums = s.sums.double()
    for b, n in enumerate(lengths(case)):
        t = torch.arange(n, device="cuda")
        page = s.table[b].long()[t // case["page"]]
        for h in range(case["kv_heads"]):
            K, V = s.k[page, t % case["page"], h].double(), s.v[page, t % case["page"], h].double()
            p = torch.softmax(s.q[b, h * g:(h + 1) * g].double() @ K.t() / math.sqrt(d), 1)
            out[b, h * g:(h + 1) * g] = p @ V
            sums[b, h, :n] += p.sum(0)
    return {"out": out, "weights": sums} if case["weights"] else {"out": out}


def work(case):
    op = case["op"]
    if op == "logprobs":
        T, V, k = case["T"], case["V"], case["top"]
        return dict(bytes=4 * T * V + T * (8 + 8 + 12 * k), flops=5 * T * V)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "append":
        T = case["T"]
        return dict(bytes=T * (4 * d * (2 * hq + 2 * hk) + 2 * 2 * d * hk + 16), flops=3 * T * d * (hq + hk))
    B = case["B"]
    if op == "attn":
        total = sum(lengths(case))
        b = total * hk * d * 4 + 8 * B * hq * d + 4 * (total // case["page"] + B)
        if case["weights"]:
            b += 8 * total * hk
        return dict(bytes=b, flops=4 * total * hq * d)
    n, budget, recent = case["len"], case["budget"], case["recent"]
    # the newest ones, and the holes that random weights leave below the cut
    moved = recent + (budget - recent) * (n - budget) / (n - recent)
    return dict(bytes=B * hk * (4 * n + moved * (2 * 2 * 2 * d + 4) + 4 * (n - budget)), flops=B * hk * 4 * n)
