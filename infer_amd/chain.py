"""Stage programs of dependent 1-row GEMVs (include/iq.h, iq_chain_*), and
the decode step built from them.

DecodeStep is the quantised part of the reference's decode step,
GpuBatch::Impl::launch_sequence (kernels/batch_gpu.cu:186-215), for B
sequences (B = 1..32, GpuBatch::kMaxRows, kernels/batch_gpu.h:80) of one
token each at position 0: the quantised embedding gather of the B tokens
(launch_embedding_q), then per layer, for each of the B rows

    q|k|v  = rmsnorm(h, input_ln) . W_qkv^T + b_qkv          (one stage)
    h'     = h + attn . W_o^T                                  (one stage)
    act    = silu(n . W_gate^T) * (n . W_up^T),
             n = rmsnorm(h', post_attn_ln)                    (one stage)
    h''    = h' + act . W_down^T                               (one stage)

and logits = rmsnorm(h, final_norm) . W_head^T.  At position 0 the
attention over the single cached key has softmax weight 1, so attn is the
value row of each query head's key/value head (IQ_IN_GQA); RoPE changes q
and k only.  Every intermediate vector has its own buffer (static
single-assignment), so all of them can be inspected after a step.
"""
import ctypes

import torch

from . import ops

IN_PLAIN, IN_RMSNORM, IN_GQA = 0, 1, 2
OUT_STORE, OUT_RESIDUAL, OUT_SWIGLU = 0, 1, 2


IqStage = ops.IqStage


def _lib():
    return ops.lib()


def _p(t):
    return None if t is None else t.data_ptr()


class Stage:
    """One stage: y_i = out_op(dequant(Ws[i]) . in_op(x) + biases[i])."""

    def __init__(self, Ws, x, ys, in_op=IN_PLAIN, out_op=OUT_STORE, biases=None, norm=None, eps=0.0,
                 residual=None, gqa=(0, 0), rows=1):
        self.Ws, self.x, self.ys = list(Ws), x, list(ys)
        self.rows = rows
        self.in_op, self.out_op = in_op, out_op
        self.biases = list(biases) if biases is not None else [None] * len(self.Ws)
        self.norm, self.eps, self.residual, self.gqa = norm, eps, residual, gqa

    def to_c(self):
        s = IqStage()
        s.in_op, s.out_op, s.n = self.in_op, self.out_op, len(self.Ws)
        s.gqa_head_dim, s.gqa_group = self.gqa
        s.eps = self.eps
        s.rows = self.rows
        s.x, s.norm, s.residual = _p(self.x), _p(self.norm), _p(self.residual)
        for i, W in enumerate(self.Ws):
            s.W[i] = W._c
            s.bias[i] = _p(self.biases[i])
        for i, y in enumerate(self.ys):
            s.y[i] = _p(y)
        return s


class Chain:
    """A validated program on the current device (iq_chain_create)."""

    def __init__(self, stages):
        self.stages = list(stages)  # keeps the tensors alive
        arr = (IqStage * len(self.stages))(*[s.to_c() for s in self.stages])
        h = ctypes.c_void_p()
        rc = _lib().iq_chain_create(arr, len(self.stages), ctypes.byref(h))
        ops._check(rc, "iq_chain_create")
        self._h = h

    def run(self, stream=None):
        ops._check(_lib().iq_chain_run(self._h, ops._stream(stream)), "iq_chain_run")

    def close(self):
        if getattr(self, "_h", None):
            _lib().iq_chain_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Arena:
    """fp32 vectors carved from one device tensor, each starting on its own
    1 KiB boundary (no two vectors share a cache line)."""

    def __init__(self, sizes, device="cuda"):
        pad = [(n + 255) // 256 * 256 for n in sizes]
        self.buf = torch.zeros(sum(pad) + 256, dtype=torch.float32, device=device)
        base = (-(self.buf.data_ptr() // 4)) % 256
        self.views, off = [], base
        for n, p in zip(sizes, pad):
            self.views.append(self.buf[off:off + n])
            off += p


class DecodeStep:
    """The quantised decode step of one token at position 0 (module
    docstring).  `model` has: cfg dict (hidden, inter, heads, kv_heads,
    head_dim, vocab, layers, eps), embed / head (QuantView), final_norm
    (bf16 int16 tensor), layers: list of dicts with QuantViews q, k, v, o,
    gate, up, down, bf16 tensors input_ln, post_ln and optional q_b, k_b, v_b.
    rows: B sequences; every vector below is [B][n] row-major."""

    def __init__(self, model, device="cuda", rows=1):
        c = model["cfg"]
        H, I, V = c["hidden"], c["inter"], c["vocab"]
        nh, nkv, hd, L = c["heads"], c["kv_heads"], c["head_dim"], c["layers"]
        qo, kvo = nh * hd, nkv * hd
        B = self.rows = int(rows)
        sizes = [H]
        for _ in range(L):
            sizes += [qo, kvo, kvo, H, I, H]
        sizes += [V]
        self.arena = Arena([B * n for n in sizes], device)
        vs = iter(self.arena.views)
        self.h0 = next(vs)
        self.ids = torch.zeros(B, dtype=torch.int64, device=device)
        self.model = model
        self.per_layer = []
        stages = []
        h = self.h0
        for li in range(L):
            Lw = model["layers"][li]
            q, k, v, h1, act, h2 = (next(vs) for _ in range(6))
            stages.append(Stage([Lw["q"], Lw["k"], Lw["v"]], h, [q, k, v], IN_RMSNORM, OUT_STORE,
                                biases=[Lw.get("q_b"), Lw.get("k_b"), Lw.get("v_b")], norm=Lw["input_ln"],
                                eps=c["eps"], rows=B))
            stages.append(Stage([Lw["o"]], v, [h1], IN_GQA, OUT_RESIDUAL, residual=h, gqa=(hd, nh // nkv), rows=B))
            stages.append(Stage([Lw["gate"], Lw["up"]], h1, [act], IN_RMSNORM, OUT_SWIGLU, norm=Lw["post_ln"],
                                eps=c["eps"], rows=B))
            stages.append(Stage([Lw["down"]], act, [h2], IN_PLAIN, OUT_RESIDUAL, residual=h1, rows=B))
            self.per_layer.append(dict(h=h, q=q, k=k, v=v, h1=h1, act=act, h2=h2))
            h = h2
        self.logits = next(vs)
        stages.append(Stage([model["head"]], h, [self.logits], IN_RMSNORM, OUT_STORE, norm=model["final_norm"],
                            eps=c["eps"], rows=B))
        self.h_last = h
        self.chain = Chain(stages)

    def step(self, token_id=None, stream=None):
        """Embedding gather of the B token ids `token_id` (an int for every
        row, or a sequence of B ints; None: the ids already in self.ids),
        then the chain.  Asynchronous on the stream."""
        if token_id is not None:
            if isinstance(token_id, int):
                self.ids.fill_(int(token_id))
            else:
                self.ids.copy_(torch.tensor([int(t) for t in token_id], dtype=torch.int64))
        H = self.model["cfg"]["hidden"]
        ops.launch_embedding_q(self.model["embed"], self.ids, self.rows, H, self.h0, stream)
        self.chain.run(stream)

    def weight_bytes(self):
        n = self.rows * (self.model["embed"].nbytes() // self.model["embed"].rows)  # the gathered rows
        for Lw in self.model["layers"]:
            n += sum(Lw[k].nbytes() for k in ("q", "k", "v", "o", "gate", "up", "down"))
        return n + self.model["head"].nbytes()


def next_slots(lens, table, page_size, pages=2 ** 31, out=None):
    """The cache slot (int64, page * page_size + slot) behind each sequence's
    first lens[b] tokens, and whether there is one.  There is none where the
    table is full, the page id outside [0, pages) or the length below 0; the
    slot is then outside the pool.  (Few operations: a step makes them all, at
    about 2 us each in a graph.)"""
    at = lens.clamp(0, table.shape[1] * page_size - 1)  # (of any length: the index has to lie in the table)
    nth = (at // page_size).long()
    # page * page_size + at % page_size
    slot = torch.add(at, table.gather(1, nth[:, None])[:, 0] - nth, alpha=page_size, out=out)
    slot.masked_fill_(lens != at, -1)
    return slot, slot == slot.clamp(0, pages * page_size - 1)


class CachedDecodeStep:
    """One decode step of B sequences over paged key/value caches, one
    ops.KvCache a layer: every sequence's next token, at the position and
    cache length that `positions` and `lens` hold, through all layers to
    logits.  `model` as for DecodeStep, with cfg["theta"] (rotary base) and, in
    its layers, optional bf16 tensors q_norm, k_norm [head_dim]: norms of every
    head of q and k (with cfg["eps"]) ahead of the rotation.

    caches: of any type; an 8-bit one's blocks fill in the order of the steps.
    window > 0: attention sees the newest `window` tokens in the cache and its
    first `sinks` only (ops.attn_decode); pages without any of these may be given
    to other sequences.

    table: int32 [B, pages], the pages of every sequence (the same ids in all
    layers); enough of them have to be there before the step that fills them.
    weights: keep the attention weight every cached token has received, per
    layer [B, kv_heads, pages * page_size], for evict(); with 16-bit caches and
    no window.

    Device state, which the caller may set between steps: lens (int32 [B],
    tokens of each sequence), positions (int64 [B], of the next token; they
    part from lens after an eviction), and for a new sequence in a row its
    weights, to 0.  held (int32 [B]) is how many of the tokens lie in the cache:
    lens, less those that found no place (see step) since the caller or evict()
    last set lens.  step() without a list of ids issues only device work, so it
    can be captured into a graph (after ops.init on the capturing stream)."""

    def __init__(self, model, caches, table, weights=False, device="cuda", window=0, sinks=0):
        c = model["cfg"]
        H, I, V = c["hidden"], c["inter"], c["vocab"]
        nh, nkv, hd, L = c["heads"], c["kv_heads"], c["head_dim"], c["layers"]
        if window < 0 or sinks < 0:
            raise ValueError("CachedDecodeStep: window and sinks must not be negative")
        if weights and (window or any(k.block for k in caches)):
            raise ValueError("CachedDecodeStep: weights are kept over 16-bit caches and without a window")
        if len(caches) != L or any((k.kv_heads, k.head_dim) != (nkv, hd) for k in caches):
            raise ValueError("CachedDecodeStep: one cache a layer, of the model's key/value heads and head size")
        if len({k.page_size for k in caches}) != 1:
            raise ValueError("CachedDecodeStep: caches of one page size")
        B = self.rows = table.shape[0]
        self.model, self.caches, self.table = model, list(caches), table
        self.window, self.sinks = window, sinks
        # layers whose tokens are added by kv_extend: 8-bit caches, or norms
        self._norms = [(Lw.get("q_norm"), Lw.get("k_norm")) for Lw in model["layers"]]
        self._extends = [bool(k.block) or any(n is not None for n in w) for k, w in zip(caches, self._norms)]
        self.page = caches[0].page_size
        self.pages = min(k.pages for k in caches)
        self.capacity = table.shape[1] * self.page
        qo, kvo = nh * hd, nkv * hd
        sizes = [H] + [qo, kvo, kvo, qo, qo, H, I, H] * L + [V]
        self.arena = Arena([B * n for n in sizes], device)
        vs = iter(self.arena.views)
        self.h0 = next(vs)
        self.ids = torch.zeros(B, dtype=torch.int64, device=device)
        self.lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.held = torch.zeros(B, dtype=torch.int32, device=device)
        self._left = torch.zeros(B, dtype=torch.int32, device=device)  # lens as step() or evict() left it
        self._attend = torch.zeros(B, dtype=torch.int32, device=device)
        self._behind = torch.zeros(B, dtype=torch.int32, device=device)  # held before the step, -1 without a place
        self._none = torch.full((B,), -1, dtype=torch.int32, device=device)
        self.positions = torch.zeros(B, dtype=torch.int64, device=device)
        self.slots = torch.full((B,), -1, dtype=torch.int64, device=device)
        self.freqs = ops.rope_freqs(hd, c["theta"], device)
        self.weights = [torch.zeros(B, nkv, self.capacity, device=device) for _ in range(L)] if weights else None
        self._new_lens = torch.zeros(B, dtype=torch.int32, device=device)
        self.per_layer, self.chains = [], []
        h, stages = self.h0, []
        for li in range(L):
            Lw = model["layers"][li]
            q, k, v, q_rot, attn, h1, act, h2 = (next(vs) for _ in range(8))
            stages.append(Stage([Lw["q"], Lw["k"], Lw["v"]], h, [q, k, v], IN_RMSNORM, OUT_STORE,
                                biases=[Lw.get("q_b"), Lw.get("k_b"), Lw.get("v_b")], norm=Lw["input_ln"],
                                eps=c["eps"], rows=B))
            self.chains.append(Chain(stages))
            stages = [Stage([Lw["o"]], attn, [h1], IN_PLAIN, OUT_RESIDUAL, residual=h, rows=B),
                      Stage([Lw["gate"], Lw["up"]], h1, [act], IN_RMSNORM, OUT_SWIGLU, norm=Lw["post_ln"],
                            eps=c["eps"], rows=B),
                      Stage([Lw["down"]], act, [h2], IN_PLAIN, OUT_RESIDUAL, residual=h1, rows=B)]
            self.per_layer.append(dict(h=h, q=q, k=k, v=v, q_rot=q_rot, attn=attn, h1=h1, act=act, h2=h2))
            h = h2
        self.logits = next(vs).view(B, V)
        stages.append(Stage([model["head"]], h, [self.logits], IN_RMSNORM, OUT_STORE, norm=model["final_norm"],
                            eps=c["eps"], rows=B))
        self.chains.append(Chain(stages))
        self.h_last = h

    def _held_now(self):
        """held, or lens where the caller has set it since."""
        return torch.where(self.lens == self._left, self.held, self.lens)

    def step(self, token_id=None, stream=None):
        """The tokens `token_id` (an int for every row, or a sequence of B ints;
        None: the ids already in self.ids) are added to the caches, attend to
        them and leave their logits; lens, held and positions move on by one.
        A token finds no place where its sequence's pages are full or the next
        page id is none of the pool's: the sequence keeps its cache, its weights
        and its position, its logits are NaN, and of the three only lens counts
        the token.  With a page, or after evict(), the next step goes on behind
        the tokens in the cache.  A row whose length is below 0 is idle: NaN
        logits, and nothing of it changes."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.step(token_id)
        if token_id is not None:
            if isinstance(token_id, int):
                self.ids.fill_(int(token_id))
            else:
                self.ids.copy_(torch.tensor([int(t) for t in token_id], dtype=torch.int64))
        held = self._held_now()
        _, stored = next_slots(held, self.table, self.page, self.pages, self.slots)
        torch.add(held, stored, out=self.held)
        # (a row without its token attends to nothing: no length, so that its
        # output is NaN and its weights stay)
        torch.where(stored, self.held, self._none, out=self._attend)
        if any(self._extends):
            torch.where(stored, held, self._none, out=self._behind)
        self.lens.add_(self.lens >= 0)
        self._left.copy_(self.lens)
        ops.launch_embedding_q(self.model["embed"], self.ids, self.rows, self.model["cfg"]["hidden"], self.h0)
        self.chains[0].run()
        for li, b in enumerate(self.per_layer):
            if self._extends[li]:
                q_norm, k_norm = self._norms[li]
                ops.kv_extend(b["q"], b["k"], b["v"], self.positions, self.freqs, self.caches[li], self.table,
                              self._behind, q_norm=q_norm, k_norm=k_norm, eps=self.model["cfg"]["eps"],
                              q_out=b["q_rot"])
            else:
                ops.kv_append(b["q"], b["k"], b["v"], self.positions, self.slots, self.freqs, self.caches[li],
                              q_out=b["q_rot"])
            ops.attn_decode(b["q_rot"], self.caches[li], self.table, self._attend, out=b["attn"],
                            weights=self.weights[li] if self.weights else None, window=self.window, sinks=self.sinks)
            self.chains[li + 1].run()
        self.positions.add_(stored)

    def evict(self, budget, recent):
        """Every layer's caches cut to `budget` tokens a sequence by the weights
        they have received (ops.kv_evict); the pages past them are free, and
        lens and held are what is left.  `recent` must not be more than the
        last evict()'s `recent` and the tokens added since: the rows before
        those are no longer in the order of their age."""
        if not self.weights:
            raise ValueError("CachedDecodeStep.evict: made without weights")
        self.held.copy_(self._held_now())
        for cache, w in zip(self.caches, self.weights):
            ops.kv_evict(cache, self.table, self.held, w, budget, recent, new_lens=self._new_lens)
        for t in (self.held, self.lens, self._left):
            t.copy_(self._new_lens)

    def logprobs(self, tokens=None, top=0, out=None):
        """Log probabilities, entropy and top alternatives of the last step's
        logits (ops.logprobs)."""
        return ops.logprobs(self.logits, tokens, top, out)
