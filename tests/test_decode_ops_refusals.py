"""What the decode-step operators refuse, on the host and before anything
touches a device (no GPU needed): error codes of the C ABI, and what the
Python mirror checks of its tensors."""
import ctypes

import pytest
import torch

from infer_amd import ops

KIND, SHAPE, NULL, LARGE, ALIAS = -1, -2, -3, -4, -7
P = 1 << 20  # stands for a device pointer that nothing reads


def kv(**c):
    f = dict(type=0, kv_heads=2, head_dim=64, page_size=16, pages=9, page_stride=2048, slot_stride=128, head_stride=64,
             k=P, v=2 * P)
    f.update(c)
    return ctypes.byref(ops.IqKv(**f))


BAD_KV = [(dict(type=2), KIND), (dict(type=-1), KIND), (dict(kv_heads=0), SHAPE), (dict(kv_heads=1025), SHAPE),
          (dict(head_dim=0), SHAPE), (dict(head_dim=68), SHAPE), (dict(head_dim=264), SHAPE), (dict(page_size=0), SHAPE),
          (dict(pages=0), SHAPE), (dict(pages=2 ** 31), SHAPE), (dict(page_stride=2044), SHAPE),
          (dict(slot_stride=-128), SHAPE), (dict(head_stride=0), SHAPE), (dict(page_stride=2 ** 31), SHAPE),
          (dict(k=P + 8), SHAPE), (dict(v=P + 2), SHAPE), (dict(k=None), NULL), (dict(v=None), NULL)]


@pytest.mark.parametrize("change,code", BAD_KV)
def test_bad_caches(change, code):
    L = ops.lib()
    c = kv(**change)
    assert L.iq_kv_append(P, P, P, P, P, 4, 4, P, 64, c, P, None) == code
    assert L.iq_attn_decode(P, c, P, 8, 8, P, 4, 4, 0.1, 2 * P, None, 0, None) == code
    assert L.iq_kv_evict(c, P, 8, 8, P, 4, 64, 16, P, 128, 2 * P, None) == code


def test_append():
    L = ops.lib()
    big = 64 * P

    def call(q=P, k=2 * P, v=3 * P, pos=P, slots=P, T=4, hq=4, freqs=P, rot=64, c=None, out=big):
        return L.iq_kv_append(q, k, v, pos, slots, T, hq, freqs, rot, c or kv(), out, None)
    assert L.iq_kv_append(P, P, P, P, P, 4, 4, P, 64, None, big, None) == NULL
    for bad in (dict(T=0), dict(T=-1), dict(hq=-1), dict(hq=16385), dict(rot=-8), dict(rot=4), dict(rot=72)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(slots=None), dict(freqs=None),
                dict(out=None)):
        assert call(**bad) == NULL, bad
    assert call(T=2 ** 31) == LARGE
    assert call(out=P + 256) == ALIAS           # partly q
    assert call(out=2 * P - 16) == ALIAS        # reaches into k
    assert call(out=3 * P) == ALIAS             # v


def test_attention():
    L = ops.lib()

    def call(q=P, c=None, table=P, ld=8, pages=8, lens=P, B=4, hq=4, scale=0.1, out=2 * P, w=None, wld=0):
        return L.iq_attn_decode(q, c or kv(), table, ld, pages, lens, B, hq, scale, out, w, wld, None)
    for bad in (dict(B=0), dict(B=1025), dict(hq=0), dict(hq=3), dict(hq=-2), dict(hq=16386), dict(pages=0), dict(ld=7),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(w=P, wld=127)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(q=None), dict(table=None), dict(lens=None), dict(out=None)):
        assert call(**bad) == NULL, bad
    assert L.iq_attn_decode(P, None, P, 8, 8, P, 4, 4, 0.1, 2 * P, None, 0, None) == NULL
    assert call(out=P + 4) == ALIAS and call(out=P) == ALIAS
    assert call(pages=2 ** 27, ld=2 ** 27) == LARGE  # 2^31 tokens a sequence


def test_evict():
    L = ops.lib()

    def call(c=None, table=P, ld=8, pages=8, lens=P, B=4, budget=64, recent=16, w=P, wld=128, new=2 * P):
        return L.iq_kv_evict(c or kv(), table, ld, pages, lens, B, budget, recent, w, wld, new, None)
    for bad in (dict(B=0), dict(B=1025), dict(budget=0), dict(budget=-5), dict(recent=-1), dict(recent=65), dict(pages=0),
                dict(ld=7), dict(wld=127)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(table=None), dict(lens=None), dict(w=None), dict(new=None)):
        assert call(**bad) == NULL, bad
    assert call(new=P) == ALIAS and call(new=P + 12) == ALIAS
    assert call(pages=2 ** 27, ld=2 ** 27, wld=2 ** 31) == LARGE


def test_logprobs():
    L = ops.lib()

    def call(x=P, ld=100, T=3, V=100, tok=P, top=5, lp=P, ent=P, ids=P, tlp=P):
        return L.iq_logprobs(x, ld, T, V, tok, top, lp, ent, ids, tlp, None)
    for bad in (dict(T=0), dict(V=0), dict(ld=99), dict(top=-1), dict(top=65), dict(V=4)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(x=None), dict(tok=None), dict(lp=None), dict(ids=None), dict(tlp=None),
                dict(tok=None, lp=None, ent=None, top=0)):
        assert call(**bad) == NULL, bad
    assert call(V=2 ** 31 - 1, ld=2 ** 31) == LARGE
    assert call(T=2 ** 31) == LARGE


def cache(device="cpu", **kw):
    return ops.alloc_kv(5, 16, 2, 64, device=device, **kw)


def test_python_checks():
    i32, i64 = torch.int32, torch.int64
    c = cache()
    q, k, pos = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=i64)
    fr = ops.rope_freqs(64, 1e6, device="cpu")
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.kv_append(q, k, k, pos, pos, fr, c)
    for bad in (dict(q=q.half()), dict(k=k.double()), dict(pos=pos.int()), dict(freqs=fr.float())):
        a = dict(q=q, k=k, v=k, pos=pos, slots=pos, freqs=fr)
        a.update(bad)
        with pytest.raises(TypeError):
            ops.kv_append(*a.values(), c)
    for bad in (dict(q=torch.zeros(4, 64, 3).permute(2, 0, 1)), dict(k=k[:2]), dict(v=torch.zeros(3, 2, 65)),
                dict(pos=pos[:2]), dict(q=torch.zeros(3, 4, 65))):
        a = dict(q=q, k=k, v=k, pos=pos, slots=pos, freqs=fr)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.kv_append(*a.values(), c)
    with pytest.raises(ValueError, match="positions"):
        ops.kv_append(q, k, k, None, pos, fr, c)
    table, lens, w = torch.zeros(3, 5, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(3, 2, 80)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.attn_decode(q, c, table, lens, weights=w)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.kv_evict(c, table, lens, w, 20, 4)
    for t, n, s in ((table.long(), lens, w), (table[0], lens, w), (table.t().contiguous().t(), lens, w),
                    (table, lens[:2], w), (table, lens, w.double()), (table, lens, w[:, :1]), (table, lens, w[:2]),
                    (table, lens, w.transpose(0, 1).contiguous().transpose(0, 1)), (table, lens, w[:, :, :40])):
        with pytest.raises(ValueError):
            ops.attn_decode(q, c, t, n, weights=s)
        with pytest.raises(ValueError):
            ops.kv_evict(c, t, n, s, 20, 4)
    with pytest.raises(TypeError):
        ops.attn_decode(q, c, table, lens.long())
    x = torch.zeros(4, 50)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.logprobs(x, out=ops.alloc_logprobs(4, device="cpu"))
    small = ops.alloc_logprobs(4, 3, device="cpu")
    for kw in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=torch.zeros(50, 4).t()), dict(tokens=pos),
               dict(top=2, out=small), dict(top=3, out=ops.alloc_logprobs(4, device="cpu")),
               dict(tokens=torch.zeros(4, dtype=i64), out=small._replace(logprob=None))):
        a = dict(logits=x, out=small)
        a.update(kw)
        with pytest.raises(ValueError):
            ops.logprobs(**a)
    with pytest.raises(TypeError):
        ops.logprobs(x, torch.zeros(4, dtype=i32), out=small)


def test_python_caches():
    k = torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)
    for a, b in ((k, k[:4]), (k, k.half()), (k[0], k[0]), (k, k.transpose(1, 2).contiguous().transpose(1, 2)),
                 (k.transpose(2, 3), k.transpose(2, 3))):
        with pytest.raises(ValueError):
            ops.KvCache(a, b)
    with pytest.raises(TypeError):
        ops.KvCache(k.float(), k.float())
    c = ops.KvCache(k, k)
    assert (c._c.page_stride, c._c.slot_stride, c._c.head_stride) == (2048, 128, 64)
    one = ops.KvCache(k[:1, :1, :1], k[:1, :1, :1])  # strides over one page, slot or head do not count
    assert (one._c.page_stride, one._c.slot_stride, one._c.head_stride) == (0, 0, 0)
