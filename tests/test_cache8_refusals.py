"""What the operators over caches of any type refuse, on the host and before
anything touches a device (no GPU needed)."""
import ctypes

import pytest
import torch

from infer_amd import ops

KIND, SHAPE, NULL, LARGE, ALIAS = -1, -2, -3, -4, -7
P = 1 << 20  # stands for a device pointer that nothing reads
BIG = 64 * P


def kv(**c):
    f = dict(type=2, kv_heads=2, head_dim=64, page_size=16, pages=9, page_stride=2048, slot_stride=128, head_stride=64,
             k=P, v=2 * P)
    f.update(c)
    return ctypes.byref(ops.IqKv(**f))


def scales(**c):
    f = dict(block=8, page_stride=4, block_stride=2, head_stride=1, k=3 * P, v=4 * P)
    f.update(c)
    return ctypes.byref(ops.IqKvScales(**f))


def extend(q=P, k=2 * P, v=3 * P, T=4, hq=4, qn=P, kn=P, eps=1e-6, pos=P, freqs=P, rot=64, c=None, s=None, table=P, ld=8,
           pages=8, lens=P, starts=P, B=4, out=BIG):
    return ops.lib().iq_kv_extend(q, k, v, T, hq, qn, kn, eps, pos, freqs, rot, c or kv(), s or scales(), table, ld, pages,
                                  lens, starts, B, out, None)


def read(c=None, s=None, table=P, ld=8, pages=8, first=P, starts=P, B=4, T=7, t=0, k=BIG, v=2 * BIG):
    return ops.lib().iq_kv_read(c or kv(), s or scales(), table, ld, pages, first, starts, B, T, t, k, v, None)


def attn(q=P, c=None, s=None, table=P, ld=8, pages=8, lens=P, B=4, hq=4, scale=0.1, window=0, sinks=0, out=2 * P):
    return ops.lib().iq_attn_decode_window(q, c or kv(), s or scales(), table, ld, pages, lens, B, hq, scale, window, sinks,
                                           out, None)


BAD_KV = [(dict(type=4), KIND), (dict(type=-1), KIND), (dict(kv_heads=0), SHAPE), (dict(head_dim=0), SHAPE),
          (dict(head_dim=72), SHAPE), (dict(head_dim=272), SHAPE), (dict(page_size=0), SHAPE), (dict(pages=0), SHAPE),
          (dict(pages=2 ** 31), SHAPE), (dict(page_stride=2056), SHAPE), (dict(slot_stride=-128), SHAPE),
          (dict(head_stride=8), SHAPE), (dict(k=P + 8), SHAPE), (dict(v=P + 1), SHAPE), (dict(k=None), NULL),
          (dict(page_size=12), SHAPE)]  # (blocks of 8 do not divide it)
BAD_SCALES = [(dict(block=0), SHAPE), (dict(block=-8), SHAPE), (dict(block=3), SHAPE), (dict(block=32), SHAPE),
              (dict(page_stride=0), SHAPE), (dict(block_stride=0), SHAPE), (dict(head_stride=-1), SHAPE),
              (dict(page_stride=2 ** 31), SHAPE), (dict(k=P + 2), SHAPE), (dict(k=None), NULL), (dict(v=None), NULL)]


@pytest.mark.parametrize("change,code", BAD_KV)
def test_bad_caches(change, code):
    c = kv(**change)
    assert extend(c=c) == code and read(c=c) == code and attn(c=c) == code


@pytest.mark.parametrize("change,code", BAD_SCALES)
def test_bad_scales(change, code):
    s = scales(**change)
    assert extend(s=s) == code and read(s=s) == code and attn(s=s) == code


def test_missing_scales_and_caches():
    L = ops.lib()
    assert L.iq_attn_decode_window(P, kv(), None, P, 8, 8, P, 4, 4, 0.1, 0, 0, 2 * P, None) == NULL
    assert L.iq_attn_decode_window(P, None, scales(), P, 8, 8, P, 4, 4, 0.1, 0, 0, 2 * P, None) == NULL
    assert L.iq_kv_read(kv(), None, P, 8, 8, P, P, 4, 7, 0, BIG, 2 * BIG, None) == NULL
    assert L.iq_kv_extend(P, P, P, 4, 4, P, P, 0.0, P, P, 64, kv(), None, P, 8, 8, P, P, 4, BIG, None) == NULL


@pytest.mark.parametrize("t", [2, 3])
def test_codes_where_16_bits_are_wanted(t):
    L, c = ops.lib(), kv(type=t)
    assert L.iq_kv_append(P, P, P, P, P, 4, 4, P, 64, c, P, None) == KIND
    assert L.iq_attn_decode(P, c, P, 8, 8, P, 4, 4, 0.1, 2 * P, None, 0, None) == KIND
    assert L.iq_kv_evict(c, P, 8, 8, P, 4, 64, 16, P, 128, 2 * P, None) == KIND


def test_extend():
    for bad in (dict(T=0), dict(T=-1), dict(hq=-1), dict(hq=16385), dict(rot=-8), dict(rot=4), dict(rot=72), dict(B=0),
                dict(B=1025), dict(pages=0), dict(ld=7), dict(starts=None, T=5), dict(eps=-1e-6), dict(eps=float("nan")),
                dict(eps=float("inf"))):
        assert extend(**bad) == SHAPE, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(freqs=None), dict(out=None), dict(table=None),
                dict(lens=None)):
        assert extend(**bad) == NULL, bad
    assert extend(T=2 ** 31) == LARGE and extend(pages=2 ** 27, ld=2 ** 27) == LARGE
    assert extend(out=P + 256) == ALIAS and extend(out=2 * P - 16) == ALIAS and extend(out=3 * P) == ALIAS


def test_read():
    for bad in (dict(T=0), dict(T=-4), dict(B=0), dict(B=1025), dict(pages=0), dict(ld=7)):
        assert read(**bad) == SHAPE, bad
    for bad in (dict(table=None), dict(starts=None), dict(k=None, v=None)):
        assert read(**bad) == NULL, bad
    assert read(t=3) == KIND and read(t=-1) == KIND
    assert read(T=2 ** 31) == LARGE
    assert read(v=BIG + 64) == ALIAS and read(v=BIG) == ALIAS


def test_attention():
    for bad in (dict(B=0), dict(B=1025), dict(hq=0), dict(hq=3), dict(hq=-2), dict(hq=16386), dict(pages=0), dict(ld=7),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(window=-1), dict(sinks=-1),
                dict(window=5, sinks=-2 ** 62)):
        assert attn(**bad) == SHAPE, bad
    for bad in (dict(q=None), dict(table=None), dict(lens=None), dict(out=None)):
        assert attn(**bad) == NULL, bad
    assert attn(out=P + 4) == ALIAS and attn(out=P) == ALIAS
    assert attn(pages=2 ** 27, ld=2 ** 27) == LARGE


def test_python_caches():
    k = torch.zeros(5, 16, 2, 64, dtype=torch.int8)
    s = torch.zeros(5, 2, 2)
    c = ops.KvCache(k, k, s, s)
    assert c.block == 8 and (c._s.page_stride, c._s.block_stride, c._s.head_stride) == (4, 2, 1)
    for a in ((k, k), (k, k, s, None), (k, k, s[:4], s[:4]), (k, k, s[:, :, :1], s[:, :, :1]), (k, k, s, s[:, :1]),
              (k, k, torch.zeros(5, 3, 2), torch.zeros(5, 3, 2)), (k, k, s[0], s[0]), (k, k, s, s.transpose(0, 1).contiguous().transpose(0, 1)),
              (k.bfloat16(), k.bfloat16(), s, s), (k, k.view(torch.float8_e4m3fn), s, s)):
        with pytest.raises(ValueError):
            ops.KvCache(*a)
    with pytest.raises(TypeError):
        ops.KvCache(k, k, s.double(), s.double())
    with pytest.raises(TypeError):
        ops.KvCache(k.view(torch.uint8), k.view(torch.uint8), s, s)
    assert ops.alloc_kv(3, 16, 2, 64, torch.float8_e4m3fn, "cpu").block == 16
    assert ops.alloc_kv(3, 16, 2, 64, torch.int8, "cpu", block=4).k_scales.shape == (3, 4, 2)
    for bad in (dict(dtype=torch.int8, block=5), dict(dtype=torch.int8, block=0), dict(block=16)):
        with pytest.raises(ValueError):
            ops.alloc_kv(3, 16, 2, 64, device="cpu", **bad)


def test_python_checks():
    i32, i64 = torch.int32, torch.int64
    c = ops.alloc_kv(5, 16, 2, 64, torch.int8, "cpu", block=8)
    q, k, pos = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=i64)
    fr, norm = ops.rope_freqs(64, 1e6, device="cpu"), torch.ones(64, dtype=torch.bfloat16)
    table, lens, starts = torch.zeros(3, 5, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32)

    def ext(**kw):
        a = dict(q=q, k=k, v=k, positions=pos, freqs=fr, cache=c, table=table, lens=lens)
        a.update(kw)
        return ops.kv_extend(**a)
    with pytest.raises(ValueError, match="current CUDA device"):
        ext()
    for bad in (dict(q=q.half()), dict(k=k.double()), dict(positions=pos.int()), dict(freqs=fr.float()), dict(lens=lens.long()),
                dict(starts=starts.long()), dict(q_norm=norm.float()), dict(k_norm=norm.half())):
        with pytest.raises(TypeError):
            ext(**bad)
    for bad in (dict(v=k[:2]), dict(k=k[:2], v=k[:2]), dict(positions=pos[:2]), dict(positions=None), dict(table=table[0]),
                dict(lens=lens[:2]), dict(starts=starts[:3]), dict(q_norm=norm[:32]), dict(q=torch.zeros(3, 4, 65)),
                dict(q_out=torch.zeros(3, 3, 64))):
        with pytest.raises(ValueError):
            ext(**bad)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.kv_read(c, table, starts, T=3)
    with pytest.raises(TypeError):
        ops.kv_read(c, table, starts, out=(k.double(), k.double()))
    for bad in (dict(), dict(T=3, first=lens[:2]), dict(out=(None, None)), dict(out=(k, k[:2])), dict(T=4, out=(k, k))):
        with pytest.raises(ValueError):
            ops.kv_read(c, table, starts, **bad)
    with pytest.raises(TypeError):
        ops.kv_read(c, table, starts, out=(k, k.bfloat16()))
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.attn_decode(q, c, table, lens, window=3, sinks=1)
    for bad in (dict(window=-1), dict(sinks=-1), dict(weights=torch.zeros(3, 2, 80))):
        with pytest.raises(ValueError):
            ops.attn_decode(q, c, table, lens, **bad)
    plain = ops.alloc_kv(5, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="window"):
        ops.attn_decode(q, plain, table, lens, weights=torch.zeros(3, 2, 80), window=4)
