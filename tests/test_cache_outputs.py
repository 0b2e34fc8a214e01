"""Outputs that overlap the cache which a call reads or writes: refused on the
host, before anything touches a device (no GPU needed); and iq_overlap.h,
compiled with g++ and run here."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from infer_amd import ops

HERE = os.path.dirname(os.path.abspath(__file__))
ALIAS = -7
M = 1 << 20
K, V, KS, VS, Q, X, FAR = (i * 64 * M for i in range(1, 8))  # stand for device pointers that nothing reads
# 9 pages of 16 slots of 2 heads of 64: a page has 2048 elements, blocks of 8 slots 4 scales
BYTES = {0: 9 * 2048 * 2, 1: 9 * 2048 * 2, 2: 9 * 2048, 3: 9 * 2048}


def kv(t):
    return ctypes.byref(ops.IqKv(t, 2, 64, 16, 9, 2048, 128, 64, K, V))


def scales():
    return ctypes.byref(ops.IqKvScales(8, 4, 2, 1, KS, VS))


def places(t, bytes_):
    """The first and last places that overlap each part of the cache."""
    parts = [(K, BYTES[t]), (V, BYTES[t])]
    if t >= 2:
        parts += [(KS, 9 * 16), (VS, 9 * 16)]
    for at, n in parts:
        yield from (at, at + 16, at + n - 16, at - bytes_ + 16)


@pytest.mark.parametrize("t", [0, 1, 2, 3])
def test_outputs_in_the_cache(t):
    L = ops.lib()
    T, d = 3, 64
    for at in places(t, T * 4 * d * 4):
        assert L.iq_kv_extend(Q, X, X + M, T, 4, None, None, 0.0, None, None, 0, kv(t), scales(), FAR, 9, 9, FAR, FAR, 2, at,
                              None) == ALIAS, hex(at)
        assert L.iq_attn_decode_window(Q, kv(t), scales(), FAR, 9, 9, FAR, T, 4, 0.1, 0, 0, at, None) == ALIAS, hex(at)
        if t < 2:
            assert L.iq_kv_append(Q, X, X + M, None, FAR, T, 4, None, 0, kv(t), at, None) == ALIAS, hex(at)
            assert L.iq_attn_decode(Q, kv(t), FAR, 9, 9, FAR, T, 4, 0.1, at, None, 0, None) == ALIAS, hex(at)
    for out, size in ((0, 4), (1, 2), (2, 2)):
        for at in places(t, T * 2 * d * size):
            for k, v in ((at, None), (None, at), (at, Q), (Q, at)):
                assert L.iq_kv_read(kv(t), scales(), FAR, 9, 9, None, FAR, 2, T, out, k, v, None) == ALIAS, hex(at)


def test_overlaps():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "test_overlap")
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-o", exe,
                        os.path.join(HERE, "cpp", "test_overlap.cpp")], check=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 failures" in r.stdout and "runtime error" not in r.stderr, r.stderr
