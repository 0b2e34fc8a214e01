"""Python mirror of the reference's quantised-op interface, over libiq.so.

Mirrors, with the same names, argument meaning and order:
  QuantKind, QuantView            kernels/ops/ops.cuh:165-172
  launch_gemv_batched_q           kernels/ops/ops.cuh:173-174
  launch_gemm_tiled_q             kernels/ops/ops.cuh:175-176
  launch_embedding_q              kernels/ops/ops.cuh:177-178
  linear_b (quantised branch)     kernels/batch_gpu.cu:137-147
  quantize                        src/quant.h:61 (on the device here)
  upload_q                        kernels/model_gpu_internal.cuh:67-83

and, without counterparts in the reference's quantised path, the operators of
a decode step around it: KvCache, kv_append, attn_decode, kv_evict, logprobs.

Every call goes through the C ABI of include/iq.h (ctypes); torch is used
only for device memory and the current stream.  Launches are asynchronous
on torch's current stream, like the reference's (ops.cuh:3-7).  Where the
reference would fail later inside CUDA_CHECK (exit(1)), these wrappers raise
RuntimeError with the library's message at the call.  There is no CPU
fallback: without libiq.so every entry point raises.
"""
import ctypes
import enum
import os
import typing

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libiq.so")
GROUP = 128

_lib = None


class IqView(ctypes.Structure):
    """iq_view / gpu::QuantView (kernels/ops/ops.cuh:166-172)."""
    _fields_ = [
        ("kind", ctypes.c_int32),
        ("rows", ctypes.c_int64),
        ("cols", ctypes.c_int64),
        ("groups", ctypes.c_int64),
        ("q", ctypes.c_void_p),
        ("scales", ctypes.c_void_p),
        ("zeros", ctypes.c_void_p),
    ]


class IqStage(ctypes.Structure):
    """iq_stage (include/iq.h): one stage of a chain."""
    _fields_ = [
        ("in_op", ctypes.c_int32),
        ("out_op", ctypes.c_int32),
        ("n", ctypes.c_int32),
        ("gqa_head_dim", ctypes.c_int32),
        ("gqa_group", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("x", ctypes.c_void_p),
        ("norm", ctypes.c_void_p),
        ("residual", ctypes.c_void_p),
        ("W", IqView * 3),
        ("bias", ctypes.c_void_p * 3),
        ("y", ctypes.c_void_p * 3),
        ("rows", ctypes.c_int32),
    ]


class IqKv(ctypes.Structure):
    """iq_kv (include/iq.h): a paged key/value cache."""
    _fields_ = [
        ("type", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("pages", ctypes.c_int64),
        ("page_stride", ctypes.c_int64),
        ("slot_stride", ctypes.c_int64),
        ("head_stride", ctypes.c_int64),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
    ]


# Every function include/iq.h declares, with its ctypes signature.
_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_VP = ctypes.POINTER(IqView)
_KV = ctypes.POINTER(IqKv)
_INT = ctypes.c_int
SIGNATURES = {
    "iq_gemv": ([_P, _VP, _P, ctypes.c_int, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_gemv_noalloc": ([_P, _VP, _P, ctypes.c_int, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_gemv_prep": ([_P, ctypes.c_int, _I64, ctypes.c_int, _P], ctypes.c_int),
    "iq_gemv_prepped": ([_VP, _P, ctypes.c_int, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_gemv_prepped_multi": ([_P, ctypes.c_int, _P, ctypes.c_int, _I64, _P, _P], ctypes.c_int),
    "iq_gemv_multi": ([_P, _P, ctypes.c_int, _P, ctypes.c_int, _I64, _P, _P], ctypes.c_int),
    "iq_gemm": ([_P, _VP, _P, _I64, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_gemm_bf16x": ([_P, _VP, _P, _I64, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_linear": ([_P, _VP, _P, _I64, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_embedding": ([_VP, _P, _I64, _I64, _P, _P], ctypes.c_int),
    "iq_quantize": ([_P, _I64, _I64, ctypes.c_int, _P, _P, _P, _P], ctypes.c_int),
    "iq_chain_create": ([ctypes.POINTER(IqStage), ctypes.c_int, ctypes.POINTER(_P)], ctypes.c_int),
    "iq_chain_run": ([_P, _P], ctypes.c_int),
    "iq_chain_destroy": ([_P], None),
    "iq_kv_append": ([_P, _P, _P, _P, _P, _I64, _INT, _P, _INT, _KV, _P, _P], _INT),
    "iq_attn_decode": ([_P, _KV, _P, _I64, _I64, _P, _INT, _INT, ctypes.c_float, _P, _P, _I64, _P], _INT),
    "iq_kv_evict": ([_KV, _P, _I64, _I64, _P, _INT, _I64, _I64, _P, _I64, _P, _P], _INT),
    "iq_logprobs": ([_P, _I64, _I64, _I64, _P, _INT, _P, _P, _P, _P, _P], _INT),
    "iq_init": ([ctypes.c_int], ctypes.c_int),
    "iq_init_stream": ([ctypes.c_int, _P], ctypes.c_int),
    "iq_error_string": ([ctypes.c_int], ctypes.c_char_p),
    "iq_version": ([], ctypes.c_char_p),
}


def lib():
    """Loads libiq.so (built by infer_amd.build).  Raises when it is missing:
    the quantised path has no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built; run `python -m infer_amd.build`")
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in SIGNATURES.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = res
        _lib = L
    return _lib


def _check(rc, what):
    if rc != 0:
        msg = lib().iq_error_string(rc).decode()
        raise RuntimeError(f"{what}: {msg} (code {rc})")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


# The current stream's handle without the Stream object around it (0.1 us a
# call against 2.9 for torch.cuda.current_stream(), where torch has it).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream):
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


class QuantKind(enum.IntEnum):
    """gpu::QuantKind (kernels/ops/ops.cuh:165)."""
    kInt8 = 0
    kInt4 = 1


def groups_of(cols):
    return (cols + GROUP - 1) // GROUP


class QuantView:
    """A quantised [rows x cols] matrix resident on the device (the packed
    layout of src/quant.h:34-58).  Owns its tensors (the reference's DevTensor
    owns q/scales/zeros and hands out the POD QuantView)."""

    def __init__(self, kind, rows, cols, q, scales, zeros=None):
        self.kind = QuantKind(kind)
        self.rows = int(rows)
        self.cols = int(cols)
        self.groups = groups_of(self.cols)
        self.q = q
        self.scales = scales
        self.zeros = zeros
        self._c = IqView(int(self.kind), self.rows, self.cols, self.groups,
                         q.data_ptr(), scales.data_ptr(),
                         zeros.data_ptr() if zeros is not None else None)

    @property
    def c(self):
        return ctypes.byref(self._c)

    def q_bytes(self):
        return self.rows * self.cols // 2 if self.kind == QuantKind.kInt4 else self.rows * self.cols

    def nbytes(self):
        """Packed bytes: codes + bf16 scales (+ u8 zeros)."""
        n = self.q_bytes() + 2 * self.rows * self.groups
        if self.kind == QuantKind.kInt4:
            n += self.rows * self.groups
        return n


def alloc_quant(kind, rows, cols, device="cuda"):
    kind = QuantKind(kind)
    G = groups_of(cols)
    nq = rows * cols // 2 if kind == QuantKind.kInt4 else rows * cols
    q = torch.empty(nq, dtype=torch.uint8, device=device)
    s = torch.empty(rows * G, dtype=torch.int16, device=device)
    z = torch.empty(rows * G, dtype=torch.uint8, device=device) if kind == QuantKind.kInt4 else None
    return QuantView(kind, rows, cols, q, s, z)


def quantize(w_bf16, kind, out=None, stream=None):
    """llm::quantize (src/quant.cpp:34-84) on the device: w_bf16 is a
    [rows, cols] torch.bfloat16 (or int16 bf16-bit) CUDA tensor.  Returns a
    QuantView (allocated unless `out` is given)."""
    if w_bf16.dim() != 2:
        raise ValueError("quantize: expected a 2-D weight")
    rows, cols = w_bf16.shape
    kind = QuantKind(kind)
    if kind == QuantKind.kInt4 and cols % 2:
        raise ValueError("quantize: int4 needs even cols")
    w = w_bf16.contiguous()
    if out is None:
        out = alloc_quant(kind, rows, cols, device=w.device)
    rc = lib().iq_quantize(_ptr(w), rows, cols, int(kind), _ptr(out.q), _ptr(out.scales),
                           _ptr(out.zeros), _stream(stream))
    _check(rc, "iq_quantize")
    return out


def upload_q(kind, rows, cols, q, scales, zeros=None, device="cuda"):
    """DevTensor::upload_q (kernels/model_gpu_internal.cuh:67-83): numpy
    arrays of the packed layout (q u8, scales u16 bf16 bits, zeros u8) ->
    device QuantView."""
    import numpy as np

    def dev(a, npdt, tdt):
        return torch.from_numpy(np.ascontiguousarray(a).reshape(-1).view(npdt)).to(device)

    qd = dev(q, np.uint8, torch.uint8)
    sd = dev(scales, np.int16, torch.int16)
    zd = dev(zeros, np.uint8, torch.uint8) if zeros is not None else None
    return QuantView(kind, rows, cols, qd, sd, zd)


def _bias_ptr(bias):
    if bias is None:
        return None
    if bias.dtype not in (torch.bfloat16, torch.int16):
        raise TypeError("bias must be bf16 (torch.bfloat16 or int16 bits)")
    return _ptr(bias)


def launch_gemv_batched_q(x, W, bias, B, in_, out, y, stream=None):
    """y[b, o] = sum_c dequant(W, o, c) x[b, c] (+ bias[o]) for b < B <= 32."""
    rc = lib().iq_gemv(_ptr(x), W.c, _bias_ptr(bias), int(B), int(in_), int(out), _ptr(y), _stream(stream))
    _check(rc, "iq_gemv")


def gemv_noalloc(x, W, bias, B, in_, out, y, stream=None):
    """launch_gemv_batched_q on the library's static scratch (no allocation;
    in <= 32768; calls that overlap on one device race)."""
    rc = lib().iq_gemv_noalloc(_ptr(x), W.c, _bias_ptr(bias), int(B), int(in_), int(out), _ptr(y), _stream(stream))
    _check(rc, "iq_gemv_noalloc")


def gemv_prep(x, B, in_, kind, stream=None):
    """Prepare activations x [B, in] once for several GEMVs of one kind."""
    rc = lib().iq_gemv_prep(_ptr(x), int(B), int(in_), int(kind), _stream(stream))
    _check(rc, "iq_gemv_prep")


def gemv_prepped(W, bias, B, in_, out, y, stream=None):
    """GEMV of W on the activations of the last gemv_prep."""
    rc = lib().iq_gemv_prepped(W.c, _bias_ptr(bias), int(B), int(in_), int(out), _ptr(y), _stream(stream))
    _check(rc, "iq_gemv_prepped")


def gemv_prepped_multi(Ws, biases, B, in_, ys, stream=None):
    """Several matrices (same kind and width) on the last gemv_prep's
    activations in one call: ys[i] = x @ dequant(Ws[i])^T (+ biases[i])."""
    n = len(Ws)
    views = (ctypes.c_void_p * n)(*[ctypes.addressof(W._c) for W in Ws])
    bs = (ctypes.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in (biases or [None] * n)])
    yp = (ctypes.c_void_p * n)(*[y.data_ptr() for y in ys])
    rc = lib().iq_gemv_prepped_multi(views, n, bs, int(B), int(in_), yp, _stream(stream))
    _check(rc, "iq_gemv_prepped_multi")


def gemv_multi(x, Ws, biases, B, in_, ys, stream=None):
    """Several matrices (same kind and width) sharing the activations
    x [B, in]: ys[i] = x @ dequant(Ws[i])^T (+ biases[i]); one launch at B = 1."""
    n = len(Ws)
    views = (ctypes.c_void_p * n)(*[ctypes.addressof(W._c) for W in Ws])
    bs = (ctypes.c_void_p * n)(*[(b.data_ptr() if b is not None else None) for b in (biases or [None] * n)])
    yp = (ctypes.c_void_p * n)(*[y.data_ptr() for y in ys])
    rc = lib().iq_gemv_multi(_ptr(x), views, n, bs, int(B), int(in_), yp, _stream(stream))
    _check(rc, "iq_gemv_multi")


def launch_gemm_tiled_q(x, W, bias, T, in_, out, y, stream=None):
    """Same contract for any T (the prefill GEMM), fp32 activations."""
    rc = lib().iq_gemm(_ptr(x), W.c, _bias_ptr(bias), int(T), int(in_), int(out), _ptr(y), _stream(stream))
    _check(rc, "iq_gemm")


def launch_gemm_bf16x(x_bf16, W, bias, T, in_, out, y, stream=None):
    """Prefill GEMM with bf16 activations (fp32 output)."""
    rc = lib().iq_gemm_bf16x(_ptr(x_bf16), W.c, _bias_ptr(bias), int(T), int(in_), int(out), _ptr(y),
                             _stream(stream))
    _check(rc, "iq_gemm_bf16x")


def launch_linear_q(x, W, bias, T, in_, out, y, stream=None):
    """GpuBatch::Impl::linear_b quantised branch (kernels/batch_gpu.cu:137-147)."""
    rc = lib().iq_linear(_ptr(x), W.c, _bias_ptr(bias), int(T), int(in_), int(out), _ptr(y), _stream(stream))
    _check(rc, "iq_linear")


def launch_embedding_q(table, ids, T, H, out, stream=None):
    """out[t, i] = dequant(table, ids[t], i)."""
    rc = lib().iq_embedding(table.c, _ptr(ids), int(T), int(H), _ptr(out), _stream(stream))
    _check(rc, "iq_embedding")


def linear(x, W, bias=None, stream=None):
    """Allocating convenience: y = x @ dequant(W)^T (+ bias), x [T, in] fp32."""
    T, K = x.shape
    y = torch.empty(T, W.rows, dtype=torch.float32, device=x.device)
    launch_linear_q(x.contiguous(), W, bias, T, K, W.rows, y, stream)
    return y


# ------------------------------------------------ the cache of a decode step
KV_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _addr(t):
    return None if t is None else t.data_ptr()


class KvCache:
    """A paged key/value cache (include/iq.h, iq_kv) over two tensors k, v of
    [pages, page_size, kv_heads, head_dim], torch.bfloat16 or torch.float16,
    which it keeps alive.  Any memory order of pages, slots and heads (a
    permuted view, a slice of a larger tensor) whose rows of head_dim values
    are contiguous, with the same strides for k and v."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("KvCache: k and v must be [pages, page_size, kv_heads, head_dim] of one shape and type")
        if k.dtype not in KV_TYPES:
            raise TypeError("KvCache: k and v must be torch.bfloat16 or torch.float16")
        # (the stride over a single page, slot or head means nothing)
        strides = [[0 if n == 1 else s for n, s in zip(t.shape, t.stride())] for t in (k, v)]
        if strides[0] != strides[1] or strides[0][3] not in (0, 1):
            raise ValueError("KvCache: k and v need the same strides and contiguous rows of head_dim values")
        self.k, self.v = k, v
        self.pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.device = k.get_device()
        if v.get_device() != self.device:
            raise ValueError("KvCache: k and v must be on one device")
        self._c = IqKv(KV_TYPES[k.dtype], self.kv_heads, self.head_dim, self.page_size, self.pages,
                       *strides[0][:3], k.data_ptr(), v.data_ptr())

    @property
    def c(self):
        return ctypes.byref(self._c)


def alloc_kv(pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
    """An empty cache (zeros) in the order [pages, page_size, kv_heads, head_dim]."""
    shape = (pages, page_size, kv_heads, head_dim)
    return KvCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))


def rope_freqs(rot_dim, theta, device="cuda"):
    """theta^(-2i / rot_dim), i < rot_dim / 2, in double: kv_append's freqs."""
    return torch.tensor([theta ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)], dtype=torch.float64,
                        device=device)


def _need(what, name, t, dtype, numel=None):
    """A contiguous tensor of this type (and number of elements)."""
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} must be {dtype}, not {t.dtype}")
    if not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{what}: {name} must be contiguous" + ("" if numel is None else f" with {numel} elements"))


def _on_device(what, device, *tensors):
    """Every tensor on `device`, which is the current CUDA device."""
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError(f"{what}: tensors on different devices")
    if device < 0 or device != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors must be on the current CUDA device")


def _new(stream, make, *args, **kw):
    """An output made here: from the memory of the stream that writes it."""
    if stream is None:
        return make(*args, **kw)
    with torch.cuda.stream(stream):
        return make(*args, **kw)


def kv_append(q, k, v, positions, slots, freqs, cache, q_out=None, stream=None):
    """Rotary embedding of q [T, heads, head_dim] (into q_out, may be q) and
    k [T, kv_heads, head_dim] at positions [T], k and v [T, kv_heads, head_dim]
    into cache slots [T] = page * page_size + slot (outside the pool: not
    stored; all others different).  fp32 inputs, int64 positions and slots,
    freqs: rope_freqs, or None (no rotation; positions may be None).  q may be
    None (cache only).  Returns q_out.  include/iq.h, iq_kv_append."""
    what = "kv_append"
    T, d = slots.numel(), cache.head_dim
    _need(what, "slots", slots, torch.int64)
    _need(what, "k", k, torch.float32, T * cache.kv_heads * d)
    _need(what, "v", v, torch.float32, T * cache.kv_heads * d)
    rot = 0
    if freqs is not None:
        if positions is None:
            raise ValueError(f"{what}: freqs need positions")
        _need(what, "freqs", freqs, torch.float64)
        _need(what, "positions", positions, torch.int64, T)
        rot = 2 * freqs.numel()
    heads = 0
    if q is not None:
        heads = q.numel() // max(1, T * d)
        _need(what, "q", q, torch.float32, T * heads * d)
        if q_out is not None:
            _need(what, "q_out", q_out, torch.float32, T * heads * d)
    _on_device(what, cache.device, q, k, v, positions if rot else None, slots, freqs, q_out)
    if q is not None and q_out is None:
        q_out = _new(stream, torch.empty_like, q)
    rc = lib().iq_kv_append(_addr(q), _addr(k), _addr(v), _addr(positions) if rot else None, _addr(slots), T, heads,
                            _addr(freqs) if rot else None, rot, cache.c, _addr(q_out) if heads else None,
                            _stream(stream))
    _check(rc, "iq_kv_append")
    return q_out


def _check_table(what, table, lens):
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"{what}: table must be int32 [sequences, pages] with contiguous rows")
    B, pages = table.shape
    _need(what, "lens", lens, torch.int32, B)
    ld = table.stride(0) if B > 1 else pages
    return B, pages, ld


def _check_sums(what, weights, B, kv_heads):
    """fp32 [sequences, kv_heads, tokens], sequences and heads packed."""
    if weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (B, kv_heads):
        raise ValueError(f"{what}: weights must be float32 [sequences, kv_heads, tokens]")
    if not weights.is_contiguous():
        raise ValueError(f"{what}: weights must be contiguous")
    return weights.shape[2]


def attn_decode(q, cache, table, lens, out=None, weights=None, scale=None, stream=None):
    """Attention of one token a sequence, q [B, heads, head_dim] fp32, over
    the first lens[b] (int32 [B]) tokens in the pages table[b] (int32 [B,
    pages]) of the cache; heads / kv_heads query heads share a key/value head.
    scale: head_dim^-0.5 by default.  weights: fp32 [B, kv_heads, tokens],
    tokens >= pages * page_size; every cached token's attention weight, summed
    over the heads that share it, is added to it.  Returns out, shaped as q.
    include/iq.h, iq_attn_decode."""
    what = "attn_decode"
    B, pages, ld = _check_table(what, table, lens)
    d = cache.head_dim
    heads = q.numel() // max(1, B * d)
    _need(what, "q", q, torch.float32, B * heads * d)
    wld = 0 if weights is None else _check_sums(what, weights, B, cache.kv_heads)
    if out is not None:
        _need(what, "out", out, torch.float32, B * heads * d)
    _on_device(what, cache.device, q, table, lens, out, weights)
    if out is None:
        out = _new(stream, torch.empty_like, q)
    rc = lib().iq_attn_decode(_addr(q), cache.c, _addr(table), ld, pages, _addr(lens), B, heads,
                              d ** -0.5 if scale is None else scale, _addr(out), _addr(weights), wld, _stream(stream))
    _check(rc, "iq_attn_decode")
    return out


def kv_evict(cache, table, lens, weights, budget, recent, new_lens=None, stream=None):
    """Cuts every sequence of more than `budget` tokens to `budget`, for each
    key/value head by itself: the newest `recent` stay and, of the others,
    those of the largest weights (fp32 [B, kv_heads, tokens], which move along;
    entries past the budget become 0).  The newest are the tokens in the last
    slots: after a call that cut a sequence, `recent` must not be more than that
    call's `recent` and the tokens appended since.  Returns new_lens (int32 [B]), min(lens,
    budget): the pages past it are free.  include/iq.h, iq_kv_evict."""
    what = "kv_evict"
    B, pages, ld = _check_table(what, table, lens)
    wld = _check_sums(what, weights, B, cache.kv_heads)
    if new_lens is not None:
        _need(what, "new_lens", new_lens, torch.int32, B)
    _on_device(what, cache.device, table, lens, weights, new_lens)
    if new_lens is None:
        new_lens = _new(stream, torch.empty_like, lens)
    rc = lib().iq_kv_evict(cache.c, _addr(table), ld, pages, _addr(lens), B, int(budget), int(recent), _addr(weights),
                           wld, _addr(new_lens), _stream(stream))
    _check(rc, "iq_kv_evict")
    return new_lens


class LogProbs(typing.NamedTuple):
    """logprobs' outputs; top_ids and top_logprobs are None with top = 0,
    logprob is None without tokens (or is not written, in a given buffer)."""
    logprob: typing.Optional[torch.Tensor]
    entropy: typing.Optional[torch.Tensor]
    top_ids: typing.Optional[torch.Tensor]
    top_logprobs: typing.Optional[torch.Tensor]


def alloc_logprobs(T, top=0, device="cuda"):
    """Buffers for logprobs' outputs of T rows."""
    f = dict(dtype=torch.float32, device=device)
    return LogProbs(torch.empty(T, **f), torch.empty(T, **f),
                    torch.empty(T, top, dtype=torch.int64, device=device) if top else None,
                    torch.empty(T, top, **f) if top else None)


def logprobs(logits, tokens=None, top=0, out=None, stream=None):
    """For rows of logits [T, V] fp32 (any row stride): the log probability of
    tokens[t] (int64 [T]; NaN outside [0, V)), the entropy, and the `top` (<=
    64) most likely ids with their log probabilities (equal logits: the lower
    id first).  out: alloc_logprobs(T, top).  Returns LogProbs.
    include/iq.h, iq_logprobs."""
    what = "logprobs"
    if logits.dtype != torch.float32 or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError(f"{what}: logits must be float32 [T, V] with contiguous rows")
    T, V = logits.shape
    ld = logits.stride(0) if T > 1 else V
    if tokens is not None:
        _need(what, "tokens", tokens, torch.int64, T)
    if out is None:
        out = _new(stream, alloc_logprobs, T, top, device=logits.device)
    lp, ent, ids, tlp = out
    if tokens is None:
        lp = None
    elif lp is None:
        raise ValueError(f"{what}: out has no logprob")
    for name, t, dt, n in (("logprob", lp, torch.float32, T), ("entropy", ent, torch.float32, T)):
        if t is not None:
            _need(what, name, t, dt, n)
    if top:
        if ids is None or tlp is None:
            raise ValueError(f"{what}: out has no top_ids and top_logprobs")
        _need(what, "top_ids", ids, torch.int64, T * top)
        _need(what, "top_logprobs", tlp, torch.float32, T * top)
    else:
        ids = tlp = None
    _on_device(what, logits.get_device(), logits, tokens, lp, ent, ids, tlp)
    rc = lib().iq_logprobs(_addr(logits), ld, T, V, _addr(tokens), int(top), _addr(lp), _addr(ent), _addr(ids), _addr(tlp),
                           _stream(stream))
    _check(rc, "iq_logprobs")
    return LogProbs(lp, ent, ids, tlp)


def init(device=0, stream=None):
    """Reserve the workspace of (device, stream) before a graph capture."""
    if stream is None:
        _check(lib().iq_init(int(device)), "iq_init")
    else:
        _check(lib().iq_init_stream(int(device), ctypes.c_void_p(stream.cuda_stream)), "iq_init_stream")
