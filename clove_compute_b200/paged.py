"""Tensor-level API of the paged key-value cache: the decode step's operators.

:class:`PagedCache` describes K and V pages once; :func:`qk_norm_rope` fills it,
:func:`paged_attention` reads it (the reference declares ``paged_attention``,
``include/clove/kernels/attention.cuh:85-100``, and never defines it) and
:func:`evict_cache` shortens it. Index tensors are int32 on the device and are read
there, so a captured call can be replayed while sequences grow. Over the C ABI of
``include/clove/capi.h``; wrong arguments raise ``TypeError`` / ``ValueError`` here or
:class:`CloveError` from the library. Indices outside their range are not followed:
``device_error()`` then returns 3.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import PagedCacheStruct, check, fastcall

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}


class PagedCache:
    """K and V pages of a key-value cache (kept alive by this object).

    layout "bshd": K, V [pages, page_size, kv_heads, head_dim]; "bhsd": [pages, kv_heads,
    page_size, head_dim]. fp16, bf16 or float8_e4m3fn; any strides that are multiples of
    16 bytes, the same for K and V, the last dimension contiguous (so K and V may be
    halves of one buffer). page_size a power of two; head_dim 64, 128 or 256. An e4m3
    value x stands for x * k_scale (x * v_scale)."""

    def __init__(self, K: torch.Tensor, V: torch.Tensor, layout: str = "bshd",
                 k_scale: float = 1.0, v_scale: float = 1.0):
        for t, n in ((K, "K"), (V, "V")):
            if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES:
                raise TypeError(f"{n} must be an fp16, bf16 or float8_e4m3fn tensor")
            if not t.is_cuda:
                raise ValueError(f"{n} must be a CUDA tensor")
            if t.dim() != 4:
                raise ValueError(f"{n} must be 4-D, got shape {tuple(t.shape)}")
        if layout not in ("bshd", "bhsd"):
            raise ValueError("layout must be 'bshd' or 'bhsd'")
        if K.shape != V.shape or K.dtype != V.dtype or K.device != V.device or K.stride() != V.stride():
            raise ValueError("K and V must agree in shape, strides, dtype and device")
        if K.numel() == 0:
            raise ValueError("the cache has no slots")
        if K.stride(3) != 1:
            raise ValueError("the last dimension of K and V must be contiguous")
        tok, head = (1, 2) if layout == "bshd" else (2, 1)
        self.K, self.V, self.layout = K, V, layout
        self.num_pages, self.page_size = K.shape[0], K.shape[tok]
        self.num_kv_heads, self.head_dim = K.shape[head], K.shape[3]
        self.dtype, self.device, self.index = K.dtype, K.device, K.get_device()
        self.weights_shape = (self.num_pages, self.num_kv_heads, self.page_size)  # of key_weights
        self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        self.struct = PagedCacheStruct(K.data_ptr(), V.data_ptr(), self.num_pages, self.page_size,
                                       self.num_kv_heads, self.head_dim, K.stride(0), K.stride(tok),
                                       K.stride(head), DTYPES[K.dtype], self.k_scale, self.v_scale)
        self._address = ctypes.addressof(self.struct)


# Checks of the operands. They run on every call of a decode step, so each attribute is
# read once and devices are compared by index.
def _no(t, name, want):
    raise ValueError(f"{name} must be {want}, got {tuple(t.shape)} on {t.device}")


def _dense(t, name, dtype, index, shape):
    """A contiguous tensor of this type and shape on GPU `index`; its address."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index or t.shape != shape or not t.is_contiguous():
        _no(t, name, f"contiguous {tuple(shape)} on GPU {index}")
    return t.data_ptr()


def _table(t, name, index, batch):
    """A [batch, pages] int32 tensor with contiguous rows; its address, pages and row stride."""
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be torch.int32, got {t.dtype}")
    s = t.stride()
    if t.get_device() != index or len(s) != 2 or t.shape[0] != batch or (s[1] != 1 and t.shape[1] > 1):
        _no(t, name, f"[{batch}, pages] with contiguous rows on GPU {index}")
    return t.data_ptr(), t.shape[1], s[0]


def _heads(t, name, dtype, index, shape):
    """A [rows, heads, D] operand whose rows are contiguous; its row stride."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    s = t.stride()
    if t.get_device() != index or t.shape != shape or s[2] != 1 or (s[1] != shape[2] and shape[1] > 1):
        _no(t, name, f"{tuple(shape)} with contiguous rows on GPU {index}")
    return s[0] if shape[0] > 1 else shape[1] * shape[2]


def _operand(t, name):
    """(dtype code, GPU index, shape) of the call's first operand."""
    code = DTYPES.get(t.dtype, 2) if isinstance(t, torch.Tensor) else 2
    if code == 2:
        raise TypeError(f"{name} must be an fp16 or bf16 tensor")
    index, shape = t.get_device(), t.shape
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if len(shape) != 3:
        raise ValueError(f"{name} must be 3-D, got shape {tuple(shape)}")
    return code, index, shape


# The current stream's handle and device without the objects that torch.cuda's own
# functions build or look up (3 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _elsewhere(fn, index, stream, *args):
    """fn(stream handle, ...) for a stream or device other than the current one. The stream
    is current while outputs are allocated, so that their memory belongs to it."""
    with torch.cuda.device(index):
        if stream is None:
            return fn(_raw_stream(index), *args)
        s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=index)
        with torch.cuda.stream(s):
            return fn(s.cuda_stream, *args)


def rope_table(length: int, rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """The rotation table of :func:`qk_norm_rope`: [length, rotary_dim] fp32, row p holding
    cos(p * theta^(-2i / rotary_dim)) for i < rotary_dim / 2, then the sines. The angles
    are taken in 64 bits: in 32 the far positions would lose their fraction of a turn."""
    if length <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("length must be positive, rotary_dim positive and even")
    inv = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    a = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return torch.cat([a.cos(), a.sin()], 1).to(torch.float32)


def qk_norm_rope(Q, K, rope_table, positions, q_weight=None, k_weight=None, eps: float = 1e-6,
                 interleaved: bool = False, V=None, cache: PagedCache | None = None, slots=None,
                 Q_out=None, K_out=None, stream=None):
    """Per-head RMS norm of Q [T, heads, D] and K [T, kv_heads, D] (fp16 or bf16; weights
    [D], or none), rotation of the first rope_table.shape[1] (a multiple of 16) elements by
    rope_table[positions], and, with a cache, the rotated K and
    V rows stored at its `slots`. Rows may be column blocks of a fused projection. Returns
    (Q_out, K_out); with a cache K_out is None unless it was given. Q_out may be Q and
    K_out K. Negative positions mark padding tokens (nothing written), negative slots
    tokens that are not stored; other slots must differ."""
    code, index, shape = _operand(Q, "Q")
    args = (code, index, shape, Q, K, rope_table, positions, q_weight, k_weight, eps, interleaved, V, cache,
            slots, Q_out, K_out)
    if stream is not None or index != _current_device():
        return _elsewhere(_qk_norm_rope, index, stream, *args)
    return _qk_norm_rope(_raw_stream(index), *args)


def _qk_norm_rope(stream, code, index, shape, Q, K, table, positions, q_weight, k_weight, eps, interleaved, V,
                  cache, slots, Q_out, K_out):
    dtype = Q.dtype
    T, H, D = shape
    kv = K.shape
    if len(kv) != 3 or kv[0] != T or kv[2] != D:
        raise ValueError(f"K must be [{T}, kv_heads, {D}], got {tuple(kv)}")
    qs = _heads(Q, "Q", dtype, index, shape)
    ks = _heads(K, "K", dtype, index, kv)
    ts = table.shape
    if len(ts) != 2:
        raise ValueError("rope_table must be [positions, rotary_dim]")
    tp = _dense(table, "rope_table", torch.float32, index, ts)
    pp = _dense(positions, "positions", torch.int32, index, (T,))
    wq = wk = None
    if q_weight is not None and k_weight is not None:
        wq = _dense(q_weight, "q_weight", dtype, index, (D,))
        wk = _dense(k_weight, "k_weight", dtype, index, (D,))
    elif q_weight is not k_weight:
        raise ValueError("q_weight and k_weight: both or neither")
    vs = kos = 0
    vp = sp = ref = kp = None
    if cache is not None:
        if V is None or slots is None:
            raise ValueError("a cache needs V and slots")
        if cache.index != index:
            raise ValueError(f"the cache must be on GPU {index}")
        vs = _heads(V, "V", dtype, index, kv)
        vp, sp, ref = V.data_ptr(), _dense(slots, "slots", torch.int32, index, (T,)), cache._address
    elif V is not None or slots is not None:
        raise ValueError("V and slots need a cache")
    elif K_out is None:
        K_out = torch.empty_like(K, memory_format=torch.contiguous_format)
    if Q_out is None:
        Q_out = torch.empty_like(Q, memory_format=torch.contiguous_format)
        qos = H * D
    else:
        qos = _heads(Q_out, "Q_out", dtype, index, shape)
    if K_out is not None:
        kos = _heads(K_out, "K_out", dtype, index, kv)
        kp = K_out.data_ptr()
    rc = fastcall().qk_norm_rope(
        Q.data_ptr(), K.data_ptr(), vp, qs, ks, vs, wq, wk, eps, tp, ts[0], ts[1], 1 if interleaved else 0,
        pp, ref, sp, Q_out.data_ptr(), qos, kp, kos, T, H, kv[1], D, code, stream)
    if rc:
        check(rc)
    return Q_out, K_out


def paged_attention(Q, cache: PagedCache, page_table, seq_lens, scale: float | None = None,
                    window: int = 0, lse=None, key_weights=None, accumulate: bool = False, O=None,
                    stream=None):
    """Attention of one new token per sequence, Q [B, heads, D] (fp16 or bf16), over the
    first seq_lens[b] cached tokens of page_table[b] (with `window`, the last `window` of
    them; heads a multiple of the cache's). Returns O [B, heads, D].

    lse [B, heads] fp32, if given, gets the log-sum-exp of the scaled scores. key_weights
    [pages, kv_heads, page_size] fp32, if given, gets the softmax weight of every attended
    key, summed over its query heads (added with accumulate=True); no page may then be in
    two sequences. scale defaults to 1/sqrt(D). An empty sequence gives zeros and -inf."""
    code, index, shape = _operand(Q, "Q")
    args = (code, index, shape, Q, cache, page_table, seq_lens, scale, window, lse, key_weights, accumulate, O)
    if stream is not None or index != _current_device():
        return _elsewhere(_paged_attention, index, stream, *args)
    return _paged_attention(_raw_stream(index), *args)


def _paged_attention(stream, code, index, shape, Q, cache, page_table, seq_lens, scale, window, lse,
                     key_weights, accumulate, O):
    dtype = Q.dtype
    B, H, D = shape
    if cache.index != index:
        raise ValueError(f"the cache must be on GPU {index}")
    if D != cache.head_dim:
        raise ValueError(f"Q has head_dim {D}, the cache {cache.head_dim}")
    qs = _heads(Q, "Q", dtype, index, shape)
    pt, pages, ps = _table(page_table, "page_table", index, B)
    sl = _dense(seq_lens, "seq_lens", torch.int32, index, (B,))
    lp = _dense(lse, "lse", torch.float32, index, (B, H)) if lse is not None else None
    kw = None
    if key_weights is not None:
        kw = _dense(key_weights, "key_weights", torch.float32, index, cache.weights_shape)
    elif accumulate:
        raise ValueError("accumulate needs key_weights")
    if O is None:
        O = torch.empty_like(Q, memory_format=torch.contiguous_format)
        os = H * D
    else:
        os = _heads(O, "O", dtype, index, shape)
    rc = fastcall().paged_attention(
        Q.data_ptr(), qs, cache._address, pt, ps, pages, sl, O.data_ptr(), os, lp, kw, 1 if accumulate else 0,
        B, H, D ** -0.5 if scale is None else scale, window, code, stream)
    if rc:
        check(rc)
    return O


def evict_cache(cache: PagedCache, key_weights, page_table, seq_lens, dst_table, budget: int,
                recent: int = 0, stream=None):
    """Shorten every sequence to `budget` tokens: the last `recent` ones and, per kv head,
    those of largest key_weights [pages, kv_heads, page_size] before them (ties: the lowest
    index). Their K, V and weights are copied, in order, to the fresh pages of dst_table
    [B, >= ceil(budget / page_size)], none of which may still be in use. Returns (kept
    [B, kv_heads, budget] int32 -- indices, -1 behind them -- and the new lengths [B])."""
    index = cache.index
    args = (index, cache, key_weights, page_table, seq_lens, dst_table, budget, recent)
    if stream is not None or index != _current_device():
        return _elsewhere(_evict_cache, index, stream, *args)
    return _evict_cache(_raw_stream(index), *args)


def _evict_cache(stream, index, cache, key_weights, page_table, seq_lens, dst_table, budget, recent):
    B = seq_lens.shape[0]
    kw = _dense(key_weights, "key_weights", torch.float32, index, cache.weights_shape)
    pt, pages, ps = _table(page_table, "page_table", index, B)
    dt, dst_pages, ds = _table(dst_table, "dst_table", index, B)
    sl = _dense(seq_lens, "seq_lens", torch.int32, index, (B,))
    if budget <= 0:
        raise ValueError("budget must be positive")
    kept = seq_lens.new_empty((B, cache.num_kv_heads, budget))
    new_lens = torch.empty_like(seq_lens)
    rc = fastcall().evict_cache(
        cache._address, kw, pt, ps, pages, sl, dt, ds, dst_pages, kept.data_ptr(), new_lens.data_ptr(), B,
        budget, recent, stream)
    if rc:
        check(rc)
    return kept, new_lens
