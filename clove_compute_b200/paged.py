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
_16BIT = (torch.float16, torch.bfloat16)


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
        self.dtype, self.device = K.dtype, K.device
        self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        self.struct = PagedCacheStruct(K.data_ptr(), V.data_ptr(), self.num_pages, self.page_size,
                                       self.num_kv_heads, self.head_dim, K.stride(0), K.stride(tok),
                                       K.stride(head), DTYPES[K.dtype], self.k_scale, self.v_scale)
        self._address = ctypes.addressof(self.struct)


def _ints(t, name, device, shape):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be torch.int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _table(t, name, device, batch):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be torch.int32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.dim() != 2 or t.shape[0] != batch:
        raise ValueError(f"{name} must be [{batch}, pages], got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    return t.data_ptr()


def _heads(t, name, dtype, device, shape):
    """A [rows, heads, D] operand whose rows are contiguous; its row stride."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    s = t.stride()
    if s[2] != 1 or (shape[1] > 1 and s[1] != shape[2]):
        raise ValueError(f"{name}: the last two dimensions must be contiguous")
    return s[0] if shape[0] > 1 else shape[1] * shape[2]


def _floats(t, name, device, shape):
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _operand(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in _16BIT:
        raise TypeError(f"{name} must be an fp16 or bf16 tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 3:
        raise ValueError(f"{name} must be 3-D, got shape {tuple(t.shape)}")


# The current stream's handle, without the Stream object that torch.cuda.current_stream()
# builds (2 us a call).
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(fn, device, stream, *args):
    """fn(stream handle, *args) with `device` current; an explicit stream is current while
    outputs are allocated, so that their memory belongs to it."""
    if stream is not None:
        s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=device)
        with torch.cuda.device(device), torch.cuda.stream(s):
            return fn(s.cuda_stream, *args)
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return fn(_current_stream(device.index), *args)
    return fn(_current_stream(device.index), *args)


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
    _operand(Q, "Q")
    _operand(K, "K")
    return _on(_qk_norm_rope, Q.device, stream, Q, K, rope_table, positions, q_weight, k_weight, eps,
               interleaved, V, cache, slots, Q_out, K_out)


def _qk_norm_rope(stream, Q, K, table, positions, q_weight, k_weight, eps, interleaved, V, cache, slots,
                  Q_out, K_out):
    dtype, device = Q.dtype, Q.device
    T, H, D = Q.shape
    Hkv = K.shape[1]
    kv = (T, Hkv, D)
    qs = _heads(Q, "Q", dtype, device, (T, H, D))
    ks = _heads(K, "K", dtype, device, kv)
    if table.dim() != 2:
        raise ValueError("rope_table must be [positions, rotary_dim]")
    tp = _floats(table, "rope_table", device, table.shape)
    pp = _ints(positions, "positions", device, (T,))
    wq = wk = None
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight: both or neither")
    if q_weight is not None:
        for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")):
            if w.dtype != dtype or w.device != device or w.shape != (D,) or not w.is_contiguous():
                raise ValueError(f"{n} must be a contiguous [{D}] tensor of {dtype} on {device}")
        wq, wk = q_weight.data_ptr(), k_weight.data_ptr()
    vs = 0
    vp = sp = ref = None
    if cache is not None:
        if V is None or slots is None:
            raise ValueError("a cache needs V and slots")
        if cache.device != device:
            raise ValueError(f"the cache must be on {device}")
        vs = _heads(V, "V", dtype, device, kv)
        vp, sp, ref = V.data_ptr(), _ints(slots, "slots", device, (T,)), cache._address
    elif V is not None or slots is not None:
        raise ValueError("V and slots need a cache")
    if Q_out is None:
        Q_out = torch.empty((T, H, D), dtype=dtype, device=device)
        qos = H * D
    else:
        qos = _heads(Q_out, "Q_out", dtype, device, (T, H, D))
    if K_out is None and cache is None:
        K_out = torch.empty(kv, dtype=dtype, device=device)
    kos = _heads(K_out, "K_out", dtype, device, kv) if K_out is not None else 0
    rc = fastcall().qk_norm_rope(
        Q.data_ptr(), K.data_ptr(), vp, qs, ks, vs, wq, wk, eps, tp, table.shape[0], table.shape[1],
        1 if interleaved else 0, pp, ref, sp, Q_out.data_ptr(), qos,
        K_out.data_ptr() if K_out is not None else None, kos, T, H, Hkv, D, DTYPES[dtype], stream)
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
    _operand(Q, "Q")
    return _on(_paged_attention, Q.device, stream, Q, cache, page_table, seq_lens, scale, window, lse,
               key_weights, accumulate, O)


def _paged_attention(stream, Q, cache, page_table, seq_lens, scale, window, lse, key_weights, accumulate, O):
    dtype, device = Q.dtype, Q.device
    B, H, D = Q.shape
    if cache.device != device:
        raise ValueError(f"the cache must be on {device}")
    if D != cache.head_dim:
        raise ValueError(f"Q has head_dim {D}, the cache {cache.head_dim}")
    qs = _heads(Q, "Q", dtype, device, (B, H, D))
    pt = _table(page_table, "page_table", device, B)
    sl = _ints(seq_lens, "seq_lens", device, (B,))
    if O is None:
        O = torch.empty((B, H, D), dtype=dtype, device=device)
        os = H * D
    else:
        os = _heads(O, "O", dtype, device, (B, H, D))
    lp = _floats(lse, "lse", device, (B, H)) if lse is not None else None
    kw = None
    if key_weights is not None:
        kw = _floats(key_weights, "key_weights", device,
                     (cache.num_pages, cache.num_kv_heads, cache.page_size))
    elif accumulate:
        raise ValueError("accumulate needs key_weights")
    rc = fastcall().paged_attention(
        Q.data_ptr(), qs, cache._address, pt, page_table.stride(0), page_table.shape[1], sl, O.data_ptr(), os,
        lp, kw, 1 if accumulate else 0, B, H, D ** -0.5 if scale is None else scale, window,
        DTYPES[dtype], stream)
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
    if not cache.K.is_cuda:
        raise ValueError("the cache must be on a CUDA device")
    return _on(_evict_cache, cache.device, stream, cache, key_weights, page_table, seq_lens, dst_table,
               budget, recent)


def _evict_cache(stream, cache, key_weights, page_table, seq_lens, dst_table, budget, recent):
    device = cache.device
    B = seq_lens.shape[0]
    kw = _floats(key_weights, "key_weights", device,
                 (cache.num_pages, cache.num_kv_heads, cache.page_size))
    pt = _table(page_table, "page_table", device, B)
    dt = _table(dst_table, "dst_table", device, B)
    sl = _ints(seq_lens, "seq_lens", device, (B,))
    if budget <= 0:
        raise ValueError("budget must be positive")
    kept = torch.empty((B, cache.num_kv_heads, budget), dtype=torch.int32, device=device)
    new_lens = torch.empty((B,), dtype=torch.int32, device=device)
    rc = fastcall().evict_cache(
        cache._address, kw, pt, page_table.stride(0), page_table.shape[1], sl, dt, dst_table.stride(0),
        dst_table.shape[1], kept.data_ptr(), new_lens.data_ptr(), B, budget, recent, stream)
    if rc:
        check(rc)
    return kept, new_lens
