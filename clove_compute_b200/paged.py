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

from ._lib import PagedCacheStruct, check, fastcall, library_path

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
        # (The stride of a dimension of size 1 means nothing.)
        strides, others = ([s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride())] for t in (K, V))
        if K.shape != V.shape or K.dtype != V.dtype or K.device != V.device or strides != others:
            raise ValueError("K and V must agree in shape, strides, dtype and device")
        if K.numel() == 0:
            raise ValueError("the cache has no slots")
        if K.stride(3) != 1 or V.stride(3) != 1:
            raise ValueError("the last dimension of K and V must be contiguous")
        tok, head = (1, 2) if layout == "bshd" else (2, 1)
        self.K, self.V, self.layout = K, V, layout
        self.num_pages, self.page_size = K.shape[0], K.shape[tok]
        self.num_kv_heads, self.head_dim = K.shape[head], K.shape[3]
        self.dtype, self.device, self.index = K.dtype, K.device, K.get_device()
        self.k_scale, self.v_scale = float(k_scale), float(v_scale)
        self.struct = PagedCacheStruct(K.data_ptr(), V.data_ptr(), self.num_pages, self.page_size,
                                       self.num_kv_heads, self.head_dim, strides[0], strides[tok],
                                       strides[head], DTYPES[K.dtype], self.k_scale, self.v_scale)
        self._key = (ctypes.addressof(self.struct), self.index)


# The current stream's handle and the current device, without the objects that torch.cuda's
# own functions build or look up (3 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device

_fast = None


def _load():
    """The operators' CPython entry points (``csrc/binding/fastcall.c``), which check the
    arguments and call the library."""
    global _fast
    if _fast is None:
        f = fastcall()
        f.init(library_path(), (torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32),
               torch.empty_like, torch.contiguous_format, _current_device, _raw_stream, check, PagedCache)
        _fast = f
    return _fast


def _gpu(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _elsewhere(fn, index, stream, *args):
    """fn(..., stream handle) for a stream or device other than the current one. The stream
    is current while outputs are allocated, so that their memory belongs to it."""
    if isinstance(stream, torch.cuda.Stream) and stream.device.index != index:
        raise ValueError(f"stream must be on GPU {index}, the tensors' own; it is on {stream.device}")
    with torch.cuda.device(index):
        if stream is None:
            return fn(*args, _raw_stream(index))
        s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(int(stream), device=index)
        with torch.cuda.stream(s):
            return fn(*args, s.cuda_stream)


def rope_table(length: int, rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """The rotation table of :func:`qk_norm_rope`: [length, rotary_dim] fp32, row p holding
    cos(p * theta^(-2i / rotary_dim)) for i < rotary_dim / 2, then the sines. The angles
    are taken in 64 bits: in 32 the far positions would lose their fraction of a turn."""
    if length <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("length must be positive, rotary_dim positive and even")
    if not 0.0 < float(theta) < float("inf"):
        raise ValueError("theta must be positive and finite")
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
    fn = (_fast or _load()).qk_norm_rope
    if stream is None:
        r = fn(Q, K, rope_table, positions, q_weight, k_weight, eps, interleaved, V, cache, slots, Q_out, K_out, None)
        if r is not NotImplemented:
            return r
    return _elsewhere(fn, _gpu(Q, "Q"), stream, Q, K, rope_table, positions, q_weight, k_weight, eps, interleaved,
                      V, cache, slots, Q_out, K_out)


def paged_attention(Q, cache: PagedCache, page_table, seq_lens, scale: float | None = None,
                    window: int = 0, lse=None, key_weights=None, accumulate: bool = False, O=None,
                    stream=None):
    """Attention of one new token per sequence, Q [B, heads, D] (fp16 or bf16), over the
    first seq_lens[b] cached tokens of page_table[b] (with `window`, the last `window` of
    them; heads a multiple of the cache's). Returns O [B, heads, D].

    lse [B, heads] fp32, if given, gets the log-sum-exp of the scaled scores. key_weights
    [pages, kv_heads, page_size] fp32, if given, gets the softmax weight of every attended
    key, summed over its query heads (added with accumulate=True); no page may then be in
    two sequences; and it takes 4 bytes of scratch per sequence, head and token that
    page_table can name (page_table[:, :n] will do). scale defaults to 1/sqrt(D). An empty
    sequence gives zeros and -inf; an infinite value in V gives NaN in its column."""
    fn = (_fast or _load()).paged_attention
    if stream is None:
        r = fn(Q, cache, page_table, seq_lens, scale, window, lse, key_weights, accumulate, O, None)
        if r is not NotImplemented:
            return r
    return _elsewhere(fn, _gpu(Q, "Q"), stream, Q, cache, page_table, seq_lens, scale, window, lse,
                      key_weights, accumulate, O)


def evict_cache(cache: PagedCache, key_weights, page_table, seq_lens, dst_table, budget: int,
                recent: int = 0, stream=None):
    """Shorten every sequence to `budget` tokens: the last `recent` ones and, per kv head,
    those of largest key_weights [pages, kv_heads, page_size] before them (ties: the lowest
    index). Their K, V and weights are copied, in order, to the fresh pages of dst_table
    [B, >= ceil(budget / page_size)], none of which may still be in use. Returns (kept
    [B, kv_heads, budget] int32 -- indices, -1 behind them -- and the new lengths [B])."""
    fn = (_fast or _load()).evict_cache
    if not isinstance(cache, PagedCache):
        raise TypeError("cache must be a PagedCache")
    if stream is None:
        r = fn(cache, key_weights, page_table, seq_lens, dst_table, budget, recent, None)
        if r is not NotImplemented:
            return r
    return _elsewhere(fn, cache.index, stream, cache, key_weights, page_table, seq_lens, dst_table, budget,
                      recent)
