"""Paged-cache operators without a GPU: refusals come before any device work, empty calls
are no-ops, and the tests' own plain statements agree with simpler ones."""
import ctypes
import random

import pytest
import torch

from clove_compute_b200._lib import PagedCacheStruct
from tests import paged_ref as ref

A = 4096  # an aligned address that a refused call never follows


def _cache(**kw):
    d = dict(K=A, V=A, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128, page_stride=4096,
             token_stride=256, head_stride=128, dtype=0, k_scale=1.0, v_scale=1.0)
    d.update(kw)
    return PagedCacheStruct(**d)


BAD_CACHES = [
    (dict(K=None), 1), (dict(V=None), 1), (dict(num_pages=0), 1), (dict(num_kv_heads=0), 1),
    (dict(page_size=0), 2), (dict(page_size=24), 2), (dict(num_pages=1 << 28), 2),
    (dict(head_dim=96), 2), (dict(dtype=3), 1), (dict(dtype=1), 2), (dict(K=A + 8), 2),
    (dict(token_stride=252), 2), (dict(page_stride=-4096), 1), (dict(k_scale=0.0), 1),
    (dict(dtype=2, v_scale=float("nan")), 1), (dict(k_scale=0.5), 1),
]


def _rope(lib, c=None, **kw):
    d = dict(Q=A, K=A, V=None, qs=256, ks=256, vs=0, qw=None, kw=None, eps=1e-6, table=A, tl=64, R=128,
             il=0, pos=A, cache=None, slots=None, Qo=A, qos=256, Ko=A, kos=256, T=2, H=2, Hkv=2, D=128,
             dtype=0, stream=None)
    d.update(kw)
    if c is not None:
        d["cache"] = ctypes.byref(c)
    return lib.clove_qk_norm_rope(*d.values())


def _attn(lib, c, **kw):
    d = dict(Q=A, qs=256, cache=ctypes.byref(c) if c is not None else None, pt=A, ts=4, mp=4, sl=A, O=A,
             os=256, lse=None, kw=None, acc=0, B=2, H=2, scale=0.1, window=0, dtype=0, stream=None)
    d.update(kw)
    return lib.clove_paged_attention(*d.values())


def _evict(lib, c, **kw):
    d = dict(cache=ctypes.byref(c) if c is not None else None, w=A, pt=A, ts=4, mp=4, sl=A, dt=A, ds=4, dp=4,
             kept=A, nl=A, B=2, budget=32, recent=4, stream=None)
    d.update(kw)
    return lib.clove_evict_cache(*d.values())


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_cache_descriptions_refused(clove_lib, bad, code):
    lib = clove_lib.lib()
    assert _attn(lib, _cache(**bad)) == code
    assert _rope(lib, _cache(**bad), V=A, slots=A, vs=256) == code
    if bad.get("dtype") != 1:  # eviction takes any type
        assert _evict(lib, _cache(**bad)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), 1), (dict(H=0), 1), (dict(Hkv=0), 1), (dict(dtype=2), 1), (dict(D=96), 2),
    (dict(R=0), 2), (dict(R=24), 2), (dict(R=144), 2), (dict(tl=0), 1), (dict(qw=A), 1), (dict(kw=A), 1),
    (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(V=A), 1), (dict(slots=A), 1), (dict(Q=None), 1),
    (dict(Ko=None), 1), (dict(pos=None), 1), (dict(table=None), 1), (dict(Q=A + 2), 2), (dict(table=A + 4), 2),
    (dict(pos=A + 2), 1), (dict(qs=255), 1), (dict(qs=260), 2), (dict(kos=8), 1),
])
def test_norm_rope_refusals(clove_lib, kw, code):
    assert _rope(clove_lib.lib(), **kw) == code


def test_norm_rope_cache_refusals(clove_lib):
    lib = clove_lib.lib()
    c = _cache()
    assert _rope(lib, c) == 1                                        # no V, no slots
    assert _rope(lib, c, V=A, slots=A, vs=256, Hkv=4, ks=512) == 1   # heads differ
    assert _rope(lib, c, V=A, slots=A, vs=8) == 1                    # V's rows overlap
    assert _rope(lib, T=0, Q=None, K=None) == 0                      # nothing to do


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), 1), (dict(H=0), 1), (dict(H=3), 1), (dict(dtype=2), 1), (dict(scale=0.0), 1),
    (dict(scale=float("inf")), 1), (dict(window=-1), 1), (dict(mp=-1), 1), (dict(Q=None), 1), (dict(O=None), 1),
    (dict(sl=None), 1), (dict(pt=None), 1), (dict(Q=A + 4), 2), (dict(qs=260), 2), (dict(qs=128), 1),
    (dict(os=128), 1), (dict(ts=3), 1), (dict(mp=1 << 28, ts=1 << 28), 2), (dict(lse=A + 1), 1),
])
def test_attention_refusals(clove_lib, kw, code):
    assert _attn(clove_lib.lib(), _cache(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), 1), (dict(budget=0), 1), (dict(recent=-1), 1), (dict(recent=33), 1), (dict(dp=1), 1),
    (dict(mp=-1), 1), (dict(w=None), 1), (dict(dt=None), 1), (dict(kept=None), 1), (dict(nl=None), 1),
    (dict(sl=None), 1), (dict(ts=3), 1), (dict(ds=3), 1), (dict(kept=A + 2), 1), (dict(budget=(1 << 30) + 1, dp=1 << 27, ds=1 << 27), 2), (dict(mp=1 << 28, ts=1 << 28), 2),
])
def test_evict_refusals(clove_lib, kw, code):
    assert _evict(clove_lib.lib(), _cache(), **kw) == code


def test_null_cache_and_empty_batches(clove_lib):
    lib = clove_lib.lib()
    assert _attn(lib, None) == 1 and _evict(lib, None) == 1
    assert _attn(lib, _cache(), B=0, Q=None, O=None) == 0
    assert _evict(lib, _cache(), B=0, kept=None) == 0


def test_python_refusals(clove_lib):
    x = torch.zeros(2, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        clove_lib.PagedCache(x, x)  # not on a GPU
    with pytest.raises(TypeError):
        clove_lib.PagedCache(x.float(), x.float())
    q = torch.zeros(2, 2, 64)
    with pytest.raises(TypeError):
        clove_lib.qk_norm_rope(q, q, None, None)
    with pytest.raises(ValueError):
        clove_lib.paged_attention(q.half(), None, None, None)
    with pytest.raises(ValueError):
        clove_lib.rope_table(0, 64)
    with pytest.raises(ValueError):
        clove_lib.rope_table(4, 7)


def test_rope_table_far_positions(clove_lib):
    """Row p is within half a step of cos and sin of the exact angle, far out as well."""
    import math
    from fractions import Fraction
    t = clove_lib.rope_table(200001, 64, device="cpu")
    for p in (0, 1, 4095, 131071, 200000):
        for i in (0, 5, 31):
            a = math.fmod(float(Fraction(p) * Fraction(10000.0 ** (-2 * i / 64))), 2 * math.pi)
            # 64-bit angles: p * 2^-53 absolute, far below fp32's half step of 2^-25.
            assert abs(float(t[p, i]) - math.cos(a)) <= 2.0 ** -25 + 1e-10
            assert abs(float(t[p, 32 + i]) - math.sin(a)) <= 2.0 ** -25 + 1e-10


def test_plain_statements_agree():
    """The 64-bit reference against loops."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((4, 64), (9, 2, 64), (9, 2, 64)))
    o, lse, w, *_ = ref.attention(q, k, v, 0.125, 2)
    for h in range(4):
        s = [float(q[h] @ k[t, h // 2]) * 0.125 for t in range(2, 9)]
        e = torch.tensor(s, dtype=torch.float64).exp()
        assert torch.allclose(lse[h], e.sum().log())
        assert torch.allclose(o[h], (e[:, None] * v[2:, h // 2]).sum(0) / e.sum())
    x = torch.randn(3, 2, 64, generator=g, dtype=torch.float64)
    a = torch.rand(5, 16, generator=g, dtype=torch.float64)
    table = torch.cat([a.cos(), a.sin()], 1)
    y, _ = ref.norm_rope(x, None, table, torch.tensor([0, 4, 2]), True, 0.0)
    assert torch.allclose(y[1, 1, 6], x[1, 1, 6] * a[4, 3].cos() - x[1, 1, 7] * a[4, 3].sin())
    assert torch.equal(y[..., 32:], x[..., 32:])
    r = random.Random(1)
    w = [r.choice([0.0, 1.0, 2.0, float("nan")]) for _ in range(40)]
    got = ref.evict(w, 40, 10, 3)
    assert len(got) == 10 and got == sorted(got) and got[-3:] == [37, 38, 39]


TINY, HUGE = 1e-39, 3e38


@pytest.mark.parametrize("kw,scale", [
    (dict(dtype=2, k_scale=1e30), 1e30), (dict(dtype=2, k_scale=HUGE), 3.0), (dict(), HUGE),
    (dict(dtype=2, k_scale=1e-25), 1e-25), (dict(), 1e-45),
])
def test_attention_scales_out_of_range(clove_lib, kw, scale):
    """scale * k_scale * log2(e) must be a finite fp32 number that has not lost its digits:
    scores would be NaN, or all zero."""
    assert _attn(clove_lib.lib(), _cache(**kw), scale=scale) == 1


@pytest.mark.parametrize("kw", [dict(dtype=2, k_scale=TINY), dict(dtype=2, v_scale=TINY)])
def test_cache_scales_without_an_inverse(clove_lib, kw):
    """Scales whose inverse is no fp32 number: rows are stored times the inverse."""
    assert _rope(clove_lib.lib(), _cache(**kw), V=A, slots=A, vs=256) == 1
