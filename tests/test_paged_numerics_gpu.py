"""Paged attention where the products' 16-bit operands could lose what fp32 keeps, against
plain 64-bit statements (tests/paged_ref.py)."""
import math

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _bound(q, k, v, scale, products):
    """(o, lse, bounds of both before o's rounding) as paged_ref.attention, but with the
    weights' own rounding: two halves leave 2^-17 (bf16) or 2^-23 (fp16) of each, and fp16
    halves of weights that are passed 2^15 times as large end at 2^-25, which is 2^-40 of a
    largest weight."""
    H, D = q.shape
    n, Hkv = k.shape[0], k.shape[1]
    o, lse, _, _, b_lse, _ = ref.attention(q, k, v, scale, 0)
    qg = q.double().view(Hkv, H // Hkv, D)
    s = torch.einsum("hgd,thd->hgt", qg, k) * scale
    mag = torch.einsum("hgd,thd->hgt", qg.abs(), k.abs()) * scale
    p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
    e_s = (D / 16 + 16) * 2 * ref.U * mag.amax(-1) + 8 * ref.U * s.abs().amax(-1) + 4 * ref.U
    steps = (n / 64 + 64) * 2 * ref.U
    size = torch.einsum("hgt,thd->hgd", p, v.abs())
    rel, floor = (2.0 ** -17, 0.0) if products == BF16 else (2.0 ** -23, 2.0 ** -40)
    b = size * (2 * e_s + 2 * steps + rel)[..., None] + floor * p.amax(-1, keepdim=True) * v.abs().sum(0)[:, None, :]
    return o, lse, b.reshape(H, D), b_lse


def _cache_and_table(cc, K, V, lens, k_scale=1.0, v_scale=1.0):
    """Contiguous rows [sum of lens, Hkv, D] (each a multiple of 16) as pages of 16."""
    shape = (K.shape[0] // 16, 16) + tuple(K.shape[1:])
    cache = cc.PagedCache(K.view(shape), V.view(shape), k_scale=k_scale, v_scale=v_scale)
    table = torch.zeros((len(lens), max(lens) // 16), dtype=torch.int32, device="cuda")
    first = 0
    for i, n in enumerate(lens):
        table[i, :n // 16] = torch.arange(first // 16, (first + n) // 16, device="cuda")
        first += n
    return cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype,cache_dtype,D,G", [
    (F16, F16, 128, 4), (F16, F16, 64, 1), (F16, F16, 256, 2), (F16, F16, 128, 16),
    (F16, E4M3, 128, 4), (BF16, E4M3, 128, 8), (BF16, E4M3, 64, 3), (BF16, BF16, 128, 4),
])
@pytest.mark.parametrize("gap", [12.0, 15.5, 17.0, 18.5, 22.0])
def test_attention_with_a_dominant_key(clove_lib, cuda, dtype, cache_dtype, D, G, gap):
    """One key of each sequence has a score `gap` nats above all the others and a value of
    zero: the output is the others' alone, each of weight e^-gap (2^-17 to 2^-32). Enough
    sequences that a warp has thousands of keys beside it; at the start, in the middle and
    at the end."""
    g = torch.Generator(device="cuda").manual_seed(int(gap * 10) + D + G)
    B, Hkv, n = 40, 8, 2048
    scale = D ** -0.5
    Q = (0.1 * torch.randn((B, Hkv * G, D), device="cuda", generator=g)).to(dtype)
    Q[..., 0] = 8.0
    K = 0.1 * torch.randn((B * n, Hkv, D), device="cuda", generator=g)
    V = 1.0 + 0.25 * torch.randn((B * n, Hkv, D), device="cuda", generator=g)
    K[..., 0] = 0.0
    at = torch.tensor([b * n + (0, n // 2, n - 1)[b % 3] for b in range(B)], device="cuda")
    K[at, :, 0] = gap / (8.0 * scale)
    V[at] = 0.0
    K, V = K.to(cache_dtype), V.to(cache_dtype)
    cache, table, lens = _cache_and_table(clove_lib, K, V, [n] * B)
    lse = torch.empty((B, Hkv * G), device="cuda")
    O = clove_lib.paged_attention(Q, cache, table, lens, lse=lse)
    torch.cuda.synchronize()
    assert clove_lib.device_error() == 0
    products = BF16 if cache_dtype == BF16 else F16
    for b in range(B):
        k, v = (ref.rows(c, "bshd", table[b], n, 16) for c in (cache.K, cache.V))
        o, l, b_o, b_l = _bound(Q[b], k, v, scale, products)
        err, tol = (O[b].double() - o).abs(), b_o + ref.half_step(o.abs() + b_o, dtype)
        assert torch.all(err <= tol), (b, float((err / tol).max()), float((err / o.abs().clamp(min=1e-30)).max()))
        assert torch.all((lse[b].double() - l).abs() <= b_l)


@pytest.mark.parametrize("D,G", [(64, 3), (128, 4), (128, 16), (256, 2)])
@pytest.mark.parametrize("small", [2.0 ** -12, 2.0 ** -17, 2.0 ** -20, 2.0 ** -24])
def test_attention_bf16_queries_of_wide_range(clove_lib, cuda, D, G, small):
    """bf16 query rows over an e4m3 cache, one element `1 / small` times as large as the
    others, on which every key is zero: the scores are made of the small elements alone."""
    g = torch.Generator(device="cuda").manual_seed(D + G)
    lens, Hkv = [512, 96, 16], 2
    n = sum(lens)
    for top in (1.0, 2.0 ** -100, 2.0 ** 90):
        Q = (torch.randn((3, Hkv * G, D), device="cuda", generator=g) * small).clamp(-3 * small, 3 * small)
        Q[..., 5] = 1.0
        Q = (Q * top).to(BF16)
        K = torch.randn((n, Hkv, D), device="cuda", generator=g) * 2
        K[..., 5] = 0.0
        V = torch.randn((n, Hkv, D), device="cuda", generator=g)
        scale = D ** -0.5 / (small * top)
        cache, table, sl = _cache_and_table(clove_lib, K.to(E4M3), V.to(E4M3), lens)
        lse = torch.empty((3, Hkv * G), device="cuda")
        O = clove_lib.paged_attention(Q, cache, table, sl, scale=scale, lse=lse)
        torch.cuda.synchronize()
        assert clove_lib.device_error() == 0
        for i, m in enumerate(lens):
            k, v = (ref.rows(c, "bshd", table[i], m, 16) for c in (cache.K, cache.V))
            o, l, b_o, b_l = _bound(Q[i], k, v, scale, F16)
            err, tol = (O[i].double() - o).abs(), b_o + ref.half_step(o.abs() + b_o, BF16)
            assert torch.all(err <= tol), (top, i, float((err / tol).max()))
            assert torch.all((lse[i].double() - l).abs() <= b_l), (top, i, float(((lse[i].double() - l).abs() / b_l).max()))


@pytest.mark.parametrize("B,Hkv,cache_dtype", [(70001, 2, F16), (66000, 1, E4M3)])
def test_attention_and_weights_of_huge_batches(clove_lib, cuda, B, Hkv, cache_dtype):
    """More sequences than a grid dimension has blocks, of no, one or two keys: exact where the
    answer is one value, half of two equal ones, and the weights of every key."""
    D, G = 64, 2
    g = torch.Generator(device="cuda").manual_seed(B)
    V = torch.randint(-8, 9, (B, 2, Hkv, D), device="cuda", generator=g).to(cache_dtype)
    cache = clove_lib.PagedCache(torch.zeros_like(V), V)
    table = torch.randperm(B, device="cuda", generator=g).to(torch.int32)[:, None]
    lens = (torch.arange(B, device="cuda") % 3).to(torch.int32)
    w = torch.full((B, Hkv, 2), 7.0, device="cuda")
    Q = torch.randn((B, Hkv * G, D), device="cuda", generator=g).to(F16)
    O = clove_lib.paged_attention(Q, cache, table, lens, key_weights=w)
    torch.cuda.synchronize()
    assert clove_lib.device_error() == 0
    v = V.float()[table[:, 0].long()]
    want = torch.where((lens == 0)[:, None, None], 0.0, torch.where((lens == 1)[:, None, None], v[:, 0], v.mean(1)))
    assert torch.equal(O.float(), want.repeat_interleave(G, 1))
    seen = w[table[:, 0].long()]
    n = lens[:, None].expand(-1, Hkv)
    for t in (0, 1):
        got = seen[:, :, t]
        assert torch.all(got[n <= t] == 7.0) and torch.all((got[n > t] - G / n[n > t]).abs() <= 2.0 ** -21)
