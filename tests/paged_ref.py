"""Plain 64-bit statements of the paged-cache operators and the error bounds that the
tests hold the kernels to.

Bounds. Outputs are rounded once: half a step, eps/2 relative (plus half the type's
subnormal step). Before that everything is fp32, whose unit is u = 2^-24:

* rotation: y = x * inv * w with inv = 1/sqrt(mean + eps) from a sum of D squares -- at most
  (log2 D + 8) roundings, rsqrt's 2 ulp among them -- then two products and a sum of them:
  16 u per unit of |y_i cos| + |y_j sin| covers it for D <= 256.
* attention: a score is a sum of D products, added 16 at a time into an fp32 accumulator
  (at most one unit each, 2u with truncation): error e_s <= (D/16 + 16) 2u * sum|q k| * scale,
  and its product with scale * log2(e) two more roundings. exp2 is good to 4u, its argument
  rounds |s| u. A weight p is passed as two 16-bit halves (bf16: 2^-17 relative; fp16:
  2^-25 of the largest weight at worst). Sums over n keys run over at most n/64 + 64
  sequential steps. All of it enters numerator and denominator, so twice.
"""
import math

import torch

U = 2.0 ** -24
DENORM = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float8_e4m3fn: 2.0 ** -10}


def half_step(x, dtype):
    return x.abs() * (torch.finfo(dtype).eps / 2) + DENORM[dtype]


def norm_rope(x, weight, table, positions, interleaved, eps):
    """(y, magnitude): y rounded nowhere, magnitude |y_i cos| + |y_j sin| per element."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    R = table.shape[1]
    half = R // 2
    row = table.double()[positions.long()][:, None, :]
    c, s = row[..., :half], row[..., half:]
    y, mag = x.clone(), x.abs().clone()
    i = slice(0, R, 2) if interleaved else slice(0, half)
    j = slice(1, R, 2) if interleaved else slice(half, R)
    a, b = x[..., i], x[..., j]
    y[..., i], y[..., j] = a * c - b * s, b * c + a * s
    mag[..., i], mag[..., j] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


def rows(cache, layout, page_table, n, ps):
    """[n, heads, D] of the first n tokens of one sequence, as float64."""
    t = torch.arange(n, device=cache.device)
    page, off = page_table.long()[t // ps], t % ps
    raw = cache.view(torch.uint8) if cache.element_size() == 1 else cache
    got = raw[page, off] if layout == "bshd" else raw[page, :, off]
    return (got.contiguous().view(cache.dtype) if cache.element_size() == 1 else got).double()


def attention(q, k, v, scale, first):
    """One sequence: q [H, D], k, v [n, Hkv, D] float64, keys from `first` on. Returns (o, lse,
    weights [n - first, Hkv], bounds of the three before the output's rounding)."""
    H, D = q.shape
    k, v = k[first:], v[first:]
    n, Hkv = k.shape[0], k.shape[1]
    G = H // Hkv
    q = q.double().view(Hkv, G, D)
    s = torch.einsum("hgd,thd->hgt", q, k) * scale
    mag = torch.einsum("hgd,thd->hgt", q.abs(), k.abs()) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    o = torch.einsum("hgt,thd->hgd", p, v)
    e_s = (D / 16 + 16) * 2 * U * mag.amax(-1) + 8 * U * s.abs().amax(-1) + 4 * U
    steps = (n / 64 + 64) * 2 * U
    size = torch.einsum("hgt,thd->hgd", p, v.abs())
    # fp16 halves: 2^-25 of the largest weight for each key.
    top = p.amax(-1, keepdim=True)
    tail = 2.0 ** -25 * top * v.abs().sum(0)[:, None, :]
    b_o = size * (2 * e_s + 2 * steps + 2.0 ** -17)[..., None] + tail
    b_lse = e_s + steps + 4 * U * lse.abs()
    w = p.sum(1).T  # [n, Hkv]
    b_w = (p * (2 * e_s + 2 * steps + 4 * U * lse.abs() + G * U)[..., None]).sum(1).T + 2.0 ** -120
    return o.reshape(H, D), lse.reshape(H), w, b_o.reshape(H, D), b_lse.reshape(H), b_w


def evict(weights, n, budget, recent):
    """weights [n] (python floats of one head) -> kept indices."""
    if n <= budget:
        return list(range(n))
    m = n - recent
    order = sorted(range(m), key=lambda t: (0 if math.isnan(weights[t]) else 1, 0.0 if math.isnan(weights[t]) else -weights[t], t))
    return sorted(order[:budget - recent]) + list(range(m, n))
