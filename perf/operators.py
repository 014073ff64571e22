"""Workloads of the paged-cache operators: what they compute, in plain torch, and the
calls that a decode loop makes of them.

Three operators share one paged key-value cache (K and V pages of ``page_size`` tokens,
any order of pages, one page table row per sequence):

* ``rope``  -- root-mean-square norm of every query and key head, position rotation, and
  the new keys and values written to their cache slots, in one pass;
* ``attn``  -- attention of one new token per sequence over its cached keys (ragged
  lengths, grouped heads, an optional sliding window), with the log-sum-exp and, where
  asked for, the weight that every cached key received;
* ``evict`` -- the keys of highest accumulated weight (and the most recent ones) copied
  to fresh pages, in order, per key head.

``own`` False computes the plain forms; True calls the package.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"fp16": 2, "bf16": 2, "e4m3": 1}


def listed():
    base = {"D": 128, "layout": "bshd", "ps": 16}
    rope = {**base, "op": "rope", "R": 128, "norm": True, "interleaved": False, "append": True}
    attn = {**base, "op": "attn", "window": 0, "weights": False}
    evict = {**base, "op": "evict", "dtype": "fp16", "cache": "fp16"}
    return [
        # One new token of one sequence, 32 full heads: latency alone.
        {**rope, "name": "rope_one_token", "T": 1, "H": 32, "Hkv": 32, "dtype": "fp16", "cache": "fp16"},
        # A decode step of 64 sequences, grouped heads, interleaved pairs, 8-bit cache.
        {**rope, "name": "rope_batch64_e4m3", "T": 64, "H": 32, "Hkv": 8, "dtype": "bf16", "cache": "e4m3", "interleaved": True},
        # A prefill chunk of odd length, grouped heads: bandwidth.
        {**rope, "name": "rope_prefill_8191", "T": 8191, "H": 32, "Hkv": 8, "dtype": "fp16", "cache": "fp16", "ps": 64},
        # One sequence of 4096 keys, 32 full heads: the smallest decode call.
        {**attn, "name": "attn_1x4096", "B": 1, "N": 4096, "ragged": False, "H": 32, "Hkv": 32, "dtype": "fp16", "cache": "fp16"},
        # A batch of short, ragged chats.
        {**attn, "name": "attn_32x511_ragged", "B": 32, "N": 511, "ragged": True, "H": 32, "Hkv": 8, "dtype": "bf16", "cache": "bf16"},
        # A full serving batch, lengths from one token to 16384.
        {**attn, "name": "attn_64x16384_ragged", "B": 64, "N": 16384, "ragged": True, "H": 32, "Hkv": 8, "dtype": "fp16", "cache": "fp16"},
        # Two long documents, 8-bit cache, eight query heads to a key head.
        {**attn, "name": "attn_2x131071_e4m3", "B": 2, "N": 131071, "ragged": False, "H": 64, "Hkv": 8, "dtype": "bf16", "cache": "e4m3", "ps": 64},
        # A step that also records what weight each key received, for eviction.
        {**attn, "name": "attn_8x20000_weights", "B": 8, "N": 20000, "ragged": True, "H": 32, "Hkv": 8, "dtype": "fp16", "cache": "fp16", "ps": 64, "layout": "bhsd", "weights": True},
        # One sequence cut from 4096 keys to 1024.
        {**evict, "name": "evict_1x4096", "B": 1, "N": 4096, "ragged": False, "Hkv": 8, "budget": 1024, "recent": 128},
        # A serving batch cut to a quarter, ragged: some sequences fit already.
        {**evict, "name": "evict_8x32768", "B": 8, "N": 32768, "ragged": True, "Hkv": 8, "budget": 8192, "recent": 1000, "ps": 64},
        # One long document in an 8-bit cache.
        {**evict, "name": "evict_1x131071_e4m3", "B": 1, "N": 131071, "ragged": False, "Hkv": 8, "budget": 16001, "recent": 512, "cache": "e4m3", "ps": 32, "layout": "bhsd"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "evict"])
    dtype = rng.choice(["fp16", "bf16"])
    case = {"op": op, "dtype": dtype, "cache": rng.choice([dtype, dtype, "e4m3"]), "D": rng.choice([64, 128, 128, 256]),
            "layout": rng.choice(["bshd", "bhsd"]), "ps": rng.choice([8, 16, 32, 64, 128]), "Hkv": rng.choice([1, 2, 4, 8, 8, 32])}
    width = case["Hkv"] * case["D"]
    if op == "rope":
        case["H"] = case["Hkv"] * rng.choice([1, 2, 4, 5, 8])
        most = 8191 * 48 * 128 // ((case["H"] + 2 * case["Hkv"]) * case["D"])
        case |= {"T": _log_int(rng, 1, min(16384, most)), "R": rng.choice([case["D"], case["D"], case["D"] // 2]),
                 "norm": rng.random() < 0.8, "interleaved": rng.random() < 0.4, "append": rng.random() < 0.8}
        if not case["append"]:
            case["cache"] = dtype
        return case
    if op == "attn":
        case["H"] = case["Hkv"] * rng.choice([1, 2, 3, 4, 7, 8, 8, 16] if case["Hkv"] <= 8 else [1, 2])
        case["B"] = _log_int(rng, 1, 128)
        case["N"] = _log_int(rng, 1, max(1, min(131072, (1 << 28) // (width * case["B"]))))
        case |= {"ragged": rng.random() < 0.7, "window": _log_int(rng, 1, case["N"]) if rng.random() < 0.2 else 0, "weights": rng.random() < 0.25}
        return case
    case["B"] = _log_int(rng, 1, 32)
    case["N"] = _log_int(rng, 16, max(16, min(131072, (1 << 28) // (width * case["B"]))))
    case["budget"] = _log_int(rng, 1, case["N"])
    case |= {"ragged": rng.random() < 0.7, "recent": rng.randrange(0, case["budget"] + 1)}
    return case


def _lengths(case, seed):
    """The sequences' lengths, as a list: equal, or spread over their logarithm with an empty one among many.
    The seed gives their order alone, so that every seed is the same work."""
    if not case["ragged"]:
        return [case["N"]] * case["B"]
    low, high = math.log(max(1, case["N"] // 64)), math.log(case["N"])
    n = np.exp(np.linspace(high, low, case["B"])).round().astype(int).clip(1, case["N"])
    if case["B"] >= 16:
        n[-1] = 0
    n = np.random.default_rng(seed).permutation(n)
    return n.tolist()


def _randn(gen, shape, dtype, scale=1.0):
    """Normal values in `dtype`, drawn in slices so that no large buffer of wider values is needed."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        m = min(step, flat.numel() - i)
        x = torch.randn(m, device="cuda", generator=gen, dtype=torch.float16 if dtype == torch.float16 else torch.float32)
        flat[i:i + m] = (x * scale).to(dtype)
    return out


def _cache(case, pages, gen, fill=True):
    ps, h, d = case["ps"], case["Hkv"], case["D"]
    shape = (pages, ps, h, d) if case["layout"] == "bshd" else (pages, h, ps, d)
    dtype = TYPES[case["cache"]]
    if not fill:
        return torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda")
    return _randn(gen, shape, dtype, 2.0 if case["cache"] == "e4m3" else 1.0), _randn(gen, shape, dtype, 2.0 if case["cache"] == "e4m3" else 1.0)


def _table(need, width, order):
    """A page table [B, width] int32: sequence b's pages are the next need[b] of `order`; zeros behind them."""
    need = torch.tensor(need, dtype=torch.int64)
    first = torch.cumsum(need, 0) - need
    at = first[:, None] + torch.arange(width)[None, :]
    inside = torch.arange(width)[None, :] < need[:, None]
    return torch.where(inside, order[at.clamp(max=order.numel() - 1)], torch.zeros((), dtype=torch.int64)).to(torch.int32)


def _rope_table(length, rotary, theta=10000.0):
    inv = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    a = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return torch.cat([a.cos(), a.sin()], 1).to(torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    s = dict(case)
    scale = 0.5 if case["cache"] == "e4m3" else 1.0
    s["k_scale"], s["v_scale"] = scale, scale
    ps, h, d = case["ps"], case["Hkv"], case["D"]
    dtype = TYPES[case["dtype"]]
    if case["op"] == "rope":
        t, heads = case["T"], case["H"]
        qkv = _randn(gen, (t, (heads + 2 * h) * d), dtype, 1.5)  # the fused projection's output
        s["q"] = qkv[:, :heads * d].view(t, heads, d)
        s["k"] = qkv[:, heads * d:(heads + h) * d].view(t, h, d)
        s["v"] = qkv[:, (heads + h) * d:].view(t, h, d)
        s["qw"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype) if case["norm"] else None
        s["kw"] = (1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(dtype) if case["norm"] else None
        s["table"] = _rope_table(32768, case["R"])
        first = int(torch.randint(0, 32768 - t, (), generator=cpu))
        s["pos"] = torch.arange(first, first + t, dtype=torch.int32, device="cuda") if t > 128 else torch.randint(0, 32768, (t,), generator=cpu).to(torch.int32).cuda()
        if case["append"]:
            pages = -(-t // ps) + 2
            s["kc"], s["vc"] = _cache(case, pages, gen, fill=False)
            s["slots"] = torch.randperm(pages * ps, generator=cpu)[:t].to(torch.int32).cuda() if t <= 128 else (torch.randperm(pages, generator=cpu)[:, None] * ps + torch.arange(ps)[None, :]).reshape(-1)[:t].to(torch.int32).cuda()
    else:
        lens = _lengths(case, seed)
        need = [-(-n // ps) for n in lens]
        width = -(-case["N"] // ps)
        keep = [min(n, case.get("budget", 0)) for n in lens]
        need_new = [-(-n // ps) for n in keep] if case["op"] == "evict" else [0]
        pages = sum(need) + sum(need_new) + 1
        order = torch.randperm(pages, generator=cpu)
        s["kc"], s["vc"] = _cache(case, pages, gen)
        s["pages"] = _table(need, width, order).cuda()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if case["op"] == "attn":
            s["q"] = _randn(gen, (case["B"], case["H"], d), dtype, 2.0)
            s["lse"] = torch.zeros(case["B"], case["H"], device="cuda")
            if case["weights"]:
                s["w"] = torch.zeros(pages, h, ps, device="cuda")
        else:
            # Accumulated weights: heavy-tailed, many of them equal zero.
            s["w"] = torch.rand(pages, h, ps, device="cuda", generator=gen).sub_(0.1).clamp_(min=0).pow_(6)
            s["dst"] = _table(need_new, -(-case["budget"] // ps), order[sum(need):]).cuda()
    if own and "kc" in s:
        from clove_compute_b200 import PagedCache
        s["handle"] = PagedCache(s["kc"], s["vc"], layout=case["layout"], k_scale=scale, v_scale=scale)
    return s


def _rows(c, s):
    """The cache as [pages, page_size, heads, D], whatever its layout."""
    return c if s["layout"] == "bshd" else c.transpose(1, 2)


def _norm_rope(x, weight, s):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = s["R"] // 2
    cs = s["table"][s["pos"].long()][:, None, :]
    c, sn = cs[..., :half], cs[..., half:]
    y = x.clone()
    if s["interleaved"]:
        a, b = x[..., 0:s["R"]:2], x[..., 1:s["R"]:2]
        y[..., 0:s["R"]:2], y[..., 1:s["R"]:2] = a * c - b * sn, b * c + a * sn
    else:
        a, b = x[..., :half], x[..., half:s["R"]]
        y[..., :half], y[..., half:s["R"]] = a * c - b * sn, b * c + a * sn
    return y


def _store(c, slots, x, scale, s):
    x = (x.float() / scale)
    x = x.clamp(-448, 448) if c.dtype == torch.float8_e4m3fn else x
    slots = slots.long()
    rows = _rows(c, s)
    # 8-bit types have no scatter: their bytes are moved.
    view = rows.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else rows
    new = x.to(c.dtype)
    view[slots // s["ps"], slots % s["ps"]] = new.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else new


def _plain_rope(s):
    q = _norm_rope(s["q"], s["qw"], s)
    k = _norm_rope(s["k"], s["kw"], s)
    if not s["append"]:
        return {"q": q.to(s["q"].dtype), "k": k.to(s["k"].dtype)}
    _store(s["kc"], s["slots"], k, s["k_scale"], s)
    _store(s["vc"], s["slots"], s["v"], s["v_scale"], s)
    return {"q": q.to(s["q"].dtype), "kc": s["kc"], "vc": s["vc"]}


def _gathered(c, s):
    """[B, N, heads, D] of every sequence's pages, in the cache's type."""
    rows = _rows(c, s)
    b, width = s["pages"].shape
    got = rows.view(torch.uint8)[s["pages"].long()].view(c.dtype) if c.dtype == torch.float8_e4m3fn else rows[s["pages"].long()]
    return got.reshape(b, width * s["ps"], s["Hkv"], s["D"])


def _plain_attn(s):
    b, heads, d = s["q"].shape
    group = heads // s["Hkv"]
    t = torch.arange(s["pages"].shape[1] * s["ps"], device="cuda")
    live = t[None, :] < s["lens"][:, None]
    if s["window"]:
        live = live & (t[None, :] >= s["lens"][:, None] - s["window"])
    q = s["q"].float().view(b, s["Hkv"], group, d) * (s["k_scale"] / math.sqrt(d))
    score = torch.matmul(q, _gathered(s["kc"], s).float().permute(0, 2, 3, 1))  # [B, Hkv, group, N]
    score = score.masked_fill(~live[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _gathered(s["vc"], s).float().permute(0, 2, 1, 3)) * s["v_scale"] / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf).view(b, heads)
    got = {"o": out.view(b, heads, d).to(s["q"].dtype), "lse": lse}
    if s["weights"]:
        w = (p / total.clamp(min=1e-30)).sum(2)  # [B, Hkv, N]
        at = torch.nonzero(live.view(-1)).view(-1)
        row, col = at // t.numel(), at % t.numel()
        s["w"][s["pages"][row, col // s["ps"]].long(), :, col % s["ps"]] = w[row, :, col]
        got["w"] = s["w"]
    return got


def _plain_evict(s):
    ps, budget = s["ps"], s["budget"]
    width = s["pages"].shape[1] * ps
    b, h = s["lens"].shape[0], s["Hkv"]
    t = torch.arange(width, device="cuda")
    lens = s["lens"].long()[:, None, None]
    w = s["w"][s["pages"].long()].transpose(1, 2).reshape(b, h, width)
    w = torch.where(t >= lens - s["recent"], math.inf, w)
    w = torch.where(t >= lens, -math.inf, w)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    new = torch.clamp(s["lens"], max=budget)
    j = torch.arange(min(budget, width), device="cuda")
    kept = torch.where(j < new.long()[:, None, None], order, width)
    kept = torch.sort(kept, dim=-1).values
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=width)
    kept = torch.where(kept == width, -1, kept)
    bi, hi, ji = torch.nonzero(kept >= 0, as_tuple=True)
    src = kept[bi, hi, ji]
    sp, so = s["pages"][bi, src // ps].long(), src % ps
    dp, do = s["dst"][bi, ji // ps].long(), ji % ps
    bits = torch.uint8 if s["kc"].dtype == torch.float8_e4m3fn else torch.int16
    kr, vr = _rows(s["kc"], s).view(bits), _rows(s["vc"], s).view(bits)
    kr[dp, do, hi] = kr[sp, so, hi]
    vr[dp, do, hi] = vr[sp, so, hi]
    s["w"][dp, hi, do] = s["w"][sp, hi, so]
    return {"kept": kept.to(torch.int32), "lens": new, **_copied(s)}


def _copied(s):
    """The buffers that an eviction writes into; an 8-bit cache as its bytes, which are only copied."""
    eight = s["kc"].dtype == torch.float8_e4m3fn
    return {"kc": s["kc"].view(torch.uint8) if eight else s["kc"], "vc": s["vc"].view(torch.uint8) if eight else s["vc"], "w": s["w"]}


def run(state):
    s = state
    if not own:
        return {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict}[s["op"]](s)
    import clove_compute_b200 as cc
    if s["op"] == "rope":
        if not s["append"]:
            q, k = cc.qk_norm_rope(s["q"], s["k"], s["table"], s["pos"], s["qw"], s["kw"], eps=1e-6, interleaved=s["interleaved"])
            return {"q": q, "k": k}
        q, _ = cc.qk_norm_rope(s["q"], s["k"], s["table"], s["pos"], s["qw"], s["kw"], eps=1e-6, interleaved=s["interleaved"],
                               V=s["v"], cache=s["handle"], slots=s["slots"])
        return {"q": q, "kc": s["kc"], "vc": s["vc"]}
    if s["op"] == "attn":
        if s["weights"]:
            o = cc.paged_attention(s["q"], s["handle"], s["pages"], s["lens"], window=s["window"], lse=s["lse"], key_weights=s["w"])
            return {"o": o, "lse": s["lse"], "w": s["w"]}
        o = cc.paged_attention(s["q"], s["handle"], s["pages"], s["lens"], window=s["window"], lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    kept, lens = cc.evict_cache(s["handle"], s["w"], s["pages"], s["lens"], s["dst"], s["budget"], s["recent"])
    return {"kept": kept, "lens": lens, **_copied(s)}


def work(case):
    b, h, d = BYTES[case["cache"]], case["Hkv"], case["D"]
    if case["op"] == "rope":
        t, q = case["T"], case["H"]
        out = 2 * q * d + 2 * h * d * (b if case["append"] else 1)
        moved = t * (2 * (q + 2 * h if case["append"] else q + h) * d + (out if case["append"] else 2 * (q + h) * d) + 4 * case["R"] + 4 + (4 if case["append"] else 0))
        return {"bytes": moved, "flops": t * (q + h) * (4 * d + 3 * case["R"])}
    lens = _lengths(case, 0)
    if case["op"] == "attn":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        moved = seen * h * d * 2 * b + 4 * case["B"] * case["H"] * (d + 1) + 4 * sum(-(-n // case["ps"]) for n in lens)
        return {"bytes": moved + (4 * seen * h if case["weights"] else 0), "flops": 4 * seen * case["H"] * d}
    keep = sum(min(n, case["budget"]) for n in lens)
    return {"bytes": 4 * sum(lens) * h + keep * h * (4 * d * b + 8), "flops": sum(lens) * h}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence."""
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    f64 = torch.float64
    if case["op"] == "rope":
        half = case["R"] // 2
        angle = s["table"].to(f64)[s["pos"].long()]

        def turned(x, weight):
            x = x.to(f64)
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + 1e-6) * weight.to(f64)
            head, rest = x[..., :case["R"]], x[..., case["R"]:]
            pairs = head.unflatten(-1, (half, 2)) if case["interleaved"] else head.unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_complex(pairs.contiguous()) * torch.complex(angle[:, None, :half], angle[:, None, half:])
            z = torch.view_as_real(z)
            z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            return torch.cat([z, rest], -1)

        q, k = turned(s["q"], s["qw"]), turned(s["k"], s["kw"])
        if not case["append"]:
            return {"q": q, "k": k}
        found = {"q": q, "kc": None, "vc": None}
        for name, x, scale in (("kc", k, s["k_scale"]), ("vc", s["v"].to(f64), s["v_scale"])):
            c = torch.zeros(s[name].shape, dtype=f64, device="cuda")
            at = s["slots"].long()
            x = (x / scale).clamp(-448, 448) if case["cache"] == "e4m3" else x
            if case["layout"] == "bshd":
                c[at // case["ps"], at % case["ps"]] = x
            else:
                c[at // case["ps"], :, at % case["ps"]] = x
            found[name] = c
        return found
    if case["op"] == "evict":
        return None  # copies and whole numbers
    group, ps = case["H"] // case["Hkv"], case["ps"]
    o = torch.zeros(s["q"].shape, dtype=f64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=f64, device="cuda")
    w = torch.zeros(s["w"].shape, dtype=f64, device="cuda") if case["weights"] else None
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        t = torch.arange(first, n, device="cuda")
        page, off = s["pages"][i].long()[t // ps], t % ps
        for g in range(case["Hkv"]):
            k = (s["kc"][page, off, g] if case["layout"] == "bshd" else s["kc"][page, g, off]) if case["cache"] != "e4m3" else None
            if k is None:
                raw = [c.view(torch.uint8) for c in (s["kc"], s["vc"])]
                k, v = [(c[page, off, g] if case["layout"] == "bshd" else c[page, g, off]).view(torch.float8_e4m3fn) for c in raw]
            else:
                v = s["vc"][page, off, g] if case["layout"] == "bshd" else s["vc"][page, g, off]
            heads = slice(g * group, (g + 1) * group)
            z = s["q"][i, heads].to(f64) @ (k.to(f64) * s["k_scale"]).T / math.sqrt(case["D"])
            lse[i, heads] = torch.logsumexp(z, -1)
            p = torch.exp(z - lse[i, heads, None])
            o[i, heads] = p @ (v.to(f64) * s["v_scale"])
            if w is not None:
                w[page, g, off] = p.sum(0)
    return {"o": o, "lse": lse, "w": w} if case["weights"] else {"o": o, "lse": lse}
