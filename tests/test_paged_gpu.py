"""Paged-cache operators on the GPU against plain 64-bit statements (tests/paged_ref.py,
which derives the bounds)."""
import math
import random

import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
INF = float("inf")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _pages(cc, lens, ps, Hkv, D, dtype, layout, gen, spare=2, k_scale=1.0, v_scale=1.0, width=None, joined=False):
    """A cache whose every unused slot is NaN, with pages in random order; the table's
    unused entries name no page. Returns (cache, page_table, seq_lens)."""
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + spare
    shape = (pages, ps, Hkv, D) if layout == "bshd" else (pages, Hkv, ps, D)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pages)).tolist()
    if joined:
        buf = _randn((pages, 2) + shape[1:], dtype, gen)
        K, V = buf[:, 0], buf[:, 1]
    else:
        K, V = _randn(shape, dtype, gen), _randn(shape, dtype, gen)
    width = max(need + [1]) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    raw = [t.view(torch.uint8) if dtype == E4M3 else t for t in (K, V)]
    nan = 0x7F if dtype == E4M3 else float("nan")
    at = 0
    for i, n in enumerate(lens):
        mine = order[at:at + need[i]]
        at += need[i]
        table[i, :need[i]] = torch.tensor(mine, dtype=torch.int32)
        if n % ps:
            for t in raw:
                (t[mine[-1], n % ps:] if layout == "bshd" else t[mine[-1], :, n % ps:]).fill_(nan)
    for pg in order[at:]:
        for t in raw:
            t[pg].fill_(nan)
    cache = cc.PagedCache(K, V, layout=layout, k_scale=k_scale, v_scale=v_scale)
    return cache, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _check_attention(cc, cache, table, lens, Q, window=0, scale=None, key_weights=None, before=None, **kw):
    """Runs the call and holds every output to the 64-bit statement."""
    B, H, D = Q.shape
    lse = torch.full((B, H), 7.0, device="cuda")
    O = cc.paged_attention(Q, cache, table, lens, window=window, scale=scale, lse=lse, key_weights=key_weights, **kw)
    torch.cuda.synchronize()
    assert cc.device_error() == 0
    sc = D ** -0.5 if scale is None else scale
    touched = None
    if key_weights is not None:
        touched = before.double().clone()
        slack = torch.zeros_like(touched)
    for i, n in enumerate(lens.tolist()):
        if n == 0:
            assert torch.all(O[i] == 0) and torch.all(lse[i] == -INF)
            continue
        first = max(0, n - window) if window else 0
        tab = table[i].clamp(min=0)
        k = ref.rows(cache.K, cache.layout, tab, n, cache.page_size) * cache.k_scale
        v = ref.rows(cache.V, cache.layout, tab, n, cache.page_size) * cache.v_scale
        o, l, w, b_o, b_l, b_w = ref.attention(Q[i], k, v, sc, first)
        err = (O[i].double() - o).abs()
        tol = b_o + ref.half_step(o.abs() + b_o, Q.dtype)
        assert torch.all(err <= tol), (i, n, float((err / tol).max()))
        assert torch.all((lse[i].double() - l).abs() <= b_l), (i, n, float(((lse[i].double() - l).abs() / b_l).max()))
        if key_weights is not None:
            t = torch.arange(first, n, device="cuda")
            page, off = table[i].long()[t // cache.page_size], t % cache.page_size
            touched[page, :, off] = (touched[page, :, off] if kw.get("accumulate") else 0.0) + w
            slack[page, :, off] = b_w + touched[page, :, off].abs() * ref.U
    if key_weights is not None:
        assert torch.all((key_weights.double() - touched).abs() <= slack), \
            float(((key_weights.double() - touched).abs() - slack).max())
    return O


LENS = [1, 15, 16, 17, 0, 63, 64, 65, 255, 256, 1000, 5]


@pytest.mark.parametrize("dtype,cache,D,layout,ps,Hkv,G", [
    (F16, F16, 128, "bshd", 16, 2, 4),
    (BF16, BF16, 128, "bhsd", 16, 2, 4),
    (F16, E4M3, 128, "bshd", 16, 2, 4),
    (BF16, E4M3, 128, "bhsd", 32, 1, 8),
    (F16, F16, 64, "bhsd", 64, 3, 1),
    (BF16, BF16, 64, "bshd", 128, 1, 5),
    (BF16, E4M3, 64, "bshd", 8, 2, 3),
    (F16, E4M3, 64, "bhsd", 16, 1, 12),
    (F16, F16, 256, "bshd", 16, 1, 2),
    (BF16, BF16, 256, "bhsd", 32, 2, 9),      # two blocks of heads, the second with one
    (F16, E4M3, 256, "bhsd", 16, 1, 7),
    (F16, F16, 128, "bshd", 16, 1, 9),        # blocks of 16
    (BF16, BF16, 128, "bshd", 16, 1, 16),
    (F16, F16, 128, "bhsd", 16, 1, 20),       # 16 + 4
    (F16, F16, 64, "bshd", 16, 1, 32),
    (BF16, E4M3, 128, "bshd", 16, 2, 16),
    (F16, F16, 128, "bshd", 1, 1, 4),         # one token per page
    (F16, F16, 128, "bhsd", 2, 2, 2),
    (BF16, E4M3, 128, "bshd", 4, 2, 2),
    (BF16, BF16, 64, "bhsd", 8, 1, 8),
    (F16, F16, 128, "bshd", 1024, 2, 1),      # a page longer than every sequence
])
def test_attention_matches_plain(clove_lib, cuda, dtype, cache, D, layout, ps, Hkv, G):
    g = _gen(D + ps + G)
    s = 0.75 if cache == E4M3 else 1.0
    c, table, lens = _pages(clove_lib, LENS, ps, Hkv, D, cache, layout, g, k_scale=s, v_scale=s)
    Q = _randn((len(LENS), Hkv * G, D), dtype, g, 2.0)
    _check_attention(clove_lib, c, table, lens, Q)


@pytest.mark.parametrize("lens", [
    [0], [1], [0, 0, 0], [20011], [0, 9000, 0, 1], [1] * 300, [0] * 100 + [77] + [0] * 100,
    [(i * 37) % 130 for i in range(1100)],
])
def test_attention_work_split(clove_lib, cuda, lens):
    """Batches that the even split of tiles cuts in every way: empty, one long sequence over
    all CTAs, hundreds of short ones, empty rows before, between and after."""
    g = _gen(len(lens))
    c, table, sl = _pages(clove_lib, lens, 16, 2, 64, F16, "bshd", g)
    _check_attention(clove_lib, c, table, sl, _randn((len(lens), 8, 64), F16, g, 2.0))


@pytest.mark.parametrize("lens,D,cache,G,weights", [
    ([300007, 0, 151001, 41], 64, E4M3, 3, True),
    ([200003, 40, 60000], 128, F16, 4, False),
    ([131071, 131072, 5], 128, E4M3, 12, False),
    ([130001], 256, BF16, 2, False),
])
def test_attention_long_calls(clove_lib, cuda, lens, D, cache, G, weights):
    """Hundreds of tiles for every CTA, items over dozens of CTAs, page windows refilled many
    times: right, the same bit for bit every time, and captured."""
    g = _gen(D + G)
    Hkv = 8
    s = 0.5 if cache == E4M3 else 1.0
    dtype = F16 if cache == E4M3 else cache
    c, table, sl = _pages(clove_lib, lens, 64, Hkv, D, cache, "bshd", g, k_scale=s, v_scale=s)
    Q = _randn((len(lens), Hkv * G, D), dtype, g, 2.0)
    w = torch.zeros((c.num_pages, Hkv, 64), device="cuda") if weights else None
    want = _check_attention(clove_lib, c, table, sl, Q, key_weights=w, before=torch.zeros_like(w) if weights else None)
    for _ in range(10):
        assert torch.equal(clove_lib.paged_attention(Q, c, table, sl), want)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = clove_lib.paged_attention(Q, c, table, sl)
    for _ in range(3):
        o.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
    assert clove_lib.device_error() == 0


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 4096])
@pytest.mark.parametrize("ps", [4, 32])
def test_attention_window_skips_released_pages(clove_lib, cuda, window, ps):
    """Pages that lie wholly before the window are not looked up: their entries are -1."""
    lens = [1, 16, 33, 300, 1025, 0]
    g = _gen(window)
    c, table, sl = _pages(clove_lib, lens, ps, 2, 128, BF16, "bshd", g)
    Q = _randn((len(lens), 4, 128), BF16, g, 2.0)
    cut = table.clone()
    for i, n in enumerate(lens):
        cut[i, :max(0, n - window) // ps] = -1
    O = clove_lib.paged_attention(Q, c, cut, sl, window=window)
    assert clove_lib.device_error() == 0
    assert torch.equal(O, _check_attention(clove_lib, c, table, sl, Q, window=window))


@pytest.mark.parametrize("layout,ps,G,dtype,cache,window,accumulate", [
    ("bshd", 16, 4, F16, F16, 0, False),
    ("bhsd", 64, 1, BF16, BF16, 0, True),
    ("bshd", 2, 5, F16, E4M3, 100, True),
    ("bhsd", 32, 20, BF16, BF16, 40, False),
])
def test_attention_key_weights(clove_lib, cuda, layout, ps, G, dtype, cache, window, accumulate):
    g = _gen(ps + G)
    lens = [0, 1, 64, 700, 5000]
    c, table, sl = _pages(clove_lib, lens, ps, 2, 128, cache, layout, g)
    w = torch.rand((c.num_pages, 2, ps), device="cuda", generator=g)
    _check_attention(clove_lib, c, table, sl, _randn((5, 2 * G, 128), dtype, g, 2.0), window=window,
                     key_weights=w, before=w.clone(), accumulate=accumulate)


def test_attention_large_and_masked_scores(clove_lib, cuda):
    """Scores of +-10^4 (one key takes everything), keys that raise the maximum late, and a
    scale of its own: no overflow, weights that vanish are zero."""
    g = _gen(5)
    lens = [500, 64]
    c, table, sl = _pages(clove_lib, lens, 16, 1, 128, F16, "bshd", g)
    Q = _randn((2, 4, 128), F16, g, 20.0)
    _check_attention(clove_lib, c, table, sl, Q, scale=3.0)
    last = c.K[int(table[0, 499 // 16]), 499 % 16]
    last.copy_((Q[0, :1] / Q[0, :1].float().norm() * 200).half())
    _check_attention(clove_lib, c, table, sl, Q, scale=0.5)


def test_attention_nan_and_infinity(clove_lib, cuda):
    """A NaN among the attended keys spreads to its own sequence and key head only; an
    infinite V value to its own column."""
    g = _gen(6)
    c, table, sl = _pages(clove_lib, [100, 300, 50], 16, 2, 64, F16, "bshd", g)
    Q = _randn((3, 4, 64), F16, g)
    c.K[int(table[1, 3]), 5, 1, 7] = float("nan")
    c.V[int(table[0, 2]), 1, 0, 9] = INF
    O = clove_lib.paged_attention(Q, c, table, sl)
    bad = ~torch.isfinite(O)
    assert bad[1, 2:].all() and bad[0, :2, 9].all()
    assert int(bad.sum()) == 2 * 64 + 2


def test_attention_strided_operands_and_joined_cache(clove_lib, cuda):
    """Q as a block of a fused projection's rows, O inside a larger buffer whose neighbours
    stay as they were, K and V as halves of one buffer, page-table rows inside wider ones."""
    g = _gen(7)
    lens = [100, 300, 50]
    c, table, sl = _pages(clove_lib, lens, 16, 2, 128, BF16, "bhsd", g, joined=True)
    qkv = _randn((3, 8 * 128 + 512), BF16, g, 2.0)
    Q = qkv[:, 256:256 + 8 * 128].view(3, 8, 128)
    buf = torch.full((5, 1200), 3.0, dtype=BF16, device="cuda")
    O = buf[1:4, 64:64 + 1024].view(3, 8, 128)
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table
    _check_attention(clove_lib, c, wide[:, 2:2 + table.shape[1]], sl, Q, O=O)
    buf[1:4, 64:64 + 1024] = 3.0
    assert torch.all(buf == 3.0)


def test_attention_offsets_beyond_32_bits(clove_lib, cuda):
    """Pages whose element offsets pass 2^32 (a buffer of 8.9 GB)."""
    ps, Hkv, D = 16, 4, 128
    pages = (1 << 32) // (ps * Hkv * D) + 1500
    buf = torch.empty((pages, ps, Hkv, D), dtype=F16, device="cuda")
    g = _gen(8)
    order = [pages - 1, 0, pages - 700, (1 << 31) // (ps * Hkv * D), 5]
    for pg in order:
        buf[pg] = _randn((ps, Hkv, D), F16, g)
    c = clove_lib.PagedCache(buf, buf)
    table = torch.tensor([order, order[::-1]], dtype=torch.int32, device="cuda")
    sl = torch.tensor([80, 71], dtype=torch.int32, device="cuda")
    _check_attention(clove_lib, c, table, sl, _randn((2, 8, D), F16, g, 2.0))


def test_attention_bad_pages_and_lengths_are_reported(clove_lib, cuda):
    """A page outside the cache reads as zeros, a length outside the table is clamped; both
    set device error 3, and the other sequences are not affected."""
    g = _gen(9)
    c, table, sl = _pages(clove_lib, [64, 64, 64], 16, 1, 64, F16, "bshd", g)
    Q = _randn((3, 2, 64), F16, g)
    good = clove_lib.paged_attention(Q, c, table, sl)
    for bad in (-1, c.num_pages, 1 << 30, -(1 << 31)):
        t = table.clone()
        t[1, 2] = bad
        O = clove_lib.paged_attention(Q, c, t, sl)
        assert clove_lib.device_error() == 3
        assert torch.equal(O[0], good[0]) and torch.equal(O[2], good[2]) and torch.isfinite(O[1]).all()
    for n in (65, 1 << 30, -5, -(1 << 31)):
        s = sl.clone()
        s[2] = n
        O = clove_lib.paged_attention(Q, c, table, s)
        assert clove_lib.device_error() == 3
        assert torch.equal(O[:2], good[:2])
        assert torch.equal(O[2], good[2]) if n > 0 else torch.all(O[2] == 0)
    assert clove_lib.device_error() == 0


def test_attention_repeats_bit_for_bit(clove_lib, cuda):
    g = _gen(10)
    lens = [3000, 1, 500, 7000]
    c, table, sl = _pages(clove_lib, lens, 16, 4, 128, F16, "bshd", g)
    Q = _randn((4, 16, 128), F16, g, 2.0)
    first = clove_lib.paged_attention(Q, c, table, sl)
    for _ in range(20):
        assert torch.equal(clove_lib.paged_attention(Q, c, table, sl), first)


def test_attention_streams_and_graphs(clove_lib, cuda):
    """Two calls at once on two streams; a captured call replayed while the sequences grow;
    two captured graphs replayed side by side."""
    g = _gen(11)
    lens = [900, 17, 2500]
    c, table, sl = _pages(clove_lib, lens, 16, 2, 128, F16, "bshd", g)
    Q = [_randn((3, 8, 128), F16, g, 2.0) for _ in range(2)]
    want = [clove_lib.paged_attention(q, c, table, sl) for q in Q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [clove_lib.paged_attention(q, c, table, sl, stream=s) for q, s in zip(Q, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = clove_lib.paged_attention(Q[0], c, table, sl, stream=streams[0].cuda_stream)  # a raw handle
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    graphs, outs, lsub = [], [], sl.clone()
    for q in Q:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(clove_lib.paged_attention(q, c, table, lsub))
        graphs.append(gr)
    for step in ([900, 17, 2500], [1, 0, 2499], [899, 16, 64]):
        lsub.copy_(torch.tensor(step, dtype=torch.int32))
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        now = torch.tensor(step, dtype=torch.int32, device="cuda")
        for q, o in zip(Q, outs):
            assert torch.equal(o, clove_lib.paged_attention(q, c, table, now))
    assert clove_lib.device_error() == 0


def test_attention_on_more_streams_than_are_kept(clove_lib, cuda):
    """Each stream has a workspace of its own; beyond 64 streams a call brings one."""
    from cuda.bindings import runtime as rt
    g = _gen(12)
    c, table, sl = _pages(clove_lib, [900, 17, 2500], 16, 2, 128, F16, "bshd", g)
    Q = _randn((3, 8, 128), F16, g, 2.0)
    want = clove_lib.paged_attention(Q, c, table, sl)
    torch.cuda.synchronize()
    handles = []
    for _ in range(80):
        err, s = rt.cudaStreamCreate()
        assert int(err) == 0
        handles.append(s)
    try:
        for _ in range(2):
            got = [clove_lib.paged_attention(Q, c, table, sl, stream=int(s)) for s in handles]
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in got)
    finally:
        torch.cuda.synchronize()
        for s in handles:
            rt.cudaStreamDestroy(s)
    assert clove_lib.device_error() == 0


def test_attention_from_two_threads_on_one_stream(clove_lib, cuda):
    import threading
    g = _gen(13)
    c, table, sl = _pages(clove_lib, [900, 17, 2500], 16, 2, 128, BF16, "bhsd", g)
    Q = [_randn((3, 8, 128), BF16, g, 2.0) for _ in range(2)]
    w = [torch.zeros((c.num_pages, 2, 16), device="cuda") for _ in range(2)]
    want = []
    for q, x in zip(Q, w):
        want.append((clove_lib.paged_attention(q, c, table, sl, key_weights=x), x.clone()))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        torch.cuda.set_device(0)
        for _ in range(50):
            o = clove_lib.paged_attention(Q[i], c, table, sl, key_weights=w[i])
            if not torch.equal(o, want[i][0]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad and all(torch.equal(x, y[1]) for x, y in zip(w, want))
    assert clove_lib.device_error() == 0


_CAPTURE_FIRST = r"""
import torch
import clove_compute_b200 as cc
g = torch.Generator(device="cuda").manual_seed(1)
K, V = (torch.randn((200, 16, 2, 128), device="cuda", generator=g).half() for _ in range(2))
c = cc.PagedCache(K, V)
table = torch.randperm(200, device="cuda", generator=g)[:190].to(torch.int32).view(1, 190)
sl = torch.tensor([3000], dtype=torch.int32, device="cuda")
Q = torch.randn((1, 8, 128), device="cuda", generator=g).half()
torch.cuda.synchronize()
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr):
    o = cc.paged_attention(Q, c, table, sl)
for _ in range(3):
    o.zero_()
    gr.replay()
    torch.cuda.synchronize()
    first = o.clone()
assert torch.equal(first, cc.paged_attention(Q, c, table, sl))
assert cc.device_error() == 0
print("captured first ok")
"""


def test_attention_captured_before_any_other_call(clove_lib, cuda):
    """The first call of a process may be a captured one."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _CAPTURE_FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first ok" in r.stdout, r.stderr[-2000:]


def test_attention_after_other_work_on_the_stream(clove_lib, cuda):
    """Kernels overlap their predecessors' ends: a step whose queries, lengths and cache the
    kernels just before it write, many times over, with nothing waiting in between."""
    cc = clove_lib
    g = _gen(14)
    Hkv, H, D, ps, steps = 2, 8, 128, 16, 40
    W = _randn((512, (H + 2 * Hkv) * D), F16, g, 512 ** -0.5)
    X = _randn((steps, 2, 512), F16, g)
    rope = cc.rope_table(256, D)
    outs = []
    for wait in (True, False):
        K, V = (torch.zeros((12, ps, Hkv, D), dtype=F16, device="cuda") for _ in range(2))
        cache = cc.PagedCache(K, V)
        table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
        lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        got = []
        for t in range(steps):
            qkv = cc.gemm_fp16(X[t], W)
            pos = lens.clone()
            slots = table[:, t // ps] * ps + t % ps
            lens += 1
            q, k, v = (qkv[:, a * D:b * D].view(2, b - a, D) for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
            q, _ = cc.qk_norm_rope(q, k, rope, pos, V=v, cache=cache, slots=slots.to(torch.int32))
            got.append(cc.paged_attention(q, cache, table, lens))
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        outs.append(torch.stack(got))
    assert torch.equal(outs[0], outs[1])
    assert cc.device_error() == 0


# ---------------------------------------------------------------------------
# norm + rotation + append
# ---------------------------------------------------------------------------
def _norm_rope_case(cc, T, H, Hkv, D, R, dtype, cache_dtype, interleaved, norm, layout, seed, fused=True, ps=16):
    g = _gen(seed)
    if fused:
        qkv = _randn((T, (H + 2 * Hkv) * D), dtype, g, 1.5)
        Q = qkv[:, :H * D].view(T, H, D)
        K = qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D)
        V = qkv[:, (H + Hkv) * D:].view(T, Hkv, D)
    else:
        Q, K, V = (_randn((T, h, D), dtype, g, 1.5) for h in (H, Hkv, Hkv))
    qw = kw = None
    if norm:
        qw, kw = _randn((D,), dtype, g), _randn((D,), dtype, g)
    table = cc.rope_table(5000, R)
    pos = torch.randint(0, 5000, (T,), device="cuda", generator=g, dtype=torch.int32)
    args = dict(Q=Q, K=K, rope_table=table, positions=pos, q_weight=qw, k_weight=kw, interleaved=interleaved)
    yq, mq = ref.norm_rope(Q, qw, table, pos, interleaved, 1e-6)
    yk, mk = ref.norm_rope(K, kw, table, pos, interleaved, 1e-6)
    cache = slots = None
    if cache_dtype is not None:
        pages = -(-T // ps) + 3
        shape = (pages, ps, Hkv, D) if layout == "bshd" else (pages, Hkv, ps, D)
        s = 0.3 if cache_dtype == E4M3 else 1.0
        cache = cc.PagedCache(*(torch.full(shape, 5.0, device="cuda").to(cache_dtype) for _ in range(2)),
                              layout=layout, k_scale=s, v_scale=s)
        slots = torch.randperm(pages * ps, device="cuda", generator=g)[:T].to(torch.int32)
    return args, V, cache, slots, (yq, mq), (yk, mk)


def _close(got, want, mag, dtype, scale=1.0):
    """Within half a step of the type and 16 units of fp32 per unit of magnitude; e4m3
    saturates, and its division by the scale is one more rounding."""
    want, slack = want / scale, mag / scale * 17 * ref.U
    if dtype == E4M3:
        want = want.clamp(-448, 448)
    err = (got.double() - want).abs()
    tol = ref.half_step(want.abs() + slack, dtype) + slack
    assert torch.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("T,H,Hkv,D,R,dtype,cache,interleaved,norm,layout", [
    (1, 32, 32, 128, 128, F16, F16, False, True, "bshd"),
    (1, 1, 1, 64, 64, BF16, None, False, True, "bshd"),
    (7, 8, 2, 128, 128, BF16, E4M3, True, True, "bhsd"),
    (33, 5, 1, 128, 64, F16, E4M3, False, True, "bshd"),
    (65, 4, 4, 64, 64, F16, F16, True, False, "bhsd"),
    (65, 4, 2, 64, 16, BF16, BF16, False, True, "bshd"),
    (130, 3, 1, 256, 256, F16, F16, False, True, "bshd"),
    (17, 2, 2, 256, 48, BF16, E4M3, True, True, "bhsd"),
    (9, 12, 3, 128, 112, F16, None, True, True, "bshd"),
    (9, 12, 3, 128, 128, F16, None, False, False, "bshd"),
    (3001, 32, 8, 128, 128, F16, F16, False, True, "bshd"),   # four rows per lane
    (6007, 7, 1, 64, 32, BF16, E4M3, True, True, "bhsd"),
    (4099, 6, 2, 256, 256, BF16, None, False, True, "bshd"),
    (333, 96, 16, 128, 128, F16, F16, False, True, "bshd"),    # a token's rows in two pieces
    (700, 100, 33, 256, 192, BF16, E4M3, True, True, "bhsd"),  # in six
])
@pytest.mark.parametrize("path", [0, 1, 2])  # automatic, the streaming kernel, the direct one
def test_norm_rope_matches_plain(clove_lib, cuda, T, H, Hkv, D, R, dtype, cache, interleaved, norm, layout, path):
    args, V, c, slots, (yq, mq), (yk, mk) = _norm_rope_case(clove_lib, T, H, Hkv, D, R, dtype, cache, interleaved,
                                                            norm, layout, seed=T + D)
    clove_lib.set_dispatch_override(path)
    try:
        q, k = clove_lib.qk_norm_rope(**args, **(dict(V=V, cache=c, slots=slots) if c else {}))
        torch.cuda.synchronize()
    finally:
        clove_lib.set_dispatch_override(0)
    assert clove_lib.device_error() == 0
    _close(q, yq, mq, dtype)
    if c is None:
        _close(k, yk, mk, dtype)
        return
    assert k is None
    s = slots.long()
    for buf, want, mag, scale in ((c.K, yk, mk, c.k_scale), (c.V, V.double(), torch.zeros_like(mk), c.v_scale)):
        rows = buf if layout == "bshd" else buf.transpose(1, 2)
        raw = rows.contiguous().view(torch.uint8).view(-1, Hkv, D * buf.element_size())
        got = raw[s].view(cache).view(T, Hkv, D)
        _close(got, want, mag if buf is c.K else want.abs(), cache, scale)
        rest = torch.ones(raw.shape[0], dtype=torch.bool, device="cuda")
        rest[s] = False
        assert torch.all(raw[rest].contiguous().view(cache).float() == 5.0)  # other slots stay


@pytest.mark.parametrize("path", [1, 2])
def test_norm_rope_padding_slots_and_bad_indices(clove_lib, cuda, path):
    """Padding tokens and tokens without a slot leave everything as it was; positions and
    slots outside their range are reported and not followed."""
    clove_lib.set_dispatch_override(path)
    try:
        _padding_slots_and_bad_indices(clove_lib)
    finally:
        clove_lib.set_dispatch_override(0)


def _padding_slots_and_bad_indices(clove_lib):
    T, H, Hkv, D = 12, 4, 2, 128
    args, V, c, slots, (yq, mq), (yk, mk) = _norm_rope_case(clove_lib, T, H, Hkv, D, D, F16, F16, False, True, "bshd", 3)
    args["positions"][2] = -1
    slots[5] = -3
    qo = torch.full((T, H, D), 9.0, dtype=F16, device="cuda")
    ko = torch.full((T, Hkv, D), 9.0, dtype=F16, device="cuda")
    clove_lib.qk_norm_rope(**args, V=V, cache=c, slots=slots, Q_out=qo, K_out=ko)
    assert clove_lib.device_error() == 0
    live = [t for t in range(T) if t != 2]
    assert torch.all(qo[2] == 9) and torch.all(ko[2] == 9)
    yq, _ = ref.norm_rope(args["Q"], args["q_weight"], args["rope_table"], args["positions"].clamp(min=0), False, 1e-6)
    _close(qo[live], yq[live], mq[live] + 1, F16)
    kept = (c.K.view(-1, Hkv, D) != 5).any(-1).any(-1).nonzero().view(-1).tolist()
    assert sorted(kept) == sorted(int(slots[t]) for t in live if t != 5)
    for name, value in (("positions", 5000), ("positions", 2 ** 31 - 1), ("slots", c.num_pages * 16), ("slots", 2 ** 31 - 1)):
        a = dict(args)
        sl = slots.clone()
        if name == "positions":
            a["positions"] = args["positions"].clone()
            a["positions"][0] = value
        else:
            sl[0] = value
        before = c.K.clone()
        q2 = torch.full_like(qo, 9.0)
        clove_lib.qk_norm_rope(**a, V=V, cache=c, slots=sl, Q_out=q2)
        assert clove_lib.device_error() == 3
        assert torch.equal(c.K, before)
        assert torch.all(q2[0] == 9) if name == "positions" else torch.equal(q2, torch.where(q2 == 9, q2, qo))


def test_norm_rope_in_place_and_strided_outputs(clove_lib, cuda):
    T, H, Hkv, D = 50, 6, 2, 64
    args, V, c, slots, *_ = _norm_rope_case(clove_lib, T, H, Hkv, D, D, BF16, None, True, True, "bshd", 4)
    q, k = clove_lib.qk_norm_rope(**args)
    clove_lib.qk_norm_rope(**args, Q_out=args["Q"], K_out=args["K"])  # blocks of the fused rows
    torch.cuda.synchronize()
    assert torch.equal(args["Q"], q) and torch.equal(args["K"], k)


def test_norm_rope_extreme_rows(clove_lib, cuda):
    """Zero rows stay zero, a row of the type's largest values does not overflow in the sum
    of squares, NaN stays in its row."""
    D = 128
    Q = torch.zeros(3, 2, D, dtype=F16, device="cuda")
    Q[1] = 65504.0
    Q[2, 0, 5] = float("nan")
    K = Q[:, :1].contiguous()
    w = torch.ones(D, dtype=F16, device="cuda")
    table = clove_lib.rope_table(4, D)
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    q, k = clove_lib.qk_norm_rope(Q, K, table, pos, w, w)
    assert torch.all(q[0] == 0) and torch.all(q[1] == 1) and torch.isnan(q[2, 0]).all() and torch.all(q[2, 1] == 0)


def test_norm_rope_empty_and_capture(clove_lib, cuda):
    args, V, c, slots, *_ = _norm_rope_case(clove_lib, 20, 4, 2, 128, 128, F16, E4M3, False, True, "bhsd", 5)
    empty = {n: (t[:0] if n in ("Q", "K", "positions") else t) for n, t in args.items()}
    q, _ = clove_lib.qk_norm_rope(**empty, V=V[:0], cache=c, slots=slots[:0])
    assert q.shape == (0, 4, 128)
    want, _ = clove_lib.qk_norm_rope(**args, V=V, cache=c, slots=slots)
    wk = c.K.view(torch.uint8).clone()
    c.K.view(torch.uint8).zero_()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got, _ = clove_lib.qk_norm_rope(**args, V=V, cache=c, slots=slots)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    s = slots.long()
    a, b = (x.transpose(1, 2).reshape(-1, 2, 128)[s] for x in (c.K.view(torch.uint8), wk))
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def _weights(kind, shape, gen):
    if kind == "ties":
        return torch.randint(0, 3, shape, device="cuda", generator=gen).float()
    if kind == "zeros":
        return torch.rand(shape, device="cuda", generator=gen).sub_(0.9).clamp_(min=0)
    if kind == "odd":
        w = torch.randn(shape, device="cuda", generator=gen)
        r = torch.rand(shape, device="cuda", generator=gen)
        for lo, x in ((0.0, float("nan")), (0.1, INF), (0.2, -INF), (0.3, -0.0), (0.4, 0.0), (0.5, 1e-42)):
            w = torch.where((r >= lo) & (r < lo + 0.1), torch.full_like(w, x), w)
        return w
    return torch.rand(shape, device="cuda", generator=gen).pow_(8)


def _check_evict(cc, lens, budget, recent, ps, Hkv, D, dtype, layout, kind, seed=0):
    g = _gen(seed + budget)
    keep = [min(n, budget) for n in lens]
    cache, table, sl = _pages(cc, lens, ps, Hkv, D, dtype, layout, g, spare=sum(-(-n // ps) for n in keep) + 1)
    used = set(table[table >= 0].tolist())
    free = [pg for pg in range(cache.num_pages) if pg not in used]
    width = -(-budget // ps)
    dst = torch.full((len(lens), width), -1, dtype=torch.int32)
    for i, n in enumerate(keep):
        need = -(-n // ps)
        dst[i, :need] = torch.tensor([free.pop() for _ in range(need)], dtype=torch.int32)
    dst = dst.cuda()
    w = _weights(kind, (cache.num_pages, Hkv, ps), g)
    K0, V0, w0 = cache.K.clone(), cache.V.clone(), w.clone()
    kept, new = cc.evict_cache(cache, w, table, sl, dst, budget, recent)
    torch.cuda.synchronize()
    assert cc.device_error() == 0
    assert new.tolist() == keep
    bits = torch.uint8 if dtype == E4M3 else torch.int16
    wantK, wantV, want_w = K0.clone().view(bits), V0.clone().view(bits), w0.clone()
    for i, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        mine = w0[table[i].long()[t // ps], :, t % ps].T.tolist() if n else [[]] * Hkv  # [Hkv][n]
        for h in range(Hkv):
            want = ref.evict(mine[h], n, budget, recent)
            assert kept[i, h].tolist() == want + [-1] * (budget - len(want)), (i, h)
            if not want:
                continue
            s = torch.tensor(want, device="cuda")
            j = torch.arange(len(want), device="cuda")
            sp, so, dp, do = table[i].long()[s // ps], s % ps, dst[i].long()[j // ps], j % ps
            for out, src in ((wantK, K0.view(bits)), (wantV, V0.view(bits))):
                if layout == "bshd":
                    out[dp, do, h] = src[sp, so, h]
                else:
                    out[dp, h, do] = src[sp, h, so]
            want_w[dp, h, do] = w0[sp, h, so]
    assert torch.equal(cache.K.view(bits), wantK) and torch.equal(cache.V.view(bits), wantV)  # the rest untouched
    assert torch.equal(w.view(torch.int32), want_w.view(torch.int32))


@pytest.mark.parametrize("kind", ["random", "ties", "zeros", "odd"])
@pytest.mark.parametrize("lens,budget,recent,ps,Hkv,D,dtype,layout", [
    ([0, 1, 99, 100, 101, 500], 100, 10, 16, 2, 64, F16, "bshd"),
    ([2500], 1000, 0, 32, 1, 128, BF16, "bhsd"),
    ([700, 3], 64, 64, 8, 3, 128, E4M3, "bshd"),       # only recent keys
    ([300, 40], 1, 0, 1, 1, 256, F16, "bhsd"),
    ([1030] * 40, 37, 5, 16, 8, 64, E4M3, "bhsd"),     # one CTA per row
])
def test_evict_matches_plain(clove_lib, cuda, kind, lens, budget, recent, ps, Hkv, D, dtype, layout):
    _check_evict(clove_lib, lens, budget, recent, ps, Hkv, D, dtype, layout, kind)


@pytest.mark.parametrize("n,Hkv,budget,recent", [
    (150001, 2, 20000, 777),     # slices held whole in shared memory
    (210011, 1, 9999, 1),        # slices longer than that
])
@pytest.mark.parametrize("kind", ["random", "zeros"])
def test_evict_long_sequence(clove_lib, cuda, n, Hkv, budget, recent, kind):
    _check_evict(clove_lib, [n], budget, recent, 64, Hkv, 64, E4M3, "bshd", kind)


def test_evict_repeats_bit_for_bit(clove_lib, cuda):
    """Clusters of eight CTAs that run beside each other at different speeds (other rows end
    at once, another stream is busy): every run keeps the same keys."""
    g = _gen(31)
    lens = [60001, 0, 40, 33000]
    cache, table, sl = _pages(clove_lib, lens, 32, 2, 64, E4M3, "bhsd", g, spare=4 * 100)
    used = set(table[table >= 0].tolist())
    free = [pg for pg in range(cache.num_pages) if pg not in used]
    dst = torch.tensor([free[i * 94:(i + 1) * 94] for i in range(4)], dtype=torch.int32, device="cuda")
    sets = [_weights(kind, (cache.num_pages, 2, 32), g) for kind in ("zeros", "ties", "odd", "random")]
    want = [clove_lib.evict_cache(cache, w, table, sl, dst, 3000, 17)[0].clone() for w in sets]
    torch.cuda.synchronize()
    other, x = torch.cuda.Stream(), torch.randn(1 << 24, device="cuda")
    for i in range(200):
        with torch.cuda.stream(other):
            x.mul_(1.0)
        got, _ = clove_lib.evict_cache(cache, sets[i % 4], table, sl, dst, 3000, 17)
        assert torch.equal(got, want[i % 4]), i
    torch.cuda.synchronize()


def test_evict_long_rows_in_one_cta(clove_lib, cuda):
    """Over 148 rows: one CTA each, with slices longer than its shared memory holds."""
    _check_evict(clove_lib, [30011], 5000, 100, 64, 150, 64, E4M3, "bhsd", "zeros")


def test_evict_bad_pages_are_reported(clove_lib, cuda):
    g = _gen(1)
    cache, table, sl = _pages(clove_lib, [64, 64], 16, 1, 64, F16, "bshd", g, spare=4)
    used = set(table.view(-1).tolist())
    free = [pg for pg in range(cache.num_pages) if pg not in used]
    dst = torch.tensor([free[:2], free[2:4]], dtype=torch.int32, device="cuda")
    w = torch.rand((cache.num_pages, 1, 16), device="cuda", generator=g)
    w0 = w.clone()
    for which, bad in (("src", -1), ("src", cache.num_pages), ("dst", -1), ("dst", 1 << 30)):
        t, d = table.clone(), dst.clone()
        (t if which == "src" else d)[0, 1] = bad
        K0 = cache.K.clone()
        kept, new = clove_lib.evict_cache(cache, w, t, sl, d, 32, 4)
        assert clove_lib.device_error() == 3
        assert new.tolist() == [32, 32]
        flat = cache.K[dst[1].long()].view(-1, 64)
        src = K0[table[1].long()].view(-1, 64)
        assert torch.equal(flat, src[kept[1, 0].long()])
        w.copy_(w0)
    s = sl.clone()
    s[0] = 1 << 30
    _, new = clove_lib.evict_cache(cache, w, table, s, dst, 32, 4)
    assert clove_lib.device_error() == 3 and new.tolist() == [32, 32]
    assert clove_lib.device_error() == 0


def test_evict_capture(clove_lib, cuda):
    g = _gen(2)
    cache, table, sl = _pages(clove_lib, [500, 90], 16, 2, 128, BF16, "bshd", g, spare=12)
    used = set(table[table >= 0].tolist())
    free = [pg for pg in range(cache.num_pages) if pg not in used]
    dst = torch.tensor([free[:5], free[5:10]], dtype=torch.int32, device="cuda")
    w = torch.rand((cache.num_pages, 2, 16), device="cuda", generator=g)
    want, _ = clove_lib.evict_cache(cache, w, table, sl, dst, 80, 9)
    K = cache.K.clone()
    cache.K[dst.view(-1).long()] = 0
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kept, new = clove_lib.evict_cache(cache, w, table, sl, dst, 80, 9)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, want) and new.tolist() == [80, 80] and torch.equal(cache.K.view(torch.int16), K.view(torch.int16))


# ---------------------------------------------------------------------------
# refusals of the Python layer (nothing is launched)
# ---------------------------------------------------------------------------
def _call_args(cc):
    K, V = (torch.zeros((8, 16, 2, 128), dtype=F16, device="cuda") for _ in range(2))
    cache = cc.PagedCache(K, V)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    f32 = lambda *s: torch.zeros(s, device="cuda")
    h = lambda *s: torch.zeros(s, dtype=F16, device="cuda")
    rope = dict(Q=h(3, 4, 128), K=h(3, 2, 128), rope_table=f32(64, 128), positions=i32(3), q_weight=h(128),
                k_weight=h(128), V=h(3, 2, 128), cache=cache, slots=i32(3) - 1)
    attn = dict(Q=h(3, 4, 128), cache=cache, page_table=i32(3, 2), seq_lens=i32(3), lse=f32(3, 4),
                key_weights=f32(8, 2, 16), O=h(3, 4, 128))
    evict = dict(cache=cache, key_weights=f32(8, 2, 16), page_table=i32(3, 2), seq_lens=i32(3),
                 dst_table=i32(3, 2), budget=20)
    return {"qk_norm_rope": rope, "paged_attention": attn, "evict_cache": evict}


def _wrongs(name, x):
    """Wrong values for a tensor argument and the exceptions they may raise."""
    yield x.cpu(), ValueError
    yield x.double(), TypeError
    yield None, (TypeError, ValueError)
    yield "text", TypeError
    yield torch.cat([x, x]), ValueError               # another first size
    yield x[..., :-1], ValueError                     # another last size
    yield x.unsqueeze(0), ValueError                  # another number of dimensions
    wide = torch.zeros(x.shape[:-1] + (2 * x.shape[-1],), dtype=x.dtype, device="cuda")
    yield wide[..., ::2], ValueError                  # a stride in the last dimension


@pytest.mark.parametrize("fn", ["qk_norm_rope", "paged_attention", "evict_cache"])
def test_python_layer_refuses(clove_lib, cuda, fn):
    args = _call_args(clove_lib)[fn]
    call = getattr(clove_lib, fn)
    call(**args)  # as it stands it runs
    may_differ = {("rope_table", 0), ("page_table", 1), ("dst_table", 1)}  # sizes that are the caller's choice
    optional = {"lse", "key_weights", "O"} if fn == "paged_attention" else set()
    for name, x in args.items():
        if not isinstance(x, torch.Tensor):
            continue
        for k, (bad, exc) in enumerate(_wrongs(name, x)):
            if (k == 4 and (name, 0) in may_differ) or (k == 5 and (name, 1) in may_differ):
                continue
            if k == 2 and name in optional:
                continue
            with pytest.raises(exc):
                call(**{**args, name: bad})
    with pytest.raises(TypeError):
        call(**{**args, "cache": "text"})
    if fn == "qk_norm_rope":
        for a in (dict(cache=None), dict(V=None, slots=None), dict(q_weight=None), dict(eps="x")):
            with pytest.raises((TypeError, ValueError)):
                call(**{**args, **a})
        with pytest.raises(clove_lib.CloveError):
            call(**{**args, "eps": -1.0})
    elif fn == "paged_attention":
        for a in (dict(key_weights=None, accumulate=True), dict(window="x"), dict(window=1 << 40), dict(scale="x")):
            with pytest.raises((TypeError, ValueError)):
                call(**{**args, **a})
        with pytest.raises(clove_lib.CloveError):
            call(**{**args, "scale": 0.0})
    else:
        for a in (dict(budget=0), dict(budget=1 << 40), dict(recent="x")):
            with pytest.raises((TypeError, ValueError)):
                call(**{**args, **a})
        for a in (dict(recent=21), dict(budget=100)):
            with pytest.raises(clove_lib.CloveError):
                call(**{**args, **a})
    torch.cuda.synchronize()
    assert clove_lib.device_error() == 0


def test_empty_batches_and_single_dimensions(clove_lib, cuda):
    """Calls of no sequence; caches whose dimensions of size 1 have odd strides."""
    cc = clove_lib
    g = _gen(40)
    K, V = (torch.randn((9, 16, 1, 64), device="cuda", generator=g).half() for _ in range(2))
    cache = cc.PagedCache(K, V)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    tab = torch.zeros((0, 4), dtype=torch.int32, device="cuda")
    assert cc.paged_attention(K.new_zeros((0, 3, 64)), cache, tab, none).shape == (0, 3, 64)
    w = torch.zeros((9, 1, 16), device="cuda")
    kept, new = cc.evict_cache(cache, w, tab, none, tab, 20)
    assert kept.shape == (0, 1, 20) and new.shape == (0,)
    table = torch.tensor([[3, 1, 8]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([45], dtype=torch.int32, device="cuda")
    Q = _randn((1, 3, 64), F16, g)
    want = cc.paged_attention(Q, cache, table, lens)
    odd = [t.as_strided(t.shape, (1024, 64, 7, 1)) for t in (K, V)]
    assert torch.equal(cc.paged_attention(Q, cc.PagedCache(*odd), table, lens), want)
    q1 = Q.as_strided((1, 3, 64), (13, 64, 1))
    t1 = table.as_strided((1, 3), (-0, 1))
    assert torch.equal(cc.paged_attention(q1, cache, t1, lens), want)
    torch.cuda.synchronize()
    assert cc.device_error() == 0


def test_python_layer_keeps_no_references(clove_lib, cuda):
    """Calls, refused ones too, leave their arguments' and results' reference counts alone."""
    import sys
    for fn, args in _call_args(clove_lib).items():
        call = getattr(clove_lib, fn)
        before = {n: sys.getrefcount(x) for n, x in args.items()}
        for _ in range(50):
            r = call(**args)
            with pytest.raises((TypeError, ValueError)):
                call(**{**args, "page_table" if fn != "qk_norm_rope" else "positions": None})
        fresh = [x for x in (r if isinstance(r, tuple) else (r,)) if x is not None and not any(x is y for y in args.values())]
        assert all(sys.getrefcount(x) <= 5 for x in fresh)
        del r, fresh
        assert {n: sys.getrefcount(x) for n, x in args.items()} == before


# ---------------------------------------------------------------------------
# together, as a decode loop uses them
# ---------------------------------------------------------------------------
def test_decode_loop_agrees_with_prefill_attention(clove_lib, cuda):
    """Prefill a prompt into the cache, decode token by token (projection, norm + rotation +
    append, attention, captured once and replayed): every step's output equals the last row
    of flash_attention over the whole sequence so far, to the two kernels' rounding (each
    within 2^-10 of the 64-bit value relative to the row's norm: fp16 outputs, 2^-11, and
    flash_attention's fp16 weights, 2^-11)."""
    cc = clove_lib
    g = _gen(20)
    H, Hkv, D, hid, ps, prompt, steps = 8, 2, 128, 512, 16, 77, 5
    W = _randn((hid, (H + 2 * Hkv) * D), F16, g, hid ** -0.5)
    qw, kw = (1 + 0.1 * _randn((D,), F16, g) for _ in range(2))
    X = _randn((prompt + steps, hid), F16, g)
    table = cc.rope_table(256, D)
    pages = 8
    cache = cc.PagedCache(torch.full((pages, ps, Hkv, D), float("nan"), dtype=F16, device="cuda"),
                          torch.full((pages, ps, Hkv, D), float("nan"), dtype=F16, device="cuda"))
    page_table = torch.randperm(pages, device="cuda", generator=g)[:6].to(torch.int32)[None]
    slot = lambda t: page_table[0].long()[t // ps] * ps + t % ps

    def split(qkv):
        n = qkv.shape[0]
        return (qkv[:, :H * D].view(n, H, D), qkv[:, H * D:(H + Hkv) * D].view(n, Hkv, D),
                qkv[:, (H + Hkv) * D:].view(n, Hkv, D))

    pos = torch.arange(prompt, dtype=torch.int32, device="cuda")
    q, k, v = split(cc.gemm_fp16(X[:prompt].contiguous(), W))
    cc.qk_norm_rope(q, k, table, pos, qw, kw, V=v, cache=cache, slots=slot(pos.long()).to(torch.int32))
    x = torch.zeros(1, hid, dtype=F16, device="cuda")
    p1, s1, n1 = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(3))

    def step():
        q, k, v = split(cc.gemm_fp16(x, W))
        q, _ = cc.qk_norm_rope(q, k, table, p1, qw, kw, V=v, cache=cache, slots=s1)
        return cc.paged_attention(q, cache, page_table, n1)

    def load(t):
        x.copy_(X[t:t + 1])
        p1.fill_(t)
        s1.copy_(slot(torch.tensor([t], device="cuda")))
        n1.fill_(t + 1)

    load(prompt)
    step()  # warm-up; writes the same slot that the replay writes again
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = step()
    allq, allk, allv = split(cc.gemm_fp16(X, W))
    fq, fk = cc.qk_norm_rope(allq, allk, table, torch.arange(prompt + steps, dtype=torch.int32, device="cuda"), qw, kw)
    for t in range(prompt, prompt + steps):
        load(t)
        gr.replay()
        full = cc.flash_attention(fq[None, :t + 1].contiguous(), fk[None, :t + 1].contiguous(),
                                  allv[None, :t + 1].contiguous(), causal=True, layout="bshd")
        a, b = o[0].float(), full[0, t].float()
        assert torch.all((a - b).norm(dim=-1) <= 2 * 2.0 ** -10 * b.norm(dim=-1))
    assert cc.device_error() == 0


def test_decode_loop_with_eviction(clove_lib, cuda):
    """Attention with accumulated weights, eviction to the budget, attention over what is
    left: equal to 64-bit attention over the kept keys of each head."""
    cc = clove_lib
    g = _gen(21)
    Hkv, G, D, ps, budget = 2, 4, 64, 16, 100
    lens = [400, 60, 257]
    cache, table, sl = _pages(cc, lens, ps, Hkv, D, F16, "bshd", g, spare=22)
    used = set(table[table >= 0].tolist())
    free = [pg for pg in range(cache.num_pages) if pg not in used]
    dst = torch.tensor([free[i * 7:i * 7 + 7] for i in range(3)], dtype=torch.int32, device="cuda")
    w = torch.zeros((cache.num_pages, Hkv, ps), device="cuda")
    for _ in range(4):
        cc.paged_attention(_randn((3, Hkv * G, D), F16, g, 3.0), cache, table, sl, key_weights=w, accumulate=True)
    # Four steps of softmax weights: every head's sum over the keys is 4 G (n/16 + 64 roundings).
    for i, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        total = w[table[i].long()[t // ps], :, t % ps].double().sum(0)
        assert torch.all((total - 4 * G).abs() <= 4 * G * 1e-4)
    kept, new = cc.evict_cache(cache, w, table, sl, dst, budget, 16)
    Q = _randn((3, Hkv * G, D), F16, g, 2.0)
    O = cc.paged_attention(Q, cache, dst, new)
    for i, n in enumerate(lens):
        k, v = (ref.rows(c, "bshd", table[i].clamp(min=0), n, ps) for c in (cache.K, cache.V))
        for h in range(Hkv):
            idx = kept[i, h][:min(n, budget)].long()
            o, _, _, b_o, _, _ = ref.attention(Q[i, h * G:(h + 1) * G], k[idx, h:h + 1], v[idx, h:h + 1], D ** -0.5, 0)
            err = (O[i, h * G:(h + 1) * G].double() - o).abs()
            assert torch.all(err <= b_o + ref.half_step(o.abs() + b_o, F16))
    assert cc.device_error() == 0
