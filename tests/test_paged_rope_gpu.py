"""Norm + rotation + append through both kernels (1 streaming, 2 direct) where
tests/test_paged_gpu.py runs one of them, and what must be written where."""
import pytest
import torch

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(params=[1, 2])
def path(request, clove_lib):
    clove_lib.set_dispatch_override(request.param)
    yield request.param
    clove_lib.set_dispatch_override(0)


def _fused(T, H, Hkv, D, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (1.5 * torch.randn((T, (H + 2 * Hkv) * D), device="cuda", generator=g)).to(dtype)
    parts = (qkv[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
    qw, kw = ((1 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dtype) for _ in range(2))
    pos = torch.randint(0, 5000, (T,), device="cuda", generator=g, dtype=torch.int32)
    return qkv, *parts, qw, kw, pos


@pytest.mark.parametrize("T,H,Hkv,D,R,dtype,interleaved", [
    (1, 4, 2, 128, 128, F16, False), (50, 6, 2, 64, 32, BF16, True), (3001, 32, 8, 128, 128, F16, False),
    (333, 96, 16, 128, 112, BF16, True),   # a token's rows in two pieces
    (2000, 100, 33, 256, 192, F16, False),  # in six
])
def test_in_place(clove_lib, cuda, path, T, H, Hkv, D, R, dtype, interleaved):
    """Q and K turned where they stand, blocks of the projection's rows: as into buffers of
    their own, the values' block untouched, and K and V in the cache."""
    cc = clove_lib
    qkv, Q, K, V, qw, kw, pos = _fused(T, H, Hkv, D, dtype, T + D)
    table = cc.rope_table(5000, R)
    want_q, want_k = cc.qk_norm_rope(Q, K, table, pos, qw, kw, interleaved=interleaved)
    v = V.clone()
    caches = []
    slots = torch.randperm(-(-T // 16) * 16, device="cuda")[:T].to(torch.int32)
    for inside in (False, True):
        c = cc.PagedCache(*(torch.full((-(-T // 16), 16, Hkv, D), 5.0, dtype=dtype, device="cuda") for _ in range(2)))
        kw_args = dict(Q_out=Q, K_out=K) if inside else {}
        cc.qk_norm_rope(Q, K, table, pos, qw, kw, interleaved=interleaved, V=V, cache=c, slots=slots, **kw_args)
        caches.append(c)
    torch.cuda.synchronize()
    assert cc.device_error() == 0
    assert torch.equal(Q, want_q) and torch.equal(K, want_k) and torch.equal(V, v)
    assert torch.equal(caches[0].K, caches[1].K) and torch.equal(caches[0].V, caches[1].V)
    assert torch.equal(caches[0].K.view(-1, Hkv, D)[slots.long()], want_k)
    assert torch.equal(caches[0].V.view(-1, Hkv, D)[slots.long()], v)


def test_extreme_rows(clove_lib, cuda, path):
    """Zero rows stay zero, the largest fp16 values do not overflow in the sum of squares,
    NaN stays in its row."""
    D = 128
    Q = torch.zeros(300, 2, D, dtype=F16, device="cuda")
    Q[1::3] = 65504.0
    Q[2::3, 0, 5] = float("nan")
    K = Q[:, :1].contiguous()
    w = torch.ones(D, dtype=F16, device="cuda")
    q, k = clove_lib.qk_norm_rope(Q, K, clove_lib.rope_table(4, D), torch.zeros(300, dtype=torch.int32, device="cuda"), w, w)
    assert torch.all(q[0::3] == 0) and torch.all(q[1::3] == 1) and torch.isnan(q[2::3, 0]).all() and torch.all(q[2::3, 1] == 0)
    assert torch.all(k[0::3] == 0) and torch.all(k[1::3] == 1) and torch.isnan(k[2::3]).all()


@pytest.mark.parametrize("name,value", [("positions", 5000), ("positions", 2 ** 31 - 1), ("positions", -1),
                                        ("slots", "end"), ("slots", 2 ** 31 - 1), ("slots", -1), ("slots", -2 ** 31)])
def test_a_bad_index_costs_its_own_token_only(clove_lib, cuda, path, name, value):
    """A position that is padding or outside the table: nothing of the token is written; a
    slot that is negative or outside the cache: its keys and values are not stored. Every
    other row of every output is, and nothing beside them."""
    cc = clove_lib
    T, H, Hkv, D, bad = 23, 4, 2, 128, 7
    _, Q, K, V, qw, kw, pos = _fused(T, H, Hkv, D, F16, 9)
    table = cc.rope_table(5000, D)
    slots = torch.randperm(64, device="cuda")[:T].to(torch.int32)
    want_q, want_k = cc.qk_norm_rope(Q, K, table, pos, qw, kw)
    index = {"positions": pos.clone(), "slots": slots.clone()}
    index[name][bad] = 64 if value == "end" else value
    c = cc.PagedCache(*(torch.full((4, 16, Hkv, D), 5.0, dtype=F16, device="cuda") for _ in range(2)))
    q, k = torch.full_like(want_q, 9.0), torch.full_like(want_k, 9.0)
    cc.qk_norm_rope(Q, K, table, index["positions"], qw, kw, V=V, cache=c, slots=index["slots"], Q_out=q, K_out=k)
    assert cc.device_error() == (0 if value != "end" and value < 0 else 3)
    exp_k, exp_v = (torch.full((64, Hkv, D), 5.0, dtype=F16, device="cuda") for _ in range(2))
    live = torch.tensor([t for t in range(T) if t != bad], device="cuda")
    exp_k[slots.long()[live]], exp_v[slots.long()[live]] = want_k[live], V[live]
    if name == "positions":
        want_q[bad], want_k[bad] = 9.0, 9.0
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(c.K.view(64, Hkv, D), exp_k) and torch.equal(c.V.view(64, Hkv, D), exp_v)
