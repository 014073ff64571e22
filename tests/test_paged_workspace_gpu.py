"""What paged attention keeps between calls: counters and partial results, per stream and
per graph (each test in a process of its own: both are the process's)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_SETUP = r"""
import torch
import clove_compute_b200 as cc
from cuda.bindings import runtime as rt
g = torch.Generator(device="cuda").manual_seed(1)
K, V = (torch.randn((400, 16, 2, 128), device="cuda", generator=g).half() for _ in range(2))
c = cc.PagedCache(K, V)
table = torch.randperm(400, device="cuda", generator=g)[:380].to(torch.int32).view(2, 190)
sl = torch.tensor([3000, 77], dtype=torch.int32, device="cuda")
Q = torch.randn((2, 8, 128), device="cuda", generator=g).half()
def ok(r):
    assert int(r[0]) == 0, r
    return r[1] if len(r) == 2 else r[1:]
"""


def _run(code, done):
    r = subprocess.run([sys.executable, "-c", _SETUP + code], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and done in r.stdout, (r.stdout[-500:], r.stderr[-2500:])


_MANY_CAPTURES = r"""
want = cc.paged_attention(Q, c, table, sl)
torch.cuda.synchronize()
memsets = []
graphs = []
for k in range(20):
    gr = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(gr):
        outs = [cc.paged_attention(Q, c, table, sl) for _ in range(80)]
    gr.instantiate()
    raw = rt.cudaGraph_t(gr.raw_cuda_graph())
    _, n = ok(rt.cudaGraphGetNodes(raw, 0))
    nodes, _ = ok(rt.cudaGraphGetNodes(raw, n))
    memsets.append(sum(ok(rt.cudaGraphNodeGetType(x)) == rt.cudaGraphNodeType.cudaGraphNodeTypeMemset for x in nodes))
    graphs.append((gr, outs))
for _ in range(2):
    for gr, outs in graphs:
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for (gr, outs), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for _, outs in graphs for o in outs)
assert cc.device_error() == 0
print("memsets", memsets)
assert sum(memsets) == 0, memsets
print("captures ok")
"""


def test_captured_models_share_counters_in_their_graph(cuda):
    """Twenty graphs of eighty calls, as of a model captured at twenty batch sizes: none
    needs counters of its own to be cleared, and their replays, side by side too, are right."""
    _run(_MANY_CAPTURES, "captures ok")


_FORKED = r"""
lens = [torch.tensor([3000 - 700 * i, 77 + i], dtype=torch.int32, device="cuda") for i in range(4)]
want = [cc.paged_attention(Q, c, table, n) for n in lens]
torch.cuda.synchronize()
gr = torch.cuda.CUDAGraph()
side = [torch.cuda.Stream() for _ in range(3)]
with torch.cuda.graph(gr):
    main = torch.cuda.current_stream()
    fork = torch.cuda.Event()
    fork.record(main)
    outs = []
    for rep in range(5):
        outs.append((0, cc.paged_attention(Q, c, table, lens[0])))
        for i, s in enumerate(side):
            s.wait_event(fork)
            outs.append((i + 1, cc.paged_attention(Q, c, table, lens[i + 1], stream=s)))
    for again in range(3):  # main goes on after the others, they beside it
        for s in side:
            join = torch.cuda.Event()
            join.record(s)
            main.wait_event(join)
        if again < 2:
            outs.append((0, cc.paged_attention(Q, c, table, lens[0])))
            for i, s in enumerate(side):
                outs.append((i + 1, cc.paged_attention(Q, c, table, lens[i + 1], stream=s)))
for _ in range(20):
    for _, o in outs:
        o.zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)
assert cc.device_error() == 0
print("forked ok")
"""


def test_streams_forked_in_one_capture(cuda):
    """Calls on four streams of one capture run beside each other when it is replayed."""
    _run(_FORKED, "forked ok")


_CAPTURE_BESIDE_EAGER = r"""
import sys, threading
cold, default = sys.argv[1] != "warm", sys.argv[1] == "default"
O = torch.empty_like(Q)
w = torch.zeros((400, 2, 16), device="cuda")
mine, theirs = torch.cuda.Stream(), torch.cuda.Stream()
want = None
if not cold:
    want = cc.paged_attention(Q, c, table, sl)
x = torch.zeros(1 << 20, device="cuda")
rope = cc.rope_table(4000, 128)
spare, w2 = cc.PagedCache(K.clone(), V.clone()), torch.zeros((400, 2, 16), device="cuda")
small, fresh = (torch.tensor([[a], [a + 1]], dtype=torch.int32, device="cuda") for a in (0, 2))
few = torch.tensor([9, 3], dtype=torch.int32, device="cuda")
k2 = Q[:, :2].contiguous()
qo, ko = torch.empty_like(Q), torch.empty_like(k2)
with torch.cuda.stream(theirs):  # (room for torch's allocator, which may not ask for more beside a capture)
    room = torch.empty(1000, device="cuda")
torch.cuda.synchronize()
bad = []
def eager():
    try:
        torch.cuda.set_device(0)
        for s in (None, None) if default else (theirs.cuda_stream, theirs.cuda_stream):
            cc.paged_attention(Q, c, table, sl, O=O, stream=s)
            cc.paged_attention(Q, c, table, sl, O=O, key_weights=w, stream=s)
            cc.qk_norm_rope(Q, k2, rope, sl, Q_out=qo, K_out=ko, stream=s)
            cc.evict_cache(spare, w2, small, few, fresh, 4, 1, stream=s)
    except Exception as e:
        bad.append(e)
gr = torch.cuda.CUDAGraph()
with torch.cuda.graph(gr, stream=mine):
    x.add_(1)
    t = threading.Thread(target=eager)
    t.start()
    t.join()
    y = cc.paged_attention(Q, c, table, sl)
torch.cuda.synchronize()
assert not bad, bad
gr.replay()
torch.cuda.synchronize()
want = cc.paged_attention(Q, c, table, sl) if want is None else want
assert torch.equal(y, want) and torch.equal(O, want)
assert cc.device_error() == 0
print("beside ok")
"""


@pytest.mark.parametrize("start", ["cold", "warm", "default"])
def test_eager_calls_while_another_thread_captures(cuda, start):
    """The eager calls of one thread, the process's first ones too, on the default stream or
    another, and a capture under way in another thread do not disturb each other."""
    r = subprocess.run([sys.executable, "-c", _SETUP + _CAPTURE_BESIDE_EAGER, start], cwd=ROOT, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0 and "beside ok" in r.stdout, (r.stdout[-500:], r.stderr[-2500:])


_STREAMS = r"""
want = cc.paged_attention(Q, c, table, sl)
O = torch.empty_like(Q)
torch.cuda.synchronize()
free0 = torch.cuda.mem_get_info()[0]
for rep in range(3):
    for k in range(100):
        s = ok(rt.cudaStreamCreate())
        for _ in range(2):
            O.zero_()
            torch.cuda.synchronize()
            cc.paged_attention(Q, c, table, sl, O=O, stream=int(s))
        ok(rt.cudaStreamSynchronize(s))
        assert torch.equal(O, want)
        ok(rt.cudaStreamDestroy(s))
torch.cuda.synchronize()
held = free0 - torch.cuda.mem_get_info()[0]
print("held", held >> 20, "MB")
assert held <= 160 << 20, held
outs = [torch.empty_like(Q) for _ in range(40)]
streams = [ok(rt.cudaStreamCreate()) for _ in outs]
for rep in range(20):  # more at a time than workspaces are kept
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(2):
        for o, s in zip(outs, streams):
            cc.paged_attention(Q, c, table, sl, O=o, stream=int(s))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
assert cc.device_error() == 0
print("streams ok")
"""


def test_workspaces_of_gone_streams_are_taken_over(cuda):
    """Hundreds of streams, one after the other: what is kept stays bounded (16 workspaces of
    8 MB, and the pool's granularity), and results right; so with 40 in use at once."""
    _run(_STREAMS, "streams ok")


_SCRATCH = r"""
wide = torch.zeros((64, 1 << 14), dtype=torch.int32, device="cuda")
wide[:, :2] = torch.arange(128, dtype=torch.int32, device="cuda").view(64, 2)
lens = torch.full((64,), 20, dtype=torch.int32, device="cuda")
q = torch.randn((64, 32, 128), device="cuda", generator=g).half()
w, w2 = torch.zeros((400, 2, 16), device="cuda"), torch.zeros((400, 2, 16), device="cuda")
want = cc.paged_attention(q, c, wide[:, :2], lens, key_weights=w2)
torch.cuda.synchronize()
free0 = torch.cuda.mem_get_info()[0]
got = cc.paged_attention(q, c, wide, lens, key_weights=w)
torch.cuda.synchronize()
torch.cuda.synchronize()
held = free0 - torch.cuda.mem_get_info()[0]
print("held", held >> 20, "MB")
assert torch.equal(got, want) and torch.equal(w, w2)
assert held <= 512 << 20, held
print("scratch ok")
"""


def test_large_scratch_goes_back(cuda):
    """Key weights over wide page tables (2 GB of scratch): what the library's pool holds on
    to afterwards is bounded."""
    _run(_SCRATCH, "scratch ok")
