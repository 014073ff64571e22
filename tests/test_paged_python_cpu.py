"""The Python layer of the paged-cache operators without a GPU: refusals that come before
any device work."""
import pytest
import torch

import clove_compute_b200 as cc
from clove_compute_b200 import paged


def test_stream_of_another_gpu_refused(monkeypatch):
    """A stream that is not on the tensors' GPU would take the launch, with their addresses,
    to its own GPU."""
    class Stream:
        def __init__(self, index):
            self.device, self.cuda_stream = torch.device("cuda", index), 1234

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    called = []
    with pytest.raises(ValueError, match="GPU 0"):
        paged._elsewhere(lambda *a: called.append(a), 0, Stream(1), "Q")
    assert not called


_NOT_A_CACHE = r"""
import torch
from clove_compute_b200 import paged
fast = paged._load()
class T:
    dtype, shape = torch.float16, (1, 2, 128)
    def get_device(self): return 0
    def data_ptr(self): return 4096
    def stride(self): return (256, 128, 1)
for wrong in ((1, 0), (16, 0, 0), (None, 0), 7, "text"):
    for call in (lambda: fast.paged_attention(T(), wrong, T(), T(), None, 0, None, None, False, None, 0),
                 lambda: fast.evict_cache(wrong, T(), T(), T(), T(), 1, 0, 0)):
        try:
            call()
        except TypeError as e:
            assert "PagedCache" in str(e), e
        else:
            raise SystemExit(f"{wrong!r} was taken for a cache")
print("refused")
"""


def test_only_a_paged_cache_is_followed():
    """A tuple of two numbers in the cache's place is refused, not read as an address (run in
    a process of its own: it used to end the interpreter)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _NOT_A_CACHE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "refused", (r.returncode, r.stdout, r.stderr[-1500:])


def test_torchs_own_refusals_are_passed_on():
    """A tensor without storage (under vmap, a transform or tracing) is refused with torch's
    reason, what is no tensor as such."""
    q = torch.zeros(2, 3, 4, 128, dtype=torch.float16)
    for call in (lambda x: cc.paged_attention(x, None, None, None), lambda x: cc.qk_norm_rope(x, x, None, None)):
        with pytest.raises(RuntimeError, match="storage"):
            torch.vmap(call)(q)
        for wrong in ("text", None, 3, [1.0]):
            with pytest.raises(TypeError, match="Q must be a torch.Tensor"):
                call(wrong)


@pytest.mark.parametrize("theta", [0.0, -1.0, float("nan"), float("inf")])
def test_rotation_base_out_of_range(theta):
    """A base that is not positive and finite gives NaN angles."""
    with pytest.raises(ValueError):
        cc.rope_table(4, 64, theta, device="cpu")
