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
