"""Register plans of the paged-cache kernels, from ptxas's report on the CPU: the attention
kernels run two CTAs of 128 threads per SM (at most 255 registers; one for head_dim 256 in
16 bits), the eviction's selection one CTA of 1024 (at most 64), the streaming norm + rotation
two of 128, and none of them spills."""
import concurrent.futures as cf
import os

import pytest

from tests.test_register_plans_cpu import KERNELS, _entries, _ptxas, _report


@pytest.fixture(scope="module")
def reports(tmp_path_factory):
    tmp = str(tmp_path_factory.mktemp("ptxas"))
    srcs = [os.path.join(KERNELS, f) for f in
            ("paged_attention_f16.cu", "paged_attention_bf16.cu", "evict_cache.cu", "qk_norm_rope.cu")]
    rep = {}
    with cf.ThreadPoolExecutor(len(srcs)) as ex:
        for log in ex.map(lambda s: _ptxas(s, tmp), srcs):
            rep.update(_report(log))
    return rep


@pytest.mark.parametrize("pattern,count,max_regs", [
    (r"paged_attention_kernel", 20, 255),
    (r"evict_select_kernel", 2, 64),
    (r"evict_copy_kernel", 4, 85),  # three CTAs of 256 threads
    (r"qk_norm_rope_kernel", 24, 128),
    (r"qk_norm_rope_stream_kernel", 24, 255),
])
def test_paged_register_plans(reports, pattern, count, max_regs):
    hits = _entries(reports, pattern)
    assert len(hits) == count, sorted(hits)
    for name, (regs, spill) in hits.items():
        assert regs is not None and regs <= max_regs, (name, regs)
        assert spill == (0, 0), (name, spill)
