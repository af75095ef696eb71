"""What a kernel that touches another CTA's shared memory has to do, read from the sources (no device): the memory is there from when that CTA runs, so the cluster's CTAs wait for one another
first (an arrival at the kernel's start costs nothing by the time something is sent)."""
import re

import pytest
from test_overlap_sources_cpu import _kernels, _sources

SHARING = {name: code for text in _sources().values() for name, code in _kernels(text) if "map_shared_rank" in code}


def test_there_are_such_kernels():
    assert {"sample_rows_kernel", "seq_attention_decode_kernel", "seq_attention_decode_mma_kernel"} <= set(SHARING)


@pytest.mark.parametrize("kernel", sorted(SHARING))
def test_all_ctas_run_before_one_touches_anothers_memory(kernel):
    code = SHARING[kernel]
    before = code[:code.index("map_shared_rank")]
    assert re.search(r"barrier_wait\(\)|barrier\.cluster\.wait|cluster\.sync\(\)", before), "shared memory of a CTA that may not have started"
