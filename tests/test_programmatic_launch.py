"""Kernels that are launched while the one before them still runs (launch.h): what their source may not do."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inference-project_b200", "csrc")
FILES = ["k_attn_chunk.cuh", "k_attn_chunk_rows.cuh", "k_attn_chunk_tc.cuh", "k_kv_pages.cuh", "k_qk_norm_rope.cuh"]


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", FILES)
def test_no_loads_through_the_read_only_path(name):
    """Such loads are for memory that nothing writes while the kernel exists, and it exists while the one before it
    writes its inputs."""
    assert not re.findall(r"__ldg|ld\.global\.nc|__restrict__", code(name))
