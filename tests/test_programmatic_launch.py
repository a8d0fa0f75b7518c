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


def kernels():
    for name in FILES:
        for body in re.split(r"__global__", code(name))[1:]:
            yield re.search(r"\b(k_\w+)\s*\(", body).group(1), body


@pytest.mark.parametrize("kernel", dict(kernels()))
def test_waits_before_it_lets_the_next_one_start(kernel):
    """Every kernel waits for the one before it, whatever its arguments say, and only then lets the next one start: what it
    reads is visible to the grid that waits, and the next one may count on all kernels before this one."""
    lines = [x.strip() for x in dict(kernels())[kernel].splitlines()]
    wait, trigger = lines.index("pdl_wait();"), lines.index("pdl_trigger();")
    assert wait < trigger
    before = " ".join(lines[:wait])
    assert "return" not in before and not re.search(r"\ba\.(q|kpool|vpool|table|q_start|ctx_len|seq_slot|part|jobs|out)\b", before)
