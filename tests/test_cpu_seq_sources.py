"""Rules of the packed and int8-cache kernels that no result shows until they fail: checked on their sources."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "l0llm_b200" / "csrc"
FILES = ["attention_packed.cu", "attention_packed_f32.cu", "attention_q8.cu", "kv_q8.cu", "packed.cuh", "packed_attn.cuh"]


def code_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", FILES)
def test_nothing_is_read_through_the_read_only_path(name):
    # Rows, codes, scales, starts, positions and lengths may come from the kernel before, which programmatic dependent
    # launch lets run while this one starts; read-only loads are for memory that stays as it is for a kernel's whole life.
    assert not re.search(r"__ldg|ld_stream|\.nc\b", code_of(name))


def test_the_row_threads_barrier_orders_tensor_memory():
    # f32 queries: two threads of different warps share a row, and each overwrites scores that the other has read. A
    # barrier between threads orders tensor-memory accesses only between a fence before the arrival and one behind the wait.
    body = re.search(r"auto rows_sync = \[&\]\(\) \{(.*?)\};", code_of("attention_packed_f32.cu"), re.S).group(1)
    calls = re.findall(r"(\w+)\(", body)
    assert calls == ["tc_before", "bar_arrive", "wait_warp", "tc_after"]
