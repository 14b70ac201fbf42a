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
