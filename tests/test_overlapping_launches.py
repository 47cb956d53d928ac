"""Kernels that start while their predecessor still runs read what it writes by ordinary loads. CPU only: a look at the sources.

The read-only path (`const T *__restrict__` arguments, `__ldg`, `ld.global.nc`) is defined for data that nobody writes while the kernel
lives, and these kernels live before their wait for the predecessor: rope writes append's rows, extend writes everybody's starts."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "yscv_b200" / "csrc"


@pytest.mark.parametrize("name", ["rope.cu", "kv_block.cu", "kv_block_attention.cu", "kv_block_prompt.cu", "kv_pages.cu"])
def test_paged_cache_kernels_do_not_take_the_read_only_path(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert "pdl_wait();" in text
    assert not re.findall(r"const\s+\w+\s*\*\s*__restrict__|__ldg\s*\(|\.nc\b", text)
