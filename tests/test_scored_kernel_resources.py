"""What the built library's kernel descriptors say of the scored attention, the cache read and the merge."""
import os
import re

import pytest

from test_kernel_resources import READELF, kernel_scratch_bytes


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_scored_kernels_keep_their_sums_in_registers(tmp_path):
    """Decode, join, read and merge keep everything there; the chunk kernel over quantised rows, with 128 sums and 64 query registers a
    lane, puts up to 24 words into scratch memory (a version that puts sums there has ten times as many)."""
    scratch = kernel_scratch_bytes(tmp_path)
    kernels = {k: v for k, v in scratch.items() if re.search("scored_decode|scored_join|kv_read|attention_merge", k)}
    assert len(kernels) >= 30, sorted(kernels)
    assert {k: v for k, v in kernels.items() if v} == {}
    chunks = {k: v for k, v in scratch.items() if "scored_chunk_kernel" in k}
    assert len(chunks) == 20, sorted(chunks)
    assert {k: v for k, v in chunks.items() if v > 96} == {}
    assert {k: v for k, v in chunks.items() if v and re.search("ILi[01]E|Li[01]ELi", k)} == {}
