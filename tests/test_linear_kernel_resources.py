"""What the built library's kernel descriptors say of linear attention, the draft verification and the page copies."""
import os
import re

import pytest

from test_kernel_resources import READELF, kernel_scratch_bytes


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_states_stay_in_registers(tmp_path):
    """A reload from scratch memory would wait for the chunk in flight as well."""
    scratch = kernel_scratch_bytes(tmp_path)
    kernels = {k: v for k, v in scratch.items() if re.search("linear_step|linear_chunk|linear_scan|draft_|kv_copy", k)}
    assert len([k for k in kernels if "linear_chunk" in k]) == 24 and len([k for k in kernels if "linear_step" in k]) >= 8, sorted(kernels)
    assert {k: v for k, v in kernels.items() if v} == {}
