"""CPU suite: what the readout kernels' sources must not hold, and what their entry points refuse."""

import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kernels_that_begin_early_load_nothing_by_the_read_only_path():
    """Data loaded that way must not change while a kernel lives, and these kernels are set up while the one before them still writes."""
    sources = glob.glob(os.path.join(ROOT, "graphtsetlinmachine_b200", "csrc", "gtm_readout*"))
    assert len(sources) >= 7
    for path in sources:
        code = re.sub(r"//[^\n]*", "", open(path).read())
        assert not re.search(r"__ldg|__restrict__|ld\.global\.nc|ld\.global\.[a-z.]*nc", code), path
        # and every kernel waits for the one before it
        kernels = re.findall(r"__global__ void[^{;]*\)\s*\n\{(.*?)\n\}", code, flags=re.S)
        assert all("wait_for_previous();" in k for k in kernels), path
