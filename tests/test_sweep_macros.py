"""CPU test: the kernel sources take the macro settings of the committed prefill sweep that the
library as a whole can be built with."""
import os
import subprocess
import sys

import pytest

from inkling_fa4 import sweep

sys.path.insert(0, sweep._PKG_ROOT)
import build  # noqa: E402


@pytest.mark.parametrize("source", ["prefill_fwd.hip", "prefill_paged.hip", "prefill_paged_fp8.hip"])
@pytest.mark.parametrize("macro", ["IFA4_DMA2=0", "IFA4_BIAS_LDS=0"])
def test_prefill_sources_take_the_macro(source, macro):
    assert source in build.LIB_SOURCES
    got = subprocess.run([build.HIPCC, *build.HIP_FLAGS, f"-D{macro}", "-x", "hip", "--cuda-device-only",
                          "-fsyntax-only", os.path.join(build.CSRC, source)], capture_output=True, text=True)
    assert got.returncode == 0, got.stderr[-2000:]
