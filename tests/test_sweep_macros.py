"""CPU tests: the kernel sources take the macro settings of the committed prefill sweep that the
library as a whole can be built with, and stay safe under them."""
import os
import subprocess
import sys

import pytest

from inkling_fa4 import sweep

sys.path.insert(0, sweep._PKG_ROOT)
import build  # noqa: E402


def compiled(source, macro, *flags):
    got = subprocess.run([build.HIPCC, *build.HIP_FLAGS, f"-D{macro}", "-x", "hip", "--cuda-device-only",
                          *flags, os.path.join(build.CSRC, source)], capture_output=True, text=True)
    assert got.returncode == 0, got.stderr[-2000:]
    return got.stdout


@pytest.mark.parametrize("source", ["prefill_fwd.hip", "prefill_paged.hip", "prefill_paged_fp8.hip"])
@pytest.mark.parametrize("macro", ["IFA4_DMA2=0", "IFA4_BIAS_LDS=0"])
def test_prefill_sources_take_the_macro(source, macro):
    assert source in build.LIB_SOURCES
    compiled(source, macro, "-fsyntax-only")


@pytest.mark.parametrize("source", ["prefill_paged.hip", "prefill_paged_fp8.hip"])
def test_paged_dmas_keep_their_hazard_cover(source):
    """A DMA's resource comes from v_readlane right before it, which takes five wait states:
    s_nop 4, also where the knob takes them off the DMAs of contiguous rows."""
    dma = "buffer_load_dwordx4 $0, $1, 0 offen lds"
    unoptimised = ("-S", "-emit-llvm", "-Xclang", "-disable-llvm-passes", "-o", "-")
    ir = compiled(source, "IFA4_DMA_COVER_EACH=0", *unoptimised)
    covered = ir.count('asm sideeffect "s_nop 4\\0A\\09' + dma)
    assert covered > 0 and ir.count(dma) == covered
