"""How the kernels' launches are written, from the source files alone.  No GPU is touched."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "okc_muse_kernels_b200", "csrc")


def test_shared_memory_limits_are_constants_of_the_kernels():
    """The limit belongs to a kernel on its device: set to a call's own size, it can be lowered by a call of another thread
    before this call's launch."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            for limit in re.findall(r"cudaFuncAttributeMaxDynamicSharedMemorySize,\s*(.+?)\);", f.read()):
                assert re.fullmatch(r"k[A-Z]\w*", limit), f"{name}: {limit}"
                found += 1
    assert found >= 10
