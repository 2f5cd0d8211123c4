"""Properties of the kernels' sources that no run can show: what a compiler may or may not reorder."""

import os
import re

_CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "optimizers_b200", "ops", "csrc")


def _source(name):
    text = open(os.path.join(_CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_loaded_tensor_memory_is_read_behind_its_wait_only():
    """The registers of an asynchronous load are valid after the wait.  The wait passes a gate through, so each statement that reads
    such registers has to take that gate too: a separate one (the move that forms a pair, say) could be scheduled ahead of the wait."""
    lines = [line for line in _source("fp8_kernels.cu").splitlines() if re.search(r"\bv\[c & 1\]", line)]
    issued = [line for line in lines if "_issue(" in line]
    read = [line for line in lines if "_issue(" not in line]
    assert len(issued) == 2 and len(read) == 2
    for line in read:
        assert re.search(r"(fma2|mul2)_loaded\(v\[c & 1\]\[[^\]]*\], v\[c & 1\]\[[^\]]*\], by\b", line), line
    for name in ("mul2_loaded", "fma2_loaded"):
        body = re.search(name + r"\(uint32_t lo, uint32_t hi, uint64_t gate[^{]*\{(.*?)\n\}", _source("ptx.cuh"), re.S).group(1)
        assert body.count("asm") == 1 and re.search(r'"r"\(lo\), "r"\(hi\), "l"\(gate\)', body)
