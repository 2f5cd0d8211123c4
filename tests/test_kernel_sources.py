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


def test_split_products_judge_their_partial_sums_by_the_flags_of_all_ranks():
    """Partial sums lie where loads go.  In a CTA that gave up a wait a load may still be under way and write over them, the NaN that
    marks a given-up result included, so the CTAs that add them up look at each other's flag, after the barrier and before they store."""
    source = _source("fp8_kernels.cu")
    join = source[source.index("float4* mine = reinterpret_cast<float4*>(smem);") :]
    join = join[: join.index("continue;")]
    at = [join.index(part) for part in ("cluster.sync();", "map_shared_rank(const_cast<int*>(abort_flag), min(lane, p.splits - 1))", "map_shared_rank(mine, r)", "if (!ok) sum.x", "store_quad")]
    assert at == sorted(at)
    assert "if (!ok && lane == 0) *p.status = 1;" in source[source.index("float4* mine") :]
