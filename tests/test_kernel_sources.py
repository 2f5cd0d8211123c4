"""Properties of the kernels' sources that no run on a GPU can show: what a compiler may reorder, what follows a wait that gave up or a
check that failed."""

import os
import re
import subprocess

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


_ONCE = """
#include "once.h"
#include <stdexcept>
#include <utility>
int main() {
  ob200::Once<std::pair<int, int>> once;
  int runs = 0, thrown = 0;
  bool fails = true;
  auto call = [&](int key) {
    try {
      once({key, 0}, [&] {
        ++runs;
        if (fails) throw std::runtime_error("check");
      });
    } catch (const std::runtime_error&) { ++thrown; }
  };
  call(1);
  call(1);  // the check failed: it is made again, and fails again
  if (runs != 2 || thrown != 2) return 1;
  fails = false;
  call(1);
  call(1);
  call(2);
  return runs == 4 && thrown == 2 ? 0 : 2;
}
"""


def test_a_check_that_failed_is_made_again(tmp_path):
    """A kernel that moves registers between its warps waits for ever if it is launched with fewer than it was written for: every launch
    has to pass the check until one has passed it."""
    (tmp_path / "once.cpp").write_text(_ONCE)
    subprocess.run(["g++", "-std=c++17", "-I", _CSRC, str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once"), "-pthread"], check=True)
    assert subprocess.run([str(tmp_path / "once")]).returncode == 0
    body = _source("fp8_kernels.cu")
    body = body[body.index("void prepare_product(") : body.index("CUtensorMap result_map(")]
    assert "once({kernel, device}" in body and body.index("once({kernel, device}") < body.index("attr.numRegs >= launch_regs")
