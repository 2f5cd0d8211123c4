"""Every variant of the 8-bit product: tile widths, pairs of CTAs, K cut among a cluster, results by TMA or by plain stores."""

import math
import random

import pytest
import torch

from optimizers_b200.models import fp8
from optimizers_b200.ops import build
from test_gpu_fp8 import BF16, F32, SIZES, _product_case, _x

# Sizes of the variants that test_gpu_fp8's do not reach: K cut in two and in eight at both widths, and results by TMA from pairs with
# 256 columns, several tiles a pair, ragged in both directions (a scale per row of B: the same products with plain stores).
MORE = [
    (40, 72, 650), (3, 5, 642), (70, 104, 15000), (1, 1, 16384), (130, 4984, 650), (1, 4806, 1441), (129, 1160, 11100), (2, 1161, 11073),
    (4096, 4104, 300), (4100, 4128, 200), (9533, 136, 130), (131, 9832, 260), (257, 4784, 130),
]
SMS = 148


def _variants(sizes):
    plan = build.load().fp8_plan
    return {(column, *plan(*size, column, SMS)) for size in sizes for column in (False, True)}


@pytest.mark.skipif(not build.available(), reason="the extension is not built")
def test_the_sizes_reach_every_variant_that_any_size_reaches():
    rng = random.Random(0)
    anywhere = [tuple(int(math.exp(rng.uniform(0, math.log(20000)))) for _ in range(3)) for _ in range(20000)]
    assert _variants(anywhere) == _variants(SIZES + MORE)
    plan = build.load().fp8_plan
    # results that leave by TMA (bf16, a scale per 128 rows of B, columns in eights), from pairs with several tiles each
    assert any(plan(M, N, K, False, SMS) == (256, 1) and N % 8 == 0 and -(-M // 256) * -(-N // 256) > 2 * (SMS // 2) for M, N, K in MORE)


@pytest.mark.gpu
@pytest.mark.parametrize("size", MORE)
@pytest.mark.parametrize("column", [False, True])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products(size, column, out):
    _product_case(*size, column, out, addend=False)
    fp8.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [(40, 72, 650), (70, 104, 15000), (130, 4984, 650), (129, 1160, 11100), (9533, 136, 130)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products_with_an_addend(size, out):
    _product_case(*size, False, out, addend=True)


# M * N is a multiple of 256, so that a result ends where its block of memory ends.
GUARDED = [(1000, 1056, 300), (1152, 1002, 500), (4104, 4128, 300), (264, 4000, 650), (264, 2080, 11100), (264, 1056, 16384)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", GUARDED)
@pytest.mark.parametrize("column", [False, True])
@pytest.mark.parametrize("out", [F32, BF16])
def test_results_keep_to_their_memory(size, column, out):
    """The memory right before and right behind a result holds a pattern, which has to survive."""
    M, N, K = size
    a, b = fp8.quantize_rows(_x(M, K, F32)), (fp8.quantize_rows if column else fp8.quantize_weight)(_x(N, K, F32, 1))
    status = fp8._status_of(a.data.device)
    need, pattern = M * N * out.itemsize, 0x5A
    product = lambda: build.load().fp8_matmul(a.data.view(torch.uint8), a.scale, b.data.view(torch.uint8), b.scale, column, out == BF16, None, status)  # noqa: E731
    memory = lambda n: torch.full((n,), pattern, dtype=torch.uint8, device="cuda")  # noqa: E731
    with torch.cuda.use_mem_pool(torch.cuda.MemPool()):
        if need > 1 << 20:  # blocks are cut from the front of what was freed, so that nothing fills them again
            side = 4 << 20
            whole = memory(need + 2 * side)
            start = whole.data_ptr()
            del whole
            front = torch.empty(side, dtype=torch.uint8, device="cuda")
            got = product()
            back = torch.empty(side, dtype=torch.uint8, device="cuda")
        else:  # small blocks lie side by side from the start; the result takes the place of the middle one
            side = 256 << 10
            front, middle, back = memory(side), memory(need), memory(side)
            start = front.data_ptr()
            del middle
            got = product()
    assert (front.data_ptr(), got.data_ptr(), back.data_ptr()) == (start, start + side, start + side + need)
    assert bool((front == pattern).all()) and bool((back == pattern).all())
    assert got.isfinite().all()


@pytest.mark.gpu
def test_variants_repeat_to_the_bit():
    for size in MORE:
        for column in (False, True):
            first = _product_case(*size, column, BF16, False)
            assert torch.equal(first, _product_case(*size, column, BF16, False))
