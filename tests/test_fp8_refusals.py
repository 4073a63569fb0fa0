"""What the 8-bit operators refuse, on the CPU: no kernel is launched, and no pointer is followed."""
import itertools

import pytest

from convnn_b200 import _capi
from test_fp8_host import P, linear, norm8, quantize


def shared(row, block, rows, blocks):
    at = [r * row + b * block for r in range(rows) for b in range(blocks)]
    return len(set(at)) < len(at)


@pytest.mark.parametrize("rows,blocks", [(1, 1), (1, 3), (4, 1), (2, 2), (3, 4), (5, 2)])
def test_scales_that_would_be_written_over_one_another(rows, blocks):
    D = 128 * blocks - 5
    for row, block in itertools.product(range(1, 8), repeat=2):
        calls = (norm8(row=row, block=block, rows=rows, D=D, ldx=D, ldq=D),
                 quantize(row=row, block=block, rows=rows, D=D, ldx=D, ldq=D),
                 quantize(row=row, block=block, rows=128 * rows - 7, D=D, ldx=D, ldq=D, block_rows=128),
                 linear(so=P, sor=row, sob=block, M=rows, N=D, ldo=D))
        for status in calls:
            assert (status == _capi.E_INVALID) == shared(row, block, rows, blocks), (row, block, status)


def test_strides_whose_products_pass_64_bits():
    big = 1 << 62
    for row, block, bad in ((big, 1, False), (1, big, False), (big, big, True), (big, big + 1, False)):
        assert (norm8(row=row, block=block, rows=3, D=300, ldx=300, ldq=300) == _capi.E_INVALID) == bad
