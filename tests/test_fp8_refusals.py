"""What the 8-bit operators refuse, on the CPU: no kernel is launched, and no pointer is followed."""
import itertools

import pytest
import torch

from convnn_b200 import _capi, ops
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


@pytest.fixture
def on_any_device(monkeypatch):
    """The Python form up to the launch on tensors without storage; -> what was launched."""
    launched = []
    monkeypatch.setattr(ops, "_device_of", lambda *tensors: 0)
    monkeypatch.setattr(ops, "_launch", lambda index, fn, *args: launched.append(args))
    return launched


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def meta8(rows, K, block_rows=1):
    return meta(rows, K, dtype=torch.float8_e4m3fn), meta(-(-rows // block_rows), -(-K // 128), dtype=torch.float32)


@pytest.mark.parametrize("over", [(1 << 30) + 16, (1 << 32) + 128])
def test_widths_that_no_32_bit_argument_holds(on_any_device, over):
    """(2^32 + 128 channels would arrive as 128)"""
    calls = [lambda: ops.rms_norm(meta(1, over), meta(over)), lambda: ops.rms_norm(meta(1, over), meta(over), quantize=True),
             lambda: ops.quantize_fp8(meta(1, over)), lambda: ops.quantize_fp8(meta(130, over), 128),
             lambda: ops.linear_fp8(meta8(1, over), meta8(8, over, 128)), lambda: ops.linear_fp8(meta8(1, 128), meta8(over, 128, 128))]
    for call in calls:
        with torch.no_grad(), pytest.raises(ValueError, match="2\\^30"):
            call()
    assert not on_any_device
    with torch.no_grad():
        ops.rms_norm(meta(2, 1 << 30), meta(1 << 30))
        ops.quantize_fp8(meta(1 << 33, 8))                   # (rows are counted in 64 bits)
    assert len(on_any_device) == 2


@pytest.mark.parametrize("which", ["a", "a scales", "w", "w scales", "bias", "residual"])
def test_a_product_of_what_wants_a_gradient(which):
    t = {"a": torch.zeros(2, 16).to(torch.float8_e4m3fn), "a scales": torch.ones(2, 1), "w": torch.zeros(8, 16).to(torch.float8_e4m3fn),
         "w scales": torch.ones(1, 1), "bias": torch.zeros(8), "residual": torch.zeros(2, 8)}
    t[which].requires_grad_()

    def call():
        return ops.linear_fp8((t["a"], t["a scales"]), (t["w"], t["w scales"]), bias=t["bias"], residual=t["residual"], dtype=torch.float32)

    with pytest.raises(RuntimeError, match="forward-only"):
        call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        call()
