"""Scales of the 8-bit product far from one: what is promised for every pair whose product is a normal float32."""
import pytest
import torch

from convnn_b200 import _capi, ops
from gpu_util import DEV
from test_gpu_fp8 import F32, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


@pytest.mark.parametrize("M,N", [(3, 130), (60, 131), (100, 20001), (300, 4001)])
@pytest.mark.parametrize("ea,ew", [(50, 50), (-63, -63), (100, -100), (-100, 100), (-126, 0), (0, -126), (100, 0), (0, 100)])
def test_scales_whose_products_are_far_from_one(M, N, ea, ew):
    """Scales that are multiplied by exact powers of two: the same sums times their product, which is a normal float32.  300 products of
    448 * 448 / 512 at most are below 2^17, so that 2^100 leaves all sums, of a part of the blocks too, below 2^128."""
    K = 300
    a, w = ops.quantize_fp8(randn(M, K, seed=1)), ops.quantize_fp8(randn(N, K, seed=2), 128)
    av = (a.values.float() / 512).to(a.values.dtype)
    room = torch.zeros(M, 304, dtype=torch.uint8, device=DEV).view(av.dtype)
    room[:, :K].view(torch.uint8).copy_(av.view(torch.uint8))
    av, sa, sw = room[:, :K], torch.ones_like(a.scales), torch.ones_like(w.scales)
    one = ops.linear_fp8((av, sa), (w.values, sw), dtype=F32).double()
    got = ops.linear_fp8((av, sa * 2.0 ** ea), (w.values, sw * 2.0 ** ew), dtype=F32).double()
    want = one * 2.0 ** (ea + ew)
    normal = want.abs() >= 2.0 ** -126
    assert normal.any() and torch.equal(got[normal], want[normal])
    if ea + ew >= 0:
        assert torch.equal(got, want)
