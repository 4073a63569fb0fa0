"""What the norm and the quantisers write, and nothing else, in every share of a row and at every alignment; and their in-place forms."""
import pytest
import torch

from convnn_b200 import _capi, ops
from gpu_util import DEV
from test_gpu_fp8 import BF16, F32, blocks_of, randn, same_bytes

pytestmark = pytest.mark.gpu

WIDTHS = [1, 7, 8, 128, 131, 192, 250, 256, 264, 700, 770, 1000, 1001, 1536, 2050, 2568, 4100, 6152, 8200, 9001]


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def code(dtype):
    return _capi.BF16 if dtype == BF16 else _capi.F32


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("extra,offset", [(0, 0), (16, 8), (1, 1), (2, 2)])
def test_the_norm_leaves_what_lies_between_its_rows(D, dtype, extra, offset):
    rows, L = 11, _capi.lib()
    x, res, w = randn(rows, D, seed=1, dtype=dtype), randn(rows, D, seed=2, dtype=dtype), randn(D, seed=3, dtype=dtype)
    want, want_sum = ops.rms_norm(x, w, residual=res)
    want8, _ = ops.rms_norm(x, w, residual=res, quantize=True)
    ld = (D + 15) // 16 * 16 + extra
    y, s = (torch.full((offset + (rows + 9) * ld,), 5.0, dtype=dtype, device=DEV) for _ in range(2))
    elt = y.element_size()
    _capi.check(L.convnn_b200_rms_norm(code(dtype), x.data_ptr(), D, res.data_ptr(), D, w.data_ptr(), 1e-6, s.data_ptr() + offset * elt, ld,
                                       y.data_ptr() + offset * elt, ld, rows, D, stream()))
    for room, exact in ((y, want), (s, want_sum)):
        out = room[offset:].view(rows + 9, ld)
        assert torch.equal(out[:rows, :D], exact) and (out[rows:] == 5).all() and (out[:, D:] == 5).all() and (room[:offset] == 5).all()
    for what in ("norm", "rows"):
        q = torch.full((offset + (rows + 9) * ld,), 0x55, dtype=torch.uint8, device=DEV)
        scales = torch.full((rows + 9, 2 * blocks_of(D) + 1), -7.0, device=DEV)
        to = (q.data_ptr() + offset, ld, scales.data_ptr(), scales.stride(0), 2, rows, D, stream())
        if what == "norm":
            exact = want8
            _capi.check(L.convnn_b200_rms_norm_fp8(code(dtype), x.data_ptr(), D, res.data_ptr(), D, w.data_ptr(), 1e-6,
                                                   s.data_ptr() + offset * elt, ld, *to))
        else:
            exact = ops.quantize_fp8(x)
            _capi.check(L.convnn_b200_quantize_fp8(code(dtype), x.data_ptr(), D, 1, *to))
        out = q[offset:].view(rows + 9, ld)
        assert same_bytes(out[:rows, :D], exact.values) and torch.equal(scales[:rows, :2 * blocks_of(D):2], exact.scales)
        assert (out[rows:] == 0x55).all() and (out[:, D:] == 0x55).all() and (q[:offset] == 0x55).all()
        assert (scales[rows:] == -7).all() and (scales[:, 1::2] == -7).all() and (scales[:, -1] == -7).all()


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_result_in_the_place_of_x_and_the_sum_in_that_of_the_residual(D, dtype):
    rows = 300
    x, res, w = randn(rows, D, seed=1, dtype=dtype), randn(rows, D, seed=2, dtype=dtype), randn(D, seed=3, dtype=dtype)
    want, want_sum = ops.rms_norm(x, w, residual=res)
    _capi.check(_capi.lib().convnn_b200_rms_norm(code(dtype), x.data_ptr(), D, res.data_ptr(), D, w.data_ptr(), 1e-6, res.data_ptr(), D,
                                                 x.data_ptr(), D, rows, D, stream()))
    assert torch.equal(x, want) and torch.equal(res, want_sum)


@pytest.mark.parametrize("D", [1, 8, 131, 136, 300, 1000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_quantiser_of_weights_leaves_what_lies_between_its_rows(D, dtype):
    for rows in (1, 100, 129, 260):
        x = randn(rows, D, seed=1, dtype=dtype)
        want = ops.quantize_fp8(x, 128)
        ld, blocks, groups = (D + 15) // 16 * 16 + 3, blocks_of(D), -(-rows // 128)
        q = torch.full((rows + 140, ld), 0x55, dtype=torch.uint8, device=DEV)
        scales = torch.full((groups + 2, blocks + 2), -7.0, device=DEV)
        _capi.check(_capi.lib().convnn_b200_quantize_fp8(code(dtype), x.data_ptr(), D, 128, q.data_ptr(), ld, scales.data_ptr(), blocks + 2, 1,
                                                         rows, D, stream()))
        assert same_bytes(q[:rows, :D], want.values) and torch.equal(scales[:groups, :blocks], want.scales)
        assert (q[rows:] == 0x55).all() and (q[:, D:] == 0x55).all() and (scales[groups:] == -7).all() and (scales[:, blocks:] == -7).all()
