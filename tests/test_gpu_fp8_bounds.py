"""What the 8-bit product writes, and nothing else: rows behind the last, columns behind the last, scales between those that it owns, in every
form and with output rows that start on 16-byte boundaries or anywhere."""
import pytest
import torch

from convnn_b200 import _capi, ops
from gpu_util import DEV
from test_gpu_fp8 import BF16, F32, blocks_of, operands, randn, same_bytes

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def call(a, w, out, ldo, M, N, K, dtype, bias=None, res=None, gelu=0, scales=None, row=0, block=0):
    (av, sa), (wv, sw) = a, w
    _capi.check(_capi.lib().convnn_b200_linear_fp8(
        av.data_ptr(), av.stride(0), sa.data_ptr(), *sa.stride(), wv.data_ptr(), wv.stride(0), sw.data_ptr(), *sw.stride(),
        _capi.BF16 if dtype == BF16 else _capi.F32, None if bias is None else bias.data_ptr(), None if res is None else res.data_ptr(),
        0 if res is None else res.stride(0), out, ldo, None if scales is None else scales.data_ptr(), row, block, M, N, K, gelu,
        torch.cuda.current_stream().cuda_stream))


# weights as rows with 16, 32 and 64 tokens, 128 x 128 tiles alone and in clusters, pairs
SIZES = [(3, 1001, 300), (20, 131, 2000), (61, 1000, 128), (100, 20001, 200), (1027, 1003, 1333), (300, 4001, 130), (2000, 1100, 200)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("extra", [0, 1, 2, 16])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_and_columns_behind_the_last(M, N, K, extra, dtype):
    a, w = operands(M, N, K, seed=5)
    bias, res = randn(N, seed=6, dtype=dtype), randn(M, N, seed=7, dtype=dtype)
    want = ops.linear_fp8(a, w, bias=bias, residual=res, dtype=dtype)
    ldo = (N + 15) // 16 * 16 + extra
    out = torch.full((M + 130, ldo), 5.0, dtype=dtype, device=DEV)
    call(a, w, out.data_ptr(), ldo, M, N, K, dtype, bias, res)
    assert torch.equal(out[:M, :N], want)
    assert (out[M:] == 5).all() and (out[:, N:] == 5).all()


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("extra,offset", [(0, 0), (16, 16), (1, 0), (0, 1), (7, 3), (8, 8)])
@pytest.mark.parametrize("row_major", [False, True])
def test_8_bit_rows_that_start_anywhere(M, N, K, extra, offset, row_major):
    a, w = operands(M, N, K, seed=5)
    bias = randn(N, seed=6, dtype=BF16)
    want = ops.linear_fp8(a, w, bias=bias, gelu=True, quantize=True)
    ldo, blocks = (N + 15) // 16 * 16 + extra, blocks_of(N)
    room = torch.full((offset + (M + 130) * ldo,), 0x55, dtype=torch.uint8, device=DEV)
    row, block = (2 * blocks + 1, 2) if row_major else (2, 2 * M + 3)
    scales = torch.full(((M + 130) * 2 * (blocks + 2),), -7.0, device=DEV)
    call(a, w, room.data_ptr() + offset, ldo, M, N, K, BF16, bias, None, 1, scales, row, block)
    out = room[offset:].view(M + 130, ldo)
    assert same_bytes(out[:M, :N], want.values)
    assert (out[M:] == 0x55).all() and (out[:, N:] == 0x55).all() and (room[:offset] == 0x55).all()
    own = torch.as_strided(scales, (M, blocks), (row, block))
    assert torch.equal(own, want.scales)
    own.fill_(-7.0)
    assert (scales == -7).all()


@pytest.mark.parametrize("M,N,K", [(3, 1001, 300), (20, 131, 1999), (61, 1000, 127), (100, 20001, 200), (1027, 1003, 1333), (300, 4001, 129),
                                   (2000, 1100, 1)])
def test_what_lies_behind_the_operands_rows_is_not_read(M, N, K):
    """NaN between a row's last channel and the next row, behind the last row, and between the scales."""
    a, w = operands(M, N, K, seed=8)
    want = ops.linear_fp8(a, w, dtype=F32)
    assert want.isfinite().all()

    def among_nan(t):
        values, scales = t
        rows = values.shape[0]
        room = torch.full((rows + 256, (K + 15) // 16 * 16 + 16), 0x7f, dtype=torch.uint8, device=DEV)
        room[:rows, :K] = values.view(torch.uint8)
        wide = torch.full((scales.shape[0] + 256, scales.shape[1] + 5), float("nan"), device=DEV)
        wide[:scales.shape[0], :scales.shape[1]] = scales
        return room.view(values.dtype)[:rows, :K], wide[:scales.shape[0], :scales.shape[1]]

    assert torch.equal(ops.linear_fp8(among_nan(a), among_nan(w), dtype=F32), want)
