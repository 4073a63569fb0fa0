"""The 8-bit operators (root-mean-square norm with 8-bit output, quantisers, block-scaled product) against their formulas in
64 bits, and as a chain.

Tolerances.  A rounding is off by half a step at most, relative to the value: ``HALF`` (bfloat16 2^-8, float32 2^-24, e4m3 2^-4,
or 2^-10 of the scale below the normal range).  Float32 sums of n terms are off by n * 2^-24 of the sum of magnitudes; in the product a
block of 128 channels is four tensor-core sums of 32 products and a running value, each taken as 33 truncations (2^-23) of at most the
sum of magnitudes, and the blocks are one rounding of the scale and one of the addition each."""
import itertools

import pytest
import torch

from convnn_b200 import _capi, ops
from convnn_b200.ops import Fp8Blocks
from gpu_util import DEV

pytestmark = pytest.mark.gpu

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U, E4M3: 2.0 ** -4}
LEAST = 2.0 ** -126


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def randn(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def blocks_of(D):
    return (D + 127) // 128


def spread(scales, rows, D, block_rows=1):
    """Scales -> one per value."""
    return scales.repeat_interleave(128, -1)[..., :D].repeat_interleave(block_rows, 0)[:rows]


def plain_quantize(v, block_rows=1):
    """The formula in v's precision on (rows, D)."""
    rows, D = v.shape
    p = torch.nn.functional.pad(v, (0, -D % 128, 0, -rows % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, -1, 128)
    scale = torch.clamp(p.abs().amax(dim=(1, 3)) * (1.0 / 448.0), min=LEAST)
    q = (p * (1.0 / scale)[:, None, :, None]).reshape(p.shape[0] * block_rows, -1)[:rows, :D]
    return q.to(E4M3), scale


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def meant(t, block_rows=1):
    values, scales = t
    v = values.reshape(-1, values.shape[-1]).double()
    return v * spread(scales.reshape(-1, scales.shape[-1]).double(), v.shape[0], v.shape[1], block_rows)


def check_blocks(got, want, err):
    """8-bit rows against exact values that are themselves known to `err` (absolute, per value)."""
    values, scales = got
    rows, D = want.shape
    assert values.dtype == E4M3 and scales.dtype == F32
    assert values.shape[-1] == D and scales.shape[-1] == blocks_of(D)
    values, scales = values.reshape(rows, D), scales.reshape(rows, -1).double()
    pad = torch.nn.functional.pad
    top = pad(want.abs(), (0, -D % 128)).view(rows, -1, 128).amax(-1)
    far = pad(err, (0, -D % 128)).view(rows, -1, 128).amax(-1)
    exact_scale = (top / 448.0).clamp(min=LEAST)
    assert torch.all((scales - exact_scale).abs() <= far / 448.0 + 4 * U * exact_scale)
    per = spread(scales, rows, D)
    off = (values.double() * per - want).abs()
    assert torch.all(off <= (HALF[E4M3] * want.abs()).maximum(2.0 ** -10 * per) + 1.1 * err + 4 * U * want.abs())


# ---- the norm -------------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 768), (3, 5), (9, 127), (8, 128), (17, 129), (33, 192), (5, 256), (6, 260), (7, 512), (3, 514), (65, 768),
               (2, 1001), (10, 1024), (4, 1028), (30, 1002), (3, 2426), (70, 250), (3, 4096), (2, 4099), (3, 8192), (2, 8196), (2, 20001), (1, 20480)]


def norm_exact(s, weight, eps):
    s, w = s.double(), weight.double()
    return s * torch.rsqrt((s * s).mean(-1, keepdim=True) + eps) * w


def norm_err(want, D):
    # a lane adds D / 32 squares at most, then at most 5 + 8 more; half of that in the root, rsqrt two steps, two products, 1 / D
    return (0.5 * (D / 32 + 16) + 6) * U * want.abs()


@pytest.mark.parametrize("rows,D", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(rows, D, dtype, with_residual):
    x, w = randn(rows, D, seed=1, dtype=dtype, scale=3.0), 1.0 + randn(D, seed=2, dtype=dtype, scale=0.3)
    res = randn(rows, D, seed=3, dtype=dtype) if with_residual else None
    y = ops.rms_norm(x, w, 1e-6, residual=res)
    q = ops.rms_norm(x, w, 1e-6, residual=res, quantize=True)
    s = x
    if with_residual:
        (y, s), (q, s2) = y, q
        assert torch.equal(s, (x.float() + res.float()).to(dtype)) and torch.equal(s, s2)
    want = norm_exact(s, w, 1e-6)
    err = norm_err(want, D)
    assert y.dtype == dtype and y.shape == x.shape
    assert torch.all((y.double() - want).abs() <= HALF[dtype] * want.abs() + 1.1 * err)
    check_blocks(q, want, err)


def test_norm_of_strided_rows_and_more_dimensions():
    wide = randn(4, 7, 300, seed=1, dtype=BF16)
    w = randn(192, seed=2, dtype=BF16)
    for x in (wide[:, :, :192], wide[:, :, 64:256], wide[:, :, 3:195], wide[:, ::2, :192], wide[:, :, :192].transpose(0, 1)):
        want, s = ops.rms_norm(x.contiguous(), w, residual=x.flip(-1).contiguous())
        got, t = ops.rms_norm(x, w, residual=x.flip(-1))
        assert torch.equal(got, want) and torch.equal(s, t) and got.shape == x.shape
        a, b = ops.rms_norm(x, w, quantize=True), ops.rms_norm(x.contiguous(), w, quantize=True)
        assert a.values.shape == x.shape and a.scales.shape == (*x.shape[:2], 2)
        assert same_bytes(a.values, b.values) and torch.equal(a.scales, b.scales)
    one = randn(192, seed=5, dtype=BF16)
    assert torch.equal(ops.rms_norm(one, w), ops.rms_norm(one[None], w)[0])
    assert ops.rms_norm(one, w, quantize=True).scales.shape == (2,)
    spread_res = randn(1, 192, seed=6, dtype=BF16).expand(7, 192)                # (a residual shared by all rows)
    x = wide[0, :, :192]
    assert torch.equal(ops.rms_norm(x, w, residual=spread_res)[0], ops.rms_norm(x, w, residual=spread_res.contiguous())[0])


def test_norm_strided_weight_and_offset_storage():
    buf = randn(1 + 6 * 192, seed=4, dtype=BF16)
    x = buf[1:].view(6, 192)                                  # rows on two-byte boundaries
    w = randn(384, seed=2, dtype=BF16)[::2]
    assert torch.equal(ops.rms_norm(x, w), ops.rms_norm(x.clone(), w.contiguous()))


# every share of a row among warps, full and with a rest, and rows that leave warps of the last CTA without one
@pytest.mark.parametrize("rows,D", [(5, 1000), (6, 1018), (3, 1280), (5, 1281), (2, 1536), (5, 1544), (7, 2040), (1, 2048), (3, 2050), (3, 2568),
                                    (5, 2560), (3, 2561), (9, 4088), (2, 4098), (3, 6144), (2, 6001), (2, 6152)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_rows_of_several_warps(rows, D, dtype):
    for with_residual in (False, True):
        test_norm(rows, D, dtype, with_residual)
    x, w = randn(1 + rows * D, seed=7, dtype=dtype), randn(D, seed=8, dtype=dtype)
    view, res = x[1:].view(rows, D), randn(rows, D, seed=9, dtype=dtype)       # (rows on two- or four-byte boundaries)
    got, s = ops.rms_norm(view, w, residual=res, quantize=True)
    want, t = ops.rms_norm(view.clone(), w, residual=res, quantize=True)
    assert torch.equal(s, t) and same_bytes(got.values, want.values) and torch.equal(got.scales, want.scales)
    assert torch.equal(ops.rms_norm(view, w), ops.rms_norm(view.clone(), w))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_zero_rows_infinities_and_nan(dtype):
    x = randn(5, 300, seed=1, dtype=dtype)
    w = torch.ones(300, device=DEV, dtype=dtype)
    clean = ops.rms_norm(x, w)
    x[1] = 0
    x[2, 130] = float("inf")
    x[3, 7] = float("nan")
    y = ops.rms_norm(x, w, 0.0)
    q = ops.rms_norm(x, w, 1e-6, quantize=True)
    assert torch.equal(ops.rms_norm(x, w)[[0, 4]], clean[[0, 4]])       # other rows are left alone
    assert y[1].isnan().all()                                            # 0 * rsqrt(0), as the formula has it
    assert (ops.rms_norm(x, w)[1] == 0).all() and (q.values[1].float() == 0).all() and torch.all(q.scales[1] == LEAST)
    assert y[2, 130].isnan() and (y[2, :130] == 0).all()
    assert y[3].isnan().all() and meant(q)[3].isnan().all()
    assert meant(q)[2, 128:256].isnan().all() and (meant(q)[2, :128] == 0).all()
    assert meant(q)[[0, 4]].isfinite().all()


# ---- the quantisers -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,D", [(1, 1), (1, 4096), (2, 127), (3, 128), (127, 129), (128, 256), (129, 260), (200, 1001), (5, 20484), (300, 384), (77, 386), (131, 130), (9, 640), (1000, 256)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_is_the_formula(rows, D, dtype, block_rows):
    x = randn(rows, D, seed=1, dtype=dtype) * torch.exp(randn(D, seed=2, dtype=dtype))
    got = ops.quantize_fp8(x, block_rows)
    q, scale = plain_quantize(x.float(), block_rows)
    assert got.scales.shape == scale.shape and torch.equal(got.scales, scale)
    assert got.values.shape == q.shape and same_bytes(got.values, q)
    exact = x.double()
    off = (meant(got, block_rows) - exact).abs()
    per = spread(got.scales.double(), rows, D, block_rows)
    assert torch.all(off <= (HALF[E4M3] * exact.abs()).maximum(2.0 ** -10 * per) + 4 * U * exact.abs())


def test_quantize_strides_shapes_and_extremes():
    wide = randn(3, 5, 400, seed=1, dtype=BF16)
    for x in (wide[:, :, 8:208], wide[:, :, 1:200], wide[:, 1::2, :256], wide.transpose(0, 1)):
        a, b = ops.quantize_fp8(x), ops.quantize_fp8(x.contiguous().view(-1, x.shape[-1]))
        assert a.values.shape == x.shape and a.scales.shape == (*x.shape[:2], blocks_of(x.shape[-1]))
        assert same_bytes(a.values.reshape(b.values.shape), b.values) and torch.equal(a.scales.reshape(b.scales.shape), b.scales)
    x = torch.zeros(4, 256, device=DEV)
    x[0, 3] = 3.4e38
    x[1] = 1e-42                                             # below what 1 / scale can be finite for
    x[2, 200] = float("nan")
    x[3, 5], x[3, 6] = float("-inf"), 1.0
    for block_rows in (1, 128):
        q, scale = plain_quantize(x, block_rows)
        got = ops.quantize_fp8(x, block_rows)
        assert torch.equal(got.scales.nan_to_num(nan=-1.0), scale.nan_to_num(nan=-1.0))
        assert same_bytes(got.values.float().nan_to_num(nan=-1.0), q.float().nan_to_num(nan=-1.0))
    assert meant(ops.quantize_fp8(x))[1].eq(0).all()         # (2^-126 * 2^-9 is above them)
    assert meant(ops.quantize_fp8(x))[3, :128].isnan().all() and meant(ops.quantize_fp8(x))[3, 128:].eq(0).all()


def test_rows_are_left_alone_behind_the_last_channel():
    """Rows of 8-bit values start on 16-byte boundaries; what lies between is not written by the norm or the quantisers."""
    L = _capi.lib()
    x, w = randn(6, 131, seed=1, dtype=BF16), randn(131, seed=2, dtype=BF16)
    st = torch.cuda.current_stream().cuda_stream
    for k in range(3):
        q = torch.full((8, 144), 0x55, dtype=torch.uint8, device=DEV)
        s = torch.full((8, 4), -7.0, device=DEV)
        args = (q.data_ptr(), 144, s.data_ptr(), 4, 1, 6, 131, st)
        if k == 0:
            _capi.check(L.convnn_b200_rms_norm_fp8(_capi.BF16, x.data_ptr(), 131, None, 0, w.data_ptr(), 1e-6, None, 0, *args))
        else:
            _capi.check(L.convnn_b200_quantize_fp8(_capi.BF16, x.data_ptr(), 131, 1 if k == 1 else 128, *args))
        torch.cuda.synchronize()
        assert (q[:6, 131:] == 0x55).all() and (q[6:] == 0x55).all()
        assert (s[:, 2:] == -7).all() and (s[6 if k < 2 else 1:] == -7).all()
        assert (s[:6 if k < 2 else 1, :2] > 0).all()


# ---- the product ----------------------------------------------------------------------------------------------------

def operands(M, N, K, seed=0):
    a = ops.quantize_fp8(randn(M, K, seed=seed) * torch.exp(randn(K, seed=seed + 1)))
    w = ops.quantize_fp8(randn(N, K, seed=seed + 2, scale=K ** -0.5), 128)
    return a, w


def linear_exact(a, w, bias=None, gelu=False, residual=None):
    """-> result in 64 bits, how far a float32 one may be from it."""
    A, W = meant(a), meant(w, 128)
    out = A @ W.t()
    blocks = blocks_of(A.shape[1])
    err = (2 * 4 * 33 + 2 * blocks + 8) * U * (A.abs() @ W.abs().t())
    if bias is not None:
        out = out + bias.double()
        err = err + U * out.abs()
    if gelu:
        err = 1.13 * err + 8 * U * out.abs()                 # |gelu'| <= 1.129; erf two steps, three roundings
        out = out * torch.special.ndtr(out)
    if residual is not None:
        out = out + residual.reshape(out.shape).double()
        err = err + U * out.abs()
    return out, err


def check_linear(a, w, bias=None, gelu=False, residual=None, dtype=BF16, quantize=False):
    got = ops.linear_fp8(a, w, bias=bias, gelu=gelu, residual=residual, dtype=dtype, quantize=quantize)
    want, err = linear_exact(a, w, bias, gelu, residual)
    if quantize:
        check_blocks(got, want, err)
        return got
    assert got.dtype == dtype
    off = (got.reshape(want.shape).double() - want).abs()
    assert torch.all(off <= HALF[dtype] * want.abs() + 1.1 * err), float((off / (HALF[dtype] * want.abs() + err)).max())
    return got


SIZES_M = [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 300]
SIZES_NK = [(1, 1), (8, 16), (100, 127), (128, 128), (130, 129), (200, 600), (257, 1333), (1000, 256), (128, 4096), (384, 8200)]


@pytest.mark.parametrize("M", SIZES_M)
@pytest.mark.parametrize("N,K", SIZES_NK)
def test_linear_sizes(M, N, K):
    a, w = operands(M, N, K, seed=M + N)
    check_linear(a, w, dtype=F32)
    check_linear(a, w, dtype=BF16)
    check_linear(a, w, quantize=True)


@pytest.mark.parametrize("M", [1, 20, 64, 200])
@pytest.mark.parametrize("bias,gelu,residual", list(itertools.product([False, True], repeat=3)))
@pytest.mark.parametrize("dtype,quantize", [(BF16, False), (F32, False), (BF16, True), (F32, True)])
def test_linear_epilogue(M, bias, gelu, residual, dtype, quantize):
    N, K = 203, 300
    a, w = operands(M, N, K, seed=3)
    check_linear(a, w, randn(N, seed=8, dtype=dtype) if bias else None, gelu,
                 randn(M, N, seed=9, dtype=dtype) if residual else None, dtype, quantize)


def test_linear_many_rows_of_a_long_batch():
    a, w = operands(256 * 197, 192, 768, seed=3)
    check_linear(a, w, randn(192, seed=8, dtype=BF16), residual=randn(256 * 197, 192, seed=9, dtype=BF16))
    a, w = operands(8 * 197, 768, 192, seed=4)
    check_linear(a, w, randn(768, seed=8, dtype=BF16), gelu=True, quantize=True)


# shapes of at least 74 tiles of 256 x 256, the persistent pairs' form
PAIR_SIZES = [(256 * 74, 256, 128), (256 * 73 + 1, 200, 100), (256 * 40 - 3, 257, 300), (2500, 2000, 1333), (5000, 1111, 640), (2304, 2304, 4096),
              (100, 20000, 200)]


@pytest.mark.parametrize("M,N,K", PAIR_SIZES)
@pytest.mark.parametrize("dtype,quantize", [(BF16, False), (F32, False), (BF16, True)])
def test_linear_many_tiles(M, N, K, dtype, quantize):
    a, w = operands(M, N, K, seed=M + N)
    check_linear(a, w, dtype=dtype, quantize=quantize)
    bias, res = randn(N, seed=8, dtype=dtype), randn(M, N, seed=9, dtype=dtype)
    check_linear(a, w, bias, False, res, dtype, quantize)
    check_linear(a, w, bias, True, None, dtype, quantize)
    check_linear(a, w, None, True, res, dtype, quantize)


def test_linear_many_tiles_strides_and_nan():
    M, N, K = 4000, 1300, 400
    a, w = operands(M, N, K, seed=2)
    res = randn(M, N + 3, seed=6)[:, 3:]
    bias = randn(N + 1, seed=5)[1:]
    want = ops.linear_fp8(a, w, bias=bias.clone(), residual=res.contiguous(), dtype=F32)
    got = ops.linear_fp8((a.values, a.scales.contiguous()), w, bias=bias, residual=res, dtype=F32)
    assert torch.equal(got, want)
    a.scales[7, 1] = float("nan")
    got = ops.linear_fp8(a, w, bias=bias, residual=res, dtype=F32)
    assert got[7].isnan().all() and torch.equal(got[:7], want[:7]) and torch.equal(got[8:], want[8:])
    q = ops.linear_fp8(a, w, gelu=True, quantize=True)
    assert meant(q)[7].isnan().all() and meant(q)[8:].isfinite().all()
    out = torch.full((M, N + 5), 3.0, device=DEV)            # rows of another stride, the rest left alone
    L = _capi.lib()
    _capi.check(L.convnn_b200_linear_fp8(a.values.data_ptr(), 400, a.scales.data_ptr(), *a.scales.stride(), w.values.data_ptr(), 400,
                                         w.scales.data_ptr(), *w.scales.stride(), _capi.F32, None, None, 0, out.data_ptr(), N + 5, None,
                                         0, 0, M, N, K, 0, torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[8:, :N], ops.linear_fp8(a, w, dtype=F32)[8:]) and (out[:, N:] == 3).all()


@pytest.mark.parametrize("M", [5, 40, 150])
def test_linear_strides_and_shapes(M):
    N, K = 160, 400
    a, w = operands(M, N, K, seed=1)
    want = ops.linear_fp8(a, w, dtype=F32)
    row_major = Fp8Blocks(a.values, a.scales.contiguous())
    wide = torch.zeros(M, 2 * 512, dtype=torch.uint8, device=DEV).view(E4M3)
    wide.view(torch.uint8)[:, 16:416] = a.values.view(torch.uint8)
    odd = torch.zeros(M, 403, dtype=torch.uint8, device=DEV).view(E4M3)          # rows on no 16-byte boundaries
    odd.view(torch.uint8)[:, 3:] = a.values.view(torch.uint8)
    turned = a.values.view(torch.uint8).t().contiguous().t().view(E4M3)
    for other in (row_major, (wide[:, 16:416], a.scales), (odd[:, 3:], a.scales), (turned, row_major.scales)):
        assert torch.equal(ops.linear_fp8(other, w, dtype=F32), want)
    w_odd = torch.zeros(N, 401, dtype=torch.uint8, device=DEV).view(E4M3)
    w_odd.view(torch.uint8)[:, 1:] = w.values.view(torch.uint8)
    w_scales = w.scales.t().contiguous().t()
    assert torch.equal(ops.linear_fp8(a, (w_odd[:, 1:], w_scales), dtype=F32), want)
    shared = a.scales[:1].expand(M, -1)                                          # one row's scales for all
    check_linear((a.values, shared), w, dtype=F32)
    bias, res = randn(2 * N, seed=5)[::2], randn(M, N + 3, seed=6)[:, 3:]
    got = ops.linear_fp8(a, w, bias=bias, residual=res, dtype=F32)
    assert torch.equal(got, ops.linear_fp8(a, w, bias=bias.contiguous(), residual=res.contiguous(), dtype=F32))
    three = Fp8Blocks(a.values.view(M // 5, 5, K), a.scales.view(M // 5, 5, -1)) if M % 5 == 0 else None
    if three is not None:
        assert torch.equal(ops.linear_fp8(three, w, dtype=F32), want.view(M // 5, 5, N))
        assert ops.linear_fp8(three, w, quantize=True).scales.shape == (M // 5, 5, 2)
    one = Fp8Blocks(a.values[0], a.scales[0])
    assert ops.linear_fp8(one, w, dtype=F32).shape == (N,)
    check_linear((a.values[:1], a.scales[:1]), w, dtype=F32)


def test_linear_of_no_rows():
    a, w = operands(3, 100, 200)
    none = Fp8Blocks(a.values[:0], a.scales[:0])
    assert ops.linear_fp8(none, w).shape == (0, 100)
    q = ops.linear_fp8(none, w, quantize=True)
    assert q.values.shape == (0, 100) and q.scales.shape == (0, 1)
    x = randn(0, 200, dtype=BF16)
    y, s = ops.rms_norm(x, randn(200, dtype=BF16), residual=x, quantize=True)
    assert y.values.shape == (0, 200) and y.scales.shape == (0, 2) and s.shape == (0, 200)
    assert ops.quantize_fp8(x, 128).scales.shape == (0, 2)


@pytest.mark.parametrize("M", [3, 90])
def test_linear_nan_stays_in_its_row(M):
    N, K = 150, 300
    x = randn(M, K, seed=1)
    a, w = ops.quantize_fp8(x), ops.quantize_fp8(randn(N, K, seed=2), 128)
    want = ops.linear_fp8(a, w, dtype=F32)
    x[1, 200] = float("nan")
    x[2, 5] = float("inf")
    got = ops.linear_fp8(ops.quantize_fp8(x), w, dtype=F32)
    assert got[1].isnan().all() and got[2].isnan().all()
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[keep], want[keep])
    q = ops.linear_fp8(ops.quantize_fp8(x), w, quantize=True)
    assert meant(q)[1].isnan().all() and meant(q)[keep].isfinite().all()


def test_linear_scales_far_apart():
    """Blocks whose scales differ by many powers of two: the sum is what the scales say."""
    M, N, K = 70, 130, 640
    a, w = operands(M, N, K)
    factors = torch.tensor([2.0 ** -60, 1.0, 2.0 ** -20, 2.0 ** 7, 0.0], device=DEV)
    check_linear((a.values, a.scales * factors), w, dtype=F32)
    check_linear((a.values[:9], (a.scales * factors)[:9]), (w.values, w.scales * factors.flip(0)), dtype=F32)


def test_results_are_the_same_bits_every_time():
    for M in (1, 30, 197, 700):
        a, w = operands(M, 768, 768, seed=M)
        first = ops.linear_fp8(a, w, gelu=True, quantize=True)
        for _ in range(3):
            again = ops.linear_fp8(a, w, gelu=True, quantize=True)
            assert same_bytes(first.values, again.values) and torch.equal(first.scales, again.scales)


def test_offsets_beyond_32_bits():
    rows, D = 1_420_000, 1536                                # 2.18e9 values
    x = torch.zeros(rows, D, dtype=BF16, device=DEV)
    x[-3:] = randn(3, D, seed=1, dtype=BF16)
    w = torch.ones(D, dtype=BF16, device=DEV)
    q = ops.quantize_fp8(x)
    want = ops.quantize_fp8(x[-3:])
    assert same_bytes(q.values[-3:], want.values) and torch.equal(q.scales[-3:], want.scales)
    y, s = ops.rms_norm(x, w, residual=x)
    assert torch.equal(y[-3:], ops.rms_norm(x[-3:], w, residual=x[-3:])[0]) and torch.equal(s[-3:], 2 * x[-3:])
    del y, s
    weight = ops.quantize_fp8(randn(1600, D, seed=2), 128)
    out = ops.linear_fp8(q, weight)                          # 2.27e9 results
    assert torch.equal(out[-3:], ops.linear_fp8(Fp8Blocks(q.values[-128 - rows % 128:], q.scales[-128 - rows % 128:]), weight)[-3:])
    assert (out[1000] == 0).all()


# ---- together -------------------------------------------------------------------------------------------------------

def encoder_mlp(x, delta, weights):
    """norm -> first half with GELU -> second half with the residual, in 8 bits: three launches."""
    gamma, w1, b1, w2, b2 = weights
    h, x = ops.rms_norm(x, gamma, residual=delta, quantize=True)
    h2 = ops.linear_fp8(h, w1, bias=b1, gelu=True, quantize=True)
    return ops.linear_fp8(h2, w2, bias=b2, residual=x), h, h2, x


def mlp_weights(D, DM, dtype=BF16):
    return (1.0 + randn(D, seed=11, dtype=dtype, scale=0.2), ops.quantize_fp8(randn(DM, D, seed=12, dtype=dtype, scale=D ** -0.5), 128),
            randn(DM, seed=13, dtype=dtype, scale=0.1), ops.quantize_fp8(randn(D, DM, seed=14, dtype=dtype, scale=DM ** -0.5), 128),
            randn(D, seed=15, dtype=dtype, scale=0.1))


@pytest.mark.parametrize("B,T,D,DM", [(1, 1, 192, 768), (2, 197, 192, 768), (3, 65, 200, 500), (1, 50, 768, 1536)])
def test_mlp_chain(B, T, D, DM):
    x, delta = randn(B, T, D, seed=1, dtype=BF16), randn(B, T, D, seed=2, dtype=BF16)
    weights = mlp_weights(D, DM)
    gamma, w1, b1, w2, b2 = weights
    out, h, h2, s = encoder_mlp(x, delta, weights)
    assert out.shape == x.shape and h.values.shape == x.shape and h2.values.shape == (B, T, DM)
    # each step against its formula on what it was given
    want = norm_exact(s, gamma, 1e-6).view(-1, D)
    check_blocks(h, want, norm_err(want, D))
    check_linear(h, w1, b1, True, quantize=True)
    check_linear(h2, w2, b2, residual=s)
    # and the whole against the block in 64 bits without 8-bit values.  An e4m3 value is off by 2^-4 at most, 2^-5 in the mean
    # square of a uniform error (2^-4 / sqrt(3) = 0.036): two operands in each product, the second with the first's error on it too
    v = want * 1.0
    g = v @ randn(DM, D, seed=12, dtype=BF16, scale=D ** -0.5).double().t() + b1.double()
    g = g * torch.special.ndtr(g)
    whole = g @ randn(D, DM, seed=14, dtype=BF16, scale=DM ** -0.5).double().t() + b2.double()
    off = (out.view(-1, D).double() - s.view(-1, D).double() - whole).norm() / whole.norm()
    assert off < 4 * 0.036


def test_captured_and_replayed_on_another_stream():
    weights = mlp_weights(192, 768)
    x, delta = randn(40, 192, seed=1, dtype=BF16), randn(40, 192, seed=2, dtype=BF16)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        st.wait_stream(torch.cuda.default_stream())
        encoder_mlp(x, delta, weights)
    st.synchronize()
    graphs = []
    for _ in range(2):                                       # two graphs, no memory in common
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = encoder_mlp(x, delta, weights)[0]
        graphs.append((g, out))
    for seed in (5, 6):
        x.copy_(randn(40, 192, seed=seed, dtype=BF16))
        want = encoder_mlp(x, delta, weights)[0]
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
    with torch.cuda.stream(st):
        got = encoder_mlp(x, delta, weights)[0]
    st.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once():
    weights = mlp_weights(192, 768)
    xs = [randn(197, 192, seed=i, dtype=BF16) for i in range(2)]
    want = [encoder_mlp(x, x, weights)[0] for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = encoder_mlp(xs[i], xs[i], weights)[0]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_beside_the_bfloat16_operators():
    """ops.layernorm's rows, quantised, through the 8-bit product against ops.linear."""
    x = randn(300, 192, seed=1, dtype=BF16)
    gamma, beta = torch.ones(192, device=DEV, dtype=BF16), torch.zeros(192, device=DEV, dtype=BF16)
    w = randn(384, 192, seed=2, dtype=BF16, scale=192 ** -0.5)
    h = ops.layernorm(x, gamma, beta)
    got = ops.linear_fp8(ops.quantize_fp8(h), ops.quantize_fp8(w, 128))
    want = ops.linear(h, w)
    assert ((got - want).double().norm() / want.double().norm()) < 2 * 0.036   # two operands, each off by 0.036 in the mean square


class _NoOrdinaryCalls:
    """Stands in for the module that makes ordinary calls: every call goes the general way."""
    rms_norm = quantize_fp8 = linear_fp8 = staticmethod(lambda *a: None)


@pytest.mark.parametrize("shape", [(1, 768), (7, 200), (3, 5, 131), (2, 2, 3, 64), (64,)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ordinary_and_general_calls_agree(monkeypatch, shape, dtype):
    D, N = shape[-1], 150
    x, res, w = randn(*shape, seed=1, dtype=dtype), randn(*shape, seed=2, dtype=dtype), randn(D, seed=3, dtype=dtype)
    bias, out_res = randn(N, seed=4, dtype=dtype), randn(*shape[:-1], N, seed=5, dtype=dtype)
    weight = randn(N, D, seed=6, dtype=dtype)

    def everything():
        found = [ops.rms_norm(x, w), ops.rms_norm(x, w, 1, residual=res), *ops.rms_norm(x, w, 1e-3, res),
                 *ops.rms_norm(x, w, quantize=True)]
        (q, s), t = ops.rms_norm(x, w, residual=res, quantize=True)
        a, b = ops.quantize_fp8(x), ops.quantize_fp8(weight, 128)
        found += [q, s, t, *a, *b, ops.linear_fp8(a, b), ops.linear_fp8(a, b, bias, True, out_res, dtype),
                  *ops.linear_fp8(a, b, bias=bias, residual=out_res, dtype=dtype, quantize=True), ops.linear_fp8([q, s], list(b), dtype=F32)]
        return [t for f in found for t in (f if isinstance(f, tuple) else (f,))]

    want = everything()
    monkeypatch.setattr(ops, "_calls", _NoOrdinaryCalls)
    got = everything()
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.shape == b.shape and a.dtype == b.dtype and (a.stride() == b.stride() or 1 in a.shape)
        assert torch.equal(a.float(), b.float())


def test_ordinary_calls_raise_what_the_library_says():
    with pytest.raises(ValueError, match="eps"):
        ops.rms_norm(randn(2, 8), randn(8), -1.0)
    x = randn(3, 64, dtype=BF16)
    assert torch.equal(ops.rms_norm(x, randn(64, seed=1, dtype=BF16)), ops.rms_norm(x, randn(64, seed=1, dtype=BF16)))


@pytest.mark.parametrize("rows,D", [(5, 192), (5, 130), (3, 131), (4, 1536), (4, 8200), (2, 9001)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_in_place(rows, D, dtype):
    """The sum may take the place of x or of the residual, and y that of x."""
    L, st, code = _capi.lib(), torch.cuda.current_stream().cuda_stream, _capi.BF16 if dtype == BF16 else _capi.F32
    x, res, w = randn(rows, D, seed=1, dtype=dtype), randn(rows, D, seed=2, dtype=dtype), randn(D, seed=3, dtype=dtype)
    y, s = ops.rms_norm(x, w, residual=res)
    for into in (0, 1):
        t = (x.clone(), res.clone())
        out = torch.empty_like(x)
        _capi.check(L.convnn_b200_rms_norm(code, t[0].data_ptr(), D, t[1].data_ptr(), D, w.data_ptr(), 1e-6, t[into].data_ptr(), D,
                                           out.data_ptr(), D, rows, D, st))
        assert torch.equal(t[into], s) and torch.equal(out, y)
    t = x.clone()
    _capi.check(L.convnn_b200_rms_norm(code, t.data_ptr(), D, None, 0, w.data_ptr(), 1e-6, None, 0, t.data_ptr(), D, rows, D, st))
    assert torch.equal(t, ops.rms_norm(x, w))


@pytest.mark.parametrize("M,N,K", [(3, 200, 300), (100, 203, 300), (300, 512, 256), (4000, 1300, 400), (4000, 1301, 200)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_in_the_place_of_its_residual(M, N, K, dtype):
    a, w = operands(M, N, K, seed=4)
    res = randn(M, N, seed=6, dtype=dtype)
    want = ops.linear_fp8(a, w, residual=res, dtype=dtype)
    code = _capi.BF16 if dtype == BF16 else _capi.F32
    av, wv = a.values, w.values
    _capi.check(_capi.lib().convnn_b200_linear_fp8(
        av.data_ptr(), av.stride(0), a.scales.data_ptr(), *a.scales.stride(), wv.data_ptr(), wv.stride(0), w.scales.data_ptr(),
        *w.scales.stride(), code, None, res.data_ptr(), N, res.data_ptr(), N, None, 0, 0, M, N, K, 0,
        torch.cuda.current_stream().cuda_stream))
    assert torch.equal(res, want)


def test_two_threads_at_once():
    import threading
    weights = mlp_weights(192, 768)
    xs = [randn(100 + 50 * i, 192, seed=i, dtype=BF16) for i in range(2)]
    want = [encoder_mlp(x, x, weights)[0] for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.no_grad(), torch.cuda.stream(st):
            for _ in range(50):
                got = encoder_mlp(xs[i], xs[i], weights)[0]
            st.synchronize()
            if not torch.equal(got, want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ---- refusals -------------------------------------------------------------------------------------------------------

def test_refusals():
    x, w = randn(4, 256, dtype=BF16), randn(256, dtype=BF16)
    a, b = operands(4, 130, 256)
    cases = [
        (TypeError, lambda: ops.rms_norm(x.half(), w.half())),
        (TypeError, lambda: ops.rms_norm(x, w.float())),
        (TypeError, lambda: ops.rms_norm(x, w, residual=x.float())),
        (ValueError, lambda: ops.rms_norm(x, w[:255])),
        (ValueError, lambda: ops.rms_norm(x, w, residual=x[:3])),
        (ValueError, lambda: ops.rms_norm(x, w, -1.0)),
        (ValueError, lambda: ops.rms_norm(x, w, float("nan"))),
        (ValueError, lambda: ops.rms_norm(x[:, :0], w[:0])),
        (RuntimeError, lambda: ops.rms_norm(x, w.cpu())),
        (RuntimeError, lambda: ops.rms_norm(x.cpu(), w.cpu())),
        (TypeError, lambda: ops.quantize_fp8(x.half())),
        (ValueError, lambda: ops.quantize_fp8(x, 64)),
        (ValueError, lambda: ops.quantize_fp8(x[None], 128)),
        (RuntimeError, lambda: ops.quantize_fp8(x.cpu())),
        (TypeError, lambda: ops.linear_fp8((x, a.scales), b)),
        (TypeError, lambda: ops.linear_fp8((a.values.view(torch.uint8), a.scales), b)),
        (TypeError, lambda: ops.linear_fp8((a.values, a.scales.double()), b)),
        (TypeError, lambda: ops.linear_fp8(a, b, dtype=torch.float16)),
        (ValueError, lambda: ops.linear_fp8((a.values, a.scales[:, :1]), b)),
        (ValueError, lambda: ops.linear_fp8((a.values, a.scales[:3]), b)),
        (ValueError, lambda: ops.linear_fp8((a.values[:, :200], a.scales), b)),
        (ValueError, lambda: ops.linear_fp8(a, (b.values, b.scales[:1]))),
        (ValueError, lambda: ops.linear_fp8(a, (b.values[:0], b.scales[:0]))),
        (ValueError, lambda: ops.linear_fp8(a, b, bias=randn(130))),
        (ValueError, lambda: ops.linear_fp8(a, b, bias=randn(131, dtype=BF16))),
        (ValueError, lambda: ops.linear_fp8(a, b, residual=randn(4, 131, dtype=BF16))),
        (ValueError, lambda: ops.linear_fp8(a, b, residual=randn(4, 130, dtype=BF16), dtype=F32)),
        (RuntimeError, lambda: ops.linear_fp8((a.values.cpu(), a.scales), b)),
        (RuntimeError, lambda: ops.linear_fp8(a, (b.values, b.scales.cpu()))),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            raise AssertionError(f"case {i} was taken")
    with torch.enable_grad():
        p = torch.nn.Parameter(w)
        for call in (lambda: ops.rms_norm(x, p), lambda: ops.quantize_fp8(x.clone().requires_grad_()),
                     lambda: ops.linear_fp8(a, b, bias=torch.nn.Parameter(randn(130, dtype=BF16)))):
            with pytest.raises(RuntimeError, match="forward-only"):
                call()
