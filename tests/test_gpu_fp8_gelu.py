"""GELU of the 8-bit product's epilogue by itself: operands of zeros make every sum exactly zero, so that what is left is GELU of
the bias.

Tolerances.  Results of 8 or 16 bits are x - |x| Q(|x|) (x > 0) or -|x| Q(|x|), Q = 1 - Phi = exp2(-c a^2) R(a), a = |x|.  R is fitted to
3.1e-7 of itself; eight multiply-adds whose terms are at most twice their sum, a reciprocal and a power of two of one and two steps (2^-23
each) are under 2^-20 more: 2^-19 in all.  The exponent -c a^2 is rounded twice, 2^-24 of itself each, which is a^2 2^-24 of the power.  The rest
is a product and a sum, 2^-24 of x each for x > 0.  Results of 32 bits are 0.5 x (1 + erf(x / sqrt 2)), whose sum is off by 2^-23 (erf: two
steps of values up to one) and a rounding: 2^-22 |x|.  A bfloat16 rounding is 2^-8 of the value at most."""
import pytest
import torch

from convnn_b200 import _capi, ops
from convnn_b200.ops import Fp8Blocks
from gpu_util import DEV, launches
from test_gpu_fp8 import BF16, E4M3, F32, HALF, U, blocks_of, check_blocks, meant

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


# (M, N, K) of every form of the product, and its kernel
SHAPES = [(3, 1000, 128), (30, 1000, 128), (60, 1001, 300), (100, 2050, 200), (100, 20000, 200), (1027, 1003, 1333), (2000, 1100, 200),
          (300, 4001, 128)]


def zeros(rows, K, block_rows):
    room = torch.zeros(rows, (K + 15) // 16 * 16, dtype=torch.uint8, device=DEV).view(E4M3)
    return Fp8Blocks(room[:, :K], torch.ones((rows + block_rows - 1) // block_rows, blocks_of(K), device=DEV))


def gelu_of(bias, M, K, dtype, quantize=False, residual=None):
    return ops.linear_fp8(zeros(M, K, 1), zeros(bias.numel(), K, 128), bias=bias, gelu=True, residual=residual, dtype=dtype,
                          quantize=quantize)


def exact(x):
    """-> GELU in 64 bits, how far the 8- and 16-bit results' may be from it before they are rounded."""
    x = x.double()
    a = x.abs()
    tail = 0.5 * a * torch.special.erfcx(a * 0.5 ** 0.5) * torch.exp(-0.5 * a * a)     # (ndtr is zero from -8.3 on)
    return x.clamp(min=0) - tail, tail * (2.0 ** -19 + a * a * U) + 2 * U * x.clamp(min=0)


def sweep(N, dtype):
    return torch.linspace(-12.5, 8.0, N, device=DEV).to(dtype)


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_bfloat16_results(M, N, K):
    x = sweep(N, BF16)
    got = gelu_of(x, M, K, BF16)
    want, err = exact(x)
    assert torch.all((got.double() - want).abs() <= HALF[BF16] * want.abs() + 1.01 * err)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_8_bit_results(M, N, K, dtype):
    """Blocks from the far tail to the positive side: each has the scale of its own values."""
    x = sweep(N, dtype)
    want, err = exact(x)
    check_blocks(gelu_of(x, M, K, dtype, quantize=True), want.expand(M, N), err.expand(M, N))


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_float32_results(M, N, K):
    x = sweep(N, F32)
    want, _ = exact(x)
    assert torch.all((gelu_of(x, M, K, F32).double() - want).abs() <= 4 * U * x.double().abs())


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_infinities_and_nan_are_what_the_formula_gives(M, N, K):
    """x Phi(x) is NaN at -inf (in 32 bits too), x at inf."""
    for dtype in (BF16, F32):
        x = torch.full((N,), -1.0, device=DEV, dtype=dtype)
        x[5], x[300], x[600], x[700], x[701] = -INF, INF, NAN, torch.finfo(dtype).min, torch.finfo(dtype).max
        got = gelu_of(x, M, K, dtype)
        assert got[:, 5].isnan().all() and (got[:, 300] == INF).all() and got[:, 600].isnan().all()
        assert (got[:, 700] == 0).all() and (got[:, 701] == x[701]).all()
        rest = [n for n in range(N) if n not in (5, 300, 600, 700, 701)]
        assert torch.equal(got[:, rest], got[:1, rest].expand(M, -1)) and ((got[:, rest].float() + 0.15865526).abs() < 1e-3).all()
        q = gelu_of(x, M, K, dtype, quantize=True)
        assert q.scales[:, 0].isnan().all() and (q.scales[:, 300 // 128] == INF).all() and q.scales[:, 600 // 128].isnan().all()
        assert q.scales[:, 1].isfinite().all() and meant(q)[:, 128:256].isfinite().all() and meant(q)[:, 5].isnan().all()


def test_the_shapes_reach_every_form():
    forms = []
    for M, N, K in SHAPES:
        x = sweep(N, BF16)
        (name,) = [n for n in launches(lambda: gelu_of(x, M, K, BF16)) if "linear_fp8" in n]
        forms.append("pair" if "linear_fp8_pair_kernel" in name else name.split("linear_fp8_kernelILi")[1].split("E")[0])
    assert {"16", "32", "64", "128", "pair"} <= set(forms), forms


def test_the_residual_comes_after():
    M, N = 300, 4001
    x = sweep(N, F32)
    res = torch.linspace(-3, 3, M, device=DEV)[:, None] * torch.linspace(1, 2, N, device=DEV)
    got = gelu_of(x, M, 128, F32, residual=res)
    want, _ = exact(x)
    want = want + res.double()
    assert torch.all((got.double() - want).abs() <= 4 * U * x.double().abs() + U * want.abs())
