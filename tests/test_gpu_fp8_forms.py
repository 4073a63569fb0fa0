"""Which kernel of the 8-bit operators runs: a size on either side of every line of their rules, the kernel's name (and, for the
product, its CTAs) read from a captured launch, and the result of each against its formula.  Sizes are for 148 SMs.  Tolerances are those of
the operators' other tests."""
import pytest
import torch

from convnn_b200 import _capi, ops
from gpu_util import DEV, launches, on_148_sms
from test_gpu_fp8 import (BF16, F32, blocks_of, check_blocks, check_linear, norm_err, norm_exact, operands, plain_quantize, randn,
                          same_bytes)

pytestmark = [pytest.mark.gpu, on_148_sms]


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


def launched(fn, what):
    """(name, CTAs) of the one kernel of `what` that fn() launches."""
    (found,) = [(n, c) for n, c in launches(fn, "GRID").items() if what in n]
    return found


# ---- the product ----------------------------------------------------------------------------------------------------

def form(M, N, K):
    a, w = operands(M, N, K, seed=1)
    name, ctas = launched(lambda: ops.linear_fp8(a, w), "linear_fp8")
    return ("pair" if "linear_fp8_pair_kernel" in name else name.split("linear_fp8_kernelILi")[1].split("EEEv")[0]), ctas


W16, W32, W64, T128 = "16ELb1", "32ELb1", "64ELb1", "128ELb0"        # columns of a tile, whether weights are its rows


@pytest.mark.parametrize("M,N,K,want,ctas", [
    # tokens as columns of a tile
    (16, 200, 128, W16, 2), (17, 200, 128, W32, 2), (32, 200, 128, W32, 2), (33, 200, 128, W64, 2), (64, 200, 128, W64, 2),
    # CTAs that share a sum: two blocks each at least
    (1, 100, 384, W16, 1), (1, 100, 385, W16, 2), (1, 100, 896, W16, 2), (1, 100, 897, W16, 4), (1, 100, 1920, W16, 4),
    (1, 100, 1921, W16, 8), (1, 100, 8000, W16, 8),
    # and an SM each
    (5, 37 * 128, 1024, W16, 148), (5, 37 * 128 + 1, 1024, W16, 76), (5, 74 * 128, 1024, W16, 148), (5, 74 * 128 + 1, 1024, W16, 75),
    # more tokens: weights as rows while that is one tile an SM and eight blocks of k a CTA
    (65, 74 * 128, 1024, W64, 148), (65, 74 * 128, 1025, T128, 148), (65, 74 * 128 + 1, 1024, T128, 75), (128, 128, 16 * 512, W64, 16),
    (197, 2304, 768, W64, 144), (100, 20001, 200, T128, 157), (1027, 1003, 1333, T128, 144),
    # pairs from 30 tiles of 256 x 256 on, with more than 128 rows
    (129, 29 * 256, 200, T128, 116), (129, 29 * 256 + 1, 200, "pair", 60), (128, 29 * 256 + 1, 200, W64, 118), (256, 30 * 256, 200, "pair", 60),
    (257, 15 * 256, 200, "pair", 60), (100, 20000, 200, T128, 157), (148 * 256, 256, 200, "pair", 148),
])
def test_the_product_takes_the_form_that_its_rule_says(M, N, K, want, ctas):
    assert form(M, N, K) == (want, ctas)


# sizes of each form whose output rows start anywhere, alone and with sums shared by a cluster; the ends of the lines above
@pytest.mark.parametrize("M,N,K", [(1027, 1003, 1333), (100, 20001, 200), (65, 74 * 128 + 1, 1024), (65, 9471, 1025), (129, 7424, 200),
                                   (129, 7423, 200), (129, 7425, 200), (257, 3841, 130), (128, 7425, 200), (5, 4737, 1024), (1, 101, 1921)])
@pytest.mark.parametrize("dtype,quantize", [(BF16, False), (F32, False), (BF16, True), (F32, True)])
def test_forms_against_the_formula(M, N, K, dtype, quantize):
    a, w = operands(M, N, K, seed=M + N)
    bias, res = randn(N, seed=8, dtype=dtype), randn(M, N, seed=9, dtype=dtype)
    check_linear(a, w, dtype=dtype, quantize=quantize)
    check_linear(a, w, bias, False, res, dtype, quantize)
    check_linear(a, w, bias, True, None, dtype, quantize)
    check_linear(a, w, bias, True, res, dtype, quantize)


# ---- the norm and the quantisers ------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,dtype,want", [
    (256, BF16, (1, 4, 1, 8)), (256, F32, (1, 2, 1, 8)), (255, BF16, (1, 2, 1, 1)), (254, BF16, (1, 2, 1, 2)), (264, BF16, (2, 1, 1, 8)),
    (512, F32, (2, 1, 1, 8)), (513, F32, (3, 1, 1, 1)), (768, BF16, (3, 1, 1, 8)), (769, BF16, (2, 1, 2, 1)), (770, F32, (2, 1, 2, 2)),
    (776, BF16, (4, 1, 1, 8)), (1024, F32, (4, 1, 1, 8)), (1023, F32, (2, 1, 2, 1)), (1032, BF16, (3, 1, 2, 8)), (1536, BF16, (3, 1, 2, 8)),
    (1544, BF16, (2, 1, 4, 8)), (2048, BF16, (2, 1, 4, 8)), (2056, BF16, (3, 1, 4, 8)), (2944, BF16, (3, 1, 4, 8)), (3080, BF16, (2, 1, 8, 8)),
    (1032, F32, (1, 1, 8, 8)), (1025, BF16, (1, 1, 8, 1)), (1026, BF16, (1, 1, 8, 2)), (2048, F32, (1, 1, 8, 8)), (2056, F32, (2, 1, 8, 8)),
    (2049, BF16, (2, 1, 8, 1)), (4096, BF16, (2, 1, 8, 8)), (4104, BF16, (3, 1, 8, 8)), (6144, F32, (3, 1, 8, 8)), (6152, BF16, (4, 1, 8, 8)),
    (8192, F32, (4, 1, 8, 8)), (8200, BF16, 8), (8193, F32, 1), (8194, BF16, 2)])
def test_the_norm_shares_a_row_as_its_rule_says(D, dtype, want):
    x, w, res = randn(5, D, seed=1, dtype=dtype), randn(D, seed=2, dtype=dtype), randn(5, D, seed=3, dtype=dtype)
    name, _ = launched(lambda: ops.rms_norm(x, w, residual=res, quantize=True), "rms_norm")
    kind = "f" if dtype == F32 else "13__nv_bfloat16"
    part = (f"rms_norm_wide_kernelI{kind}Li{want}E" if isinstance(want, int) else
            f"rms_norm_kernelI{kind}" + "".join(f"Li{v}E" for v in want))
    assert part in name, name
    q, s = ops.rms_norm(x, w, residual=res, quantize=True)
    exact = norm_exact(s, w, 1e-6)
    check_blocks(q, exact, norm_err(exact, D))


@pytest.mark.parametrize("D,dtype,want", [
    (128, BF16, (8, 1, 4)), (127, F32, (1, 1, 4)), (126, BF16, (2, 1, 4)), (136, BF16, (8, 2, 2)), (257, BF16, (1, 3, 2)), (512, F32, (8, 4, 1)),
    (520, BF16, (8, 3, 2)), (768, BF16, (8, 3, 2)), (776, BF16, (8, 4, 1)), (1152, F32, (8, 3, 2))])
def test_the_quantiser_groups_blocks_as_its_rule_says(D, dtype, want):
    x = randn(9, D, seed=1, dtype=dtype)
    name, _ = launched(lambda: ops.quantize_fp8(x), "quantize_rows")
    kind = "f" if dtype == F32 else "13__nv_bfloat16"
    assert f"quantize_rows_kernelI{kind}" + "".join(f"Li{v}E" for v in want) in name, name
    got, (q, scale) = ops.quantize_fp8(x), plain_quantize(x.float())
    assert same_bytes(got.values, q) and torch.equal(got.scales, scale) and scale.shape[1] == blocks_of(D)
