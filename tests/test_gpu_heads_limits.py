"""Calls of the heads' norm and rotation, the paged cache and the attention over it that their documentation allows and that lie at an edge:
tables without rows, values that are not finite under weights that vanish, tensors that autograd watches."""
import pytest
import torch

from convnn_b200 import _capi, ops
from heads_util import HALF, randn, turned
from test_gpu_tree_attention import cache_of, ints

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_grad():
    with torch.no_grad():
        yield
    assert _capi.device_status() == 0


@pytest.fixture(params=["host module", "Python"])
def both_ways(request, monkeypatch):
    """Every call by the host module, and through Python."""
    if request.param == "Python":
        monkeypatch.setattr(ops, "_calls", ops._GeneralCalls)


def check_turned_by_no_row(got, x, weight, R):
    """NaN in the channels that are turned; the others normed."""
    want, off = turned(x, weight, None, 1e-6, False)
    near = (got.double() - want).abs() <= HALF[x.dtype] * want.abs() + 1.01 * off
    assert torch.isnan(got[..., :R]).all() and near[..., R:].all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R", [64, 24, 2])
def test_a_rotation_table_without_rows(both_ways, dtype, R):
    """Every position is outside of it."""
    q, k = randn(2, 3, 4, 64, seed=1, dtype=dtype), randn(2, 3, 2, 64, seed=2, dtype=dtype)
    w, rope = randn(64, seed=3, dtype=dtype) + 1, torch.empty(0, R, device="cuda")
    for got, x in zip(ops.qk_norm_rope(q, k, w, w, rope), (q, k)):
        check_turned_by_no_row(got, x, w, R)
    cache = cache_of(2, 2, 16, 64, 60, dtype)
    got = ops.append_kv(cache, k, k, ints(5, 30), q=q, k_weight=w, q_weight=w, rope=rope)
    check_turned_by_no_row(got, q, w, R)
    for b, length in enumerate((5, 30)):
        for i in range(3):
            page, row = int(cache.table[b, (length + i) // 16]), (length + i) % 16
            check_turned_by_no_row(cache.k[page, :, row], k[b, i], w, R)
            assert torch.equal(cache.v[page, :, row], k[b, i])
