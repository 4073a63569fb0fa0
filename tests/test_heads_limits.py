"""Sizes and tables at the edge of what heads, the paged cache and the attention over it take, and tensors that autograd watches, on the
CPU: no kernel is launched, and no pointer is followed."""
import pytest
import torch
from torch.autograd import forward_ad

from convnn_b200 import _capi, ops
from test_heads_refusals import I32, attention, on_any_device, paged, t  # noqa: F401


@pytest.mark.parametrize("B,T", [((1 << 30) + 1, 1), ((1 << 24) + 1, 64), (1 << 25, 64), ((1 << 31) - 1, 63), (17895698, 61)])
def test_attention_of_more_tokens_than_are_counted(B, T):
    """The rows of a call are counted in 32 bits."""
    assert B * T > 1 << 30
    assert attention(B=B, T=T) == _capi.E_UNSUPPORTED
    assert b"2^30 tokens" in _capi.lib().convnn_b200_last_error()


def test_attention_of_more_tokens_from_python(on_any_device):  # noqa: F811
    B, T = (1 << 24) + 1, 64
    cache = ops.PagedCache(t(1, 1, 16, 8), t(1, 1, 16, 8), t(1, 1, dtype=I32).expand(B, 1))
    with pytest.raises(ValueError, match="2\\^30 tokens"):
        ops.tree_attention(t(1, 1, 1, 8).expand(B, T, 1, 8), cache, t(1, dtype=I32).expand(B))
    assert not on_any_device


@pytest.mark.parametrize("call", [lambda rope: ops.qk_norm_rope(t(3, 4, 64), t(3, 2, 64), rope=rope),
                                  lambda rope: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32), rope=rope)])
def test_a_table_without_rows_is_a_table(on_any_device, call):  # noqa: F811
    """torch gives an empty table no address, and no address is no rotation."""
    call(torch.empty(0, 32))
    heads = on_any_device[0][0]._obj
    assert heads.rope and heads.rotary == 32 and heads.rope_rows == 0
    call(None)
    assert not on_any_device[1][0]._obj.rope


def test_what_is_written_moves_its_version(on_any_device):  # noqa: F811
    c, q, lengths = paged(), t(2, 1, 4, 64), t(2, dtype=I32)
    ops.append_kv(c, t(2, 1, 2, 64), t(2, 1, 2, 64), lengths)
    assert c.k._version > 0 and c.v._version > 0 and c.table._version == 0
    y, z = t(2, 1, 4, 64), t(2, 1, 4, 64)
    assert ops.qk_norm_rope(q, None, out=(y, None))[0] is y and y._version > 0 and q._version == 0
    with torch.enable_grad(), pytest.raises(RuntimeError, match="forward-only"):
        ops.qk_norm_rope(q, None, out=(z.requires_grad_(), None))
    # nothing is written
    c = paged()
    ops.append_kv(c, t(2, 0, 2, 64), t(2, 0, 2, 64), lengths)
    assert c.k._version == 0


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(10))
def test_tangents_are_refused(on_any_device, which, grad):  # noqa: F811
    """Forward-only is said of forward mode too: a result would come without its tangent.  torch.no_grad() does not end that mode."""
    q, k, w = t(2, 1, 4, 64), t(2, 1, 2, 64), t(64)
    lengths, c = t(2, dtype=I32), paged()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        calls = [lambda: ops.qk_norm_rope(dual(q), None), lambda: ops.qk_norm_rope(q, dual(k)), lambda: ops.qk_norm_rope(q, None, dual(w)),
                 lambda: ops.append_kv(c, dual(k), k, lengths), lambda: ops.append_kv(c._replace(v=dual(c.v)), k, k, lengths),
                 lambda: ops.append_kv(c, k, k, lengths, q=dual(q)), lambda: ops.tree_attention(dual(q), c, lengths),
                 lambda: ops.tree_attention(q, c._replace(k=dual(c.k)), lengths), lambda: ops.rms_norm(dual(t(3, 64)), w),
                 lambda: ops.quantize_fp8(dual(t(3, 64)))]
        with pytest.raises(RuntimeError, match="no tangents"):
            calls[which]()
        assert not on_any_device
        with forward_ad._set_fwd_grad_enabled(False):
            if 3 > which or which > 7:
                calls[which]()
                assert len(on_any_device) == 1
