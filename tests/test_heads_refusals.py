"""What the heads' norm and rotation, the paged cache and the attention over it refuse, on the CPU: no kernel is launched, and no pointer is
followed."""
import ctypes

import pytest
import torch

from convnn_b200 import _capi, ops

P = 1 << 20
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def heads(**kw):
    a = _capi.ConvnnHeads(_capi.BF16, 2, 3, 4, 2, 64, 64, 0, 100, 1e-6, P, P, P, (768, 256, 64), (384, 128, 64), (384, 128, 64), P, P, P, 64,
                          P, (3, 1), P, P, (768, 256, 64), (384, 128, 64))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def cache(**kw):
    c = _capi.ConvnnCache(P, P, (2048, 1024, 64), (2048, 1024, 64), P, 8, 16, 16, 8)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def attend(**kw):
    a = _capi.ConvnnTreeAttention(_capi.BF16, 2, 3, 4, 2, 64, 0.125, P, (768, 256, 64), P, P, P, (3, 1), P, (768, 256, 64))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def norm_rope(**kw):
    return _capi.lib().convnn_b200_qk_norm_rope(ctypes.byref(heads(**kw)), None)


def append(c=None, lengths=P, counts=P, **kw):
    return _capi.lib().convnn_b200_append_kv(ctypes.byref(heads(**kw)), ctypes.byref(cache(**(c or {}))), lengths, counts, None)


def attention(c=None, workspace=P, size=1 << 30, **kw):
    return _capi.lib().convnn_b200_tree_attention(ctypes.byref(attend(**kw)), ctypes.byref(cache(**(c or {}))), workspace, size, None)


HEADS = [
    (dict(dtype=2), _capi.E_INVALID), (dict(B=-1), _capi.E_INVALID), (dict(T=-1), _capi.E_INVALID), (dict(D=0), _capi.E_INVALID),
    (dict(Hq=0), _capi.E_INVALID), (dict(Hk=0), _capi.E_INVALID), (dict(D=257), _capi.E_UNSUPPORTED),
    (dict(B=1 << 20, T=1 << 20), _capi.E_UNSUPPORTED), (dict(Hq=1 << 21), _capi.E_UNSUPPORTED), (dict(eps=-1.0), _capi.E_INVALID),
    (dict(eps=float("nan")), _capi.E_INVALID), (dict(rotary=0), _capi.E_INVALID), (dict(rotary=33), _capi.E_INVALID),
    (dict(rotary=66), _capi.E_INVALID), (dict(rope_stride=63), _capi.E_INVALID), (dict(rope_rows=-1), _capi.E_INVALID),
    (dict(position_stride=(-1, 1)), _capi.E_INVALID), (dict(q=P + 1), _capi.E_ALIGN), (dict(k_weight=P + 1), _capi.E_ALIGN),
    (dict(rope=P + 2), _capi.E_ALIGN), (dict(positions=P + 2), _capi.E_ALIGN), (dict(dtype=_capi.F32, k=P + 2), _capi.E_ALIGN),
]


@pytest.mark.parametrize("kw,status", HEADS + [
    (dict(q=None), _capi.E_NULL), (dict(k=None), _capi.E_NULL), (dict(q_out=None), _capi.E_NULL), (dict(k_out=None), _capi.E_NULL),
    (dict(q=None, k=None, q_out=None, k_out=None), _capi.E_NULL)])
def test_qk_norm_rope(kw, status):
    assert norm_rope(**kw) == status
    assert _capi.lib().convnn_b200_last_error().decode()


@pytest.mark.parametrize("kw,status", HEADS + [
    (dict(k=None), _capi.E_NULL), (dict(v=None), _capi.E_NULL), (dict(q=None), _capi.E_NULL), (dict(q_out=None), _capi.E_NULL),
    (dict(lengths=None), _capi.E_NULL), (dict(lengths=P + 1), _capi.E_ALIGN), (dict(counts=P + 2), _capi.E_ALIGN),
    (dict(c=dict(k=None)), _capi.E_NULL), (dict(c=dict(v=None)), _capi.E_NULL), (dict(c=dict(table=None)), _capi.E_NULL),
    (dict(c=dict(pages=0)), _capi.E_INVALID), (dict(c=dict(page_size=0)), _capi.E_INVALID), (dict(c=dict(width=-1)), _capi.E_INVALID),
    (dict(c=dict(table_stride=-1)), _capi.E_INVALID), (dict(c=dict(k_stride=(2048, -64, 64))), _capi.E_INVALID),
    (dict(c=dict(page_size=1 << 20, width=2000)), _capi.E_UNSUPPORTED), (dict(c=dict(k=P + 1)), _capi.E_ALIGN),
    (dict(c=dict(table=P + 1)), _capi.E_ALIGN)])
def test_append_kv(kw, status):
    assert append(**kw) == status
    assert _capi.lib().convnn_b200_last_error().decode()


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=5), _capi.E_INVALID), (dict(B=-1), _capi.E_INVALID), (dict(T=-2), _capi.E_INVALID), (dict(Hq=5), _capi.E_INVALID),
    (dict(Hk=0), _capi.E_INVALID), (dict(D=0), _capi.E_INVALID), (dict(T=65), _capi.E_UNSUPPORTED), (dict(D=264), _capi.E_UNSUPPORTED),
    (dict(scale=float("inf")), _capi.E_INVALID), (dict(scale=float("nan")), _capi.E_INVALID), (dict(q=None), _capi.E_NULL),
    (dict(out=None), _capi.E_NULL), (dict(lengths=None), _capi.E_NULL), (dict(q=P + 2), _capi.E_ALIGN), (dict(out=P + 8), _capi.E_ALIGN),
    (dict(D=60), _capi.E_ALIGN), (dict(q_stride=(768, 256, 60)), _capi.E_ALIGN), (dict(out_stride=(764, 256, 64)), _capi.E_ALIGN),
    (dict(c=dict(k=P + 8)), _capi.E_ALIGN), (dict(c=dict(v_stride=(2048, 1024, 68))), _capi.E_ALIGN),
    (dict(q_stride=(-768, 256, 64)), _capi.E_INVALID), (dict(tree_stride=(3, -1)), _capi.E_INVALID), (dict(tree=P + 4), _capi.E_ALIGN),
    (dict(lengths=P + 2), _capi.E_ALIGN), (dict(workspace=P + 8), _capi.E_ALIGN), (dict(c=dict(table=None)), _capi.E_NULL),
    (dict(Hq=1 << 21), _capi.E_UNSUPPORTED)])
def test_tree_attention(kw, status):
    assert attention(**kw) == status
    assert _capi.lib().convnn_b200_last_error().decode()


def test_no_structs():
    L = _capi.lib()
    assert L.convnn_b200_qk_norm_rope(None, None) == _capi.E_NULL
    assert L.convnn_b200_append_kv(None, ctypes.byref(cache()), P, P, None) == _capi.E_NULL
    assert L.convnn_b200_append_kv(ctypes.byref(heads()), None, P, P, None) == _capi.E_NULL
    assert L.convnn_b200_tree_attention(None, ctypes.byref(cache()), P, 0, None) == _capi.E_NULL
    assert L.convnn_b200_tree_attention(ctypes.byref(attend()), None, P, 0, None) == _capi.E_NULL
    for bad in ((0, 4, 2, 64), (65, 4, 2, 64), (1, 5, 2, 64), (1, 4, 0, 64), (1, 4, 2, 0), (1, 4, 2, 257)):
        assert L.convnn_b200_tree_attention_workspace_bytes(_capi.BF16, *bad) == 0


# ---- from Python ----------------------------------------------------------------------------------------------------

@pytest.fixture
def on_any_device(monkeypatch):
    """The Python forms up to the launch; -> what was launched."""
    launched = []
    monkeypatch.setattr(ops, "_device_of", lambda *tensors: 0)
    monkeypatch.setattr(ops, "_launch", lambda index, fn, *args: launched.append(args))
    with torch.no_grad():
        yield launched


def t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def paged(pages=6, H=2, size=16, D=64, B=2, width=3, dtype=BF16):
    return ops.PagedCache(t(pages, H, size, D, dtype=dtype), t(pages, H, size, D, dtype=dtype), t(B, width, dtype=I32))


@pytest.mark.parametrize("call,error,match", [
    (lambda: ops.qk_norm_rope(None, None), ValueError, "queries or keys"),
    (lambda: ops.qk_norm_rope(t(64), None), ValueError, "heads"),
    (lambda: ops.qk_norm_rope(t(3, 4, 260), None), ValueError, "256"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), t(2, 2, 64)), ValueError, "k must be"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), t(3, 2, 32)), ValueError, "64 channels"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), t(3, 2, 64, dtype=F32)), TypeError, "one type"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64, dtype=torch.float16), None), TypeError, "float32 or bfloat16"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, t(64, dtype=F32)), TypeError, "q_weight"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), t(3, 2, 64), None, t(63)), ValueError, "k_weight"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, rope=t(3, 64)), TypeError, "rope"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, rope=t(3, 65, dtype=F32)), ValueError, "rope"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, rope=t(3, 66, dtype=F32)), ValueError, "rope"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, rope=t(64, dtype=F32)), ValueError, "rope"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, positions=t(3, dtype=torch.int64)), TypeError, "positions"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, positions=t(4, dtype=I32)), ValueError, "positions"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, out=(t(3, 4, 64, dtype=F32), None)), ValueError, "result"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, out=(t(1, 4, 64).expand(3, 4, 64), None)), ValueError, "overlap"),
    (lambda: ops.qk_norm_rope(t(3, 4, 64), None, out=(t(3, 64, 4).transpose(1, 2), None)), ValueError, "side by side"),
    (lambda: ops.append_kv(paged(), t(2, 2, 64), t(2, 2, 64), t(2, dtype=I32)), ValueError, "keys must be"),
    (lambda: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 1, 3, 64), t(2, dtype=I32)), ValueError, "v must have"),
    (lambda: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 2, 2, 64), t(2, dtype=I32)), ValueError, "v must be"),
    (lambda: ops.append_kv(paged(H=3), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)), ValueError, "cache"),
    (lambda: ops.append_kv(paged(dtype=F32), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)), TypeError, "cache"),
    (lambda: ops.append_kv(paged(B=3), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)), ValueError, "table"),
    (lambda: ops.append_kv(paged()._replace(table=t(2, 3, dtype=torch.int64)), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)), TypeError,
     "table"),
    (lambda: ops.append_kv(paged()._replace(k=t(1, 2, 16, 64).expand(6, 2, 16, 64)), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)),
     ValueError, "overlap"),
    (lambda: ops.append_kv(paged()._replace(v=t(6, 2, 64, 16).transpose(2, 3)), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32)), ValueError,
     "side by side"),
    (lambda: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=torch.int64)), TypeError, "lengths"),
    (lambda: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 1, 2, 64), t(3, dtype=I32)), ValueError, "lengths"),
    (lambda: ops.append_kv(paged(), t(2, 1, 2, 64), t(2, 1, 2, 64), t(2, dtype=I32), counts=t(3, dtype=I32)), ValueError, "counts"),
    (lambda: ops.tree_attention(t(2, 4, 64), paged(), t(2, dtype=I32)), ValueError, "queries must be"),
    (lambda: ops.tree_attention(t(2, 65, 4, 64), paged(), t(2, dtype=I32)), ValueError, "64 drafted"),
    (lambda: ops.tree_attention(t(2, 1, 5, 64), paged(), t(2, dtype=I32)), ValueError, "evenly"),
    (lambda: ops.tree_attention(t(2, 1, 4, 60), paged(D=60), t(2, dtype=I32)), ValueError, "multiple of 8"),
    (lambda: ops.tree_attention(t(2, 1, 4, 62, dtype=F32), paged(D=62, dtype=F32), t(2, dtype=I32)), ValueError, "multiple of 4"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64), paged(D=68)._replace(k=t(6, 2, 16, 68)[..., :64], v=t(6, 2, 16, 68)[..., :64]), t(2, dtype=I32)),
     ValueError, "16-byte"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64, dtype=F32), paged(), t(2, dtype=I32)), TypeError, "cache"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64), paged(), t(2, dtype=I32), t(2, 1, dtype=I32)), TypeError, "tree"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64), paged(), t(2, dtype=I32), t(2, 2, dtype=torch.int64)), ValueError, "tree"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64), paged(), t(2, dtype=I32), out=t(2, 1, 4, 32)), ValueError, "out"),
    (lambda: ops.tree_attention(t(2, 1, 4, 64), ops.PagedCache(*(torch.empty(1, 2, 1 << 20, 64, dtype=BF16, device="meta") for _ in range(2)),
                                               t(2, 2000, dtype=I32)), t(2, dtype=I32)), ValueError, "2\\^30"),
])
def test_from_python(on_any_device, call, error, match):
    with pytest.raises(error, match=match):
        call()
    assert not on_any_device


@pytest.mark.parametrize("which", range(3))
def test_no_cpu_path_and_no_gradient(which):
    q, k, w = t(2, 1, 4, 64), t(2, 1, 2, 64), t(64)
    call = [lambda: ops.qk_norm_rope(q, k, w, w), lambda: ops.append_kv(paged(), k, k, t(2, dtype=I32), q=q, q_weight=w),
            lambda: ops.tree_attention(q, paged(), t(2, dtype=I32))][which]
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        call()
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="forward-only"):
        call()
