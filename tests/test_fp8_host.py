"""Refusals of the 8-bit operators' C entry points (no kernel is launched) and of their Python forms on CPU tensors."""
import pytest
import torch

from convnn_b200 import _capi, ops

P = 1 << 20                                                  # a pointer that is never followed: every call below is refused


def norm(dtype=_capi.BF16, x=P, ldx=8, res=None, ldr=0, w=P, eps=1e-6, s=None, lds=0, y=P, ldy=8, rows=2, D=8):
    return _capi.lib().convnn_b200_rms_norm(dtype, x, ldx, res, ldr, w, eps, s, lds, y, ldy, rows, D, None)


def norm8(dtype=_capi.BF16, x=P, ldx=8, res=None, ldr=0, w=P, eps=1e-6, s=None, lds=0, q=P, ldq=8, scales=P, row=1, block=2, rows=2,
          D=8):
    return _capi.lib().convnn_b200_rms_norm_fp8(dtype, x, ldx, res, ldr, w, eps, s, lds, q, ldq, scales, row, block, rows, D, None)


def quantize(dtype=_capi.BF16, x=P, ldx=8, block_rows=1, q=P, ldq=8, scales=P, row=1, block=2, rows=2, D=8):
    return _capi.lib().convnn_b200_quantize_fp8(dtype, x, ldx, block_rows, q, ldq, scales, row, block, rows, D, None)


def linear(a=P, lda=16, sa=P, sar=1, sab=2, w=P, ldw=16, sw=P, swr=1, swb=1, dtype=_capi.BF16, bias=None, res=None, ldr=0, out=P,
           ldo=8, so=None, sor=0, sob=0, M=2, N=8, K=16):
    return _capi.lib().convnn_b200_linear_fp8(a, lda, sa, sar, sab, w, ldw, sw, swr, swb, dtype, bias, res, ldr, out, ldo, so, sor,
                                              sob, M, N, K, 0, None)


@pytest.mark.parametrize("call,kw,status", [
    (norm, dict(dtype=2), _capi.E_INVALID), (norm, dict(x=None), _capi.E_NULL), (norm, dict(w=None), _capi.E_NULL),
    (norm, dict(y=None), _capi.E_NULL), (norm, dict(res=P, ldr=8), _capi.E_NULL), (norm, dict(s=P, lds=8), _capi.E_NULL),
    (norm, dict(ldx=7), _capi.E_INVALID), (norm, dict(ldy=7), _capi.E_INVALID), (norm, dict(D=0), _capi.E_INVALID),
    (norm, dict(D=(1 << 30) + 1, ldx=1 << 31, ldy=1 << 31), _capi.E_INVALID), (norm, dict(rows=-1), _capi.E_INVALID),
    (norm, dict(res=P, ldr=8, s=P, lds=7), _capi.E_INVALID), (norm, dict(res=P, ldr=7, s=P, lds=8), _capi.E_INVALID),
    (norm, dict(eps=-1.0), _capi.E_INVALID), (norm, dict(eps=float("nan")), _capi.E_INVALID),
    (norm, dict(x=P + 1), _capi.E_ALIGN), (norm, dict(dtype=_capi.F32, w=P + 2), _capi.E_ALIGN),
    (norm8, dict(q=None), _capi.E_NULL), (norm8, dict(scales=None), _capi.E_NULL), (norm8, dict(scales=P + 2), _capi.E_ALIGN),
    (norm8, dict(ldq=7), _capi.E_INVALID), (norm8, dict(row=0), _capi.E_INVALID), (norm8, dict(block=-2), _capi.E_INVALID),
    (quantize, dict(dtype=7), _capi.E_INVALID), (quantize, dict(x=None), _capi.E_NULL), (quantize, dict(q=None), _capi.E_NULL),
    (quantize, dict(scales=None), _capi.E_NULL), (quantize, dict(block_rows=2), _capi.E_INVALID),
    (quantize, dict(ldx=7), _capi.E_INVALID), (quantize, dict(ldq=7), _capi.E_INVALID), (quantize, dict(D=0), _capi.E_INVALID),
    (quantize, dict(x=P + 1), _capi.E_ALIGN), (quantize, dict(row=0), _capi.E_INVALID), (quantize, dict(rows=-1), _capi.E_INVALID),
    (linear, dict(dtype=2), _capi.E_INVALID), (linear, dict(a=None), _capi.E_NULL), (linear, dict(sa=None), _capi.E_NULL),
    (linear, dict(w=None), _capi.E_NULL), (linear, dict(sw=None), _capi.E_NULL), (linear, dict(out=None), _capi.E_NULL),
    (linear, dict(M=-1), _capi.E_INVALID), (linear, dict(N=0), _capi.E_INVALID), (linear, dict(K=0), _capi.E_INVALID),
    (linear, dict(K=17), _capi.E_INVALID), (linear, dict(ldo=7), _capi.E_INVALID), (linear, dict(res=P, ldr=7), _capi.E_INVALID),
    (linear, dict(M=(1 << 30) + 1), _capi.E_UNSUPPORTED), (linear, dict(a=P + 8), _capi.E_ALIGN), (linear, dict(lda=24), _capi.E_ALIGN),
    (linear, dict(w=P + 4), _capi.E_ALIGN), (linear, dict(ldw=24), _capi.E_ALIGN), (linear, dict(out=P + 1), _capi.E_ALIGN),
    (linear, dict(bias=P + 1), _capi.E_ALIGN), (linear, dict(sa=P + 1), _capi.E_ALIGN), (linear, dict(sw=P + 2), _capi.E_ALIGN),
    (linear, dict(sab=-1), _capi.E_INVALID), (linear, dict(swr=-1), _capi.E_INVALID), (linear, dict(so=P, sor=0, sob=1), _capi.E_INVALID),
    (linear, dict(so=P + 1, sor=1, sob=2), _capi.E_ALIGN),
])
def test_c_entry_points_refuse(call, kw, status):
    assert call(**kw) == status
    assert _capi.lib().convnn_b200_last_error().decode()


def test_no_cpu_path():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    q = (torch.zeros(2, 8).to(torch.float8_e4m3fn), torch.zeros(2, 1))
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.quantize_fp8(x), lambda: ops.linear_fp8(q, q)):
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call()
