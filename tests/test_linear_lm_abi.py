"""The decayed attention's, the norm's and the 8-bit products' entry points refuse bad arguments on the host, and weights
round to 8 bits on the host — no GPU needed."""
import ctypes

import numpy as np
import pytest
import torch

from helixml_amd import _ffi, lm, ssm

P = ctypes.c_void_p(4096)
SHAPE, DIM, DTYPE, INPUT, UNSUPPORTED = (c.status for c in (_ffi.ShapeMismatch, _ffi.InvalidDimension, _ffi.DTypeMismatch, _ffi.InvalidInput,
                                                              _ffi.UnsupportedOperation))


def fwd(bt=2, L=8, h=4, hq=4, hk=4, hv=4, dk=8, dv=8, dtype=0, q=P, ldq=None, k=P, ldk=None, v=P, ldv=None, decay=P, out=P, last=None, ws=None, n=0):
    ld = (hq * dk if ldq is None else ldq), (hk * dk if ldk is None else ldk), (hv * dv if ldv is None else ldv)
    return _ffi.lib().hx_decay_attention_fwd(bt, L, h, hq, hk, hv, dk, dv, dtype, q, ld[0], k, ld[1], v, ld[2], decay, 1.0, None, None, out, last, ws, n, None)


def bwd(bt=2, L=8, h=4, hq=4, hk=4, hv=4, dk=8, dv=8, dtype=0, q=P, ldq=None, k=P, ldk=None, v=P, ldv=None, decay=P, dout=P, dq=P, dk_out=P, dv_out=P,
        ws=None, n=0):
    ld = (hq * dk if ldq is None else ldq), (hk * dk if ldk is None else ldk), (hv * dv if ldv is None else ldv)
    return _ffi.lib().hx_decay_attention_bwd(bt, L, h, hq, hk, hv, dk, dv, dtype, q, ld[0], k, ld[1], v, ld[2], decay, 1.0, None, None, dout, None, dq,
                                             dk_out, dv_out, None, ws, n, None)


def step(bt=2, h=4, hq=4, hk=4, hv=4, dk=8, dv=8, dtype=0, state=P, q=P, ldq=None, k=P, ldk=None, v=P, ldv=None, decay=P, out=P):
    ld = (hq * dk if ldq is None else ldq), (hk * dk if ldk is None else ldk), (hv * dv if ldv is None else ldv)
    return _ffi.lib().hx_decay_attention_step(bt, h, hq, hk, hv, dk, dv, dtype, state, q, ld[0], k, ld[1], v, ld[2], decay, 1.0, out, None)


@pytest.mark.parametrize("call", [fwd, bwd, step])
def test_attention_sizes_and_types(call):
    for name in ("bt", "h", "hq", "hk", "hv", "dk", "dv"):
        assert call(**{name: -1}) == DIM, name
    for name in ("hq", "hk", "hv"):
        assert call(**{name: 3}) == SHAPE and call(**{name: 0}) == SHAPE and call(**{name: 8}) == SHAPE
    assert call(dtype=2) == DTYPE
    assert call(dk=0) == DIM and call(dv=0) == DIM
    assert call(dk=257) == UNSUPPORTED and call(dv=257) == UNSUPPORTED
    assert call(bt=2 ** 40) == UNSUPPORTED and call(h=2 ** 20, hq=1, hk=1, hv=1) == UNSUPPORTED and call(bt=2 ** 23, h=4) == UNSUPPORTED
    assert call(bt=0) == 0 and call(h=0, hq=0, hk=0, hv=0) == 0
    for name in ("ldq", "ldk", "ldv"):
        assert call(**{name: 31}) == INPUT, name
    if call is not step:
        assert call(L=-1) == DIM and call(L=2 ** 62) == UNSUPPORTED


@pytest.mark.parametrize("call", [fwd, bwd, step])
def test_attention_far_tokens(call):
    """A chunk's offsets are counted in 32 bits."""
    for name in ("ldq", "ldk", "ldv"):
        assert call(**{name: 2 ** 23}) == UNSUPPORTED, name
    assert call(h=2 ** 15, hq=1, hk=1, hv=1, dk=256) == UNSUPPORTED and call(h=2 ** 15, hq=1, hk=1, hv=1, dv=256) == UNSUPPORTED


def test_attention_missing_operands():
    for k in ("q", "k", "v", "decay", "out"):
        assert fwd(**{k: None}) == INPUT and step(**{k: None}) == INPUT
    assert step(state=None) == INPUT
    for k in ("q", "k", "v", "decay", "dout", "dq", "dk_out", "dv_out"):
        assert bwd(**{k: None}) == INPUT


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_workspace(dtype):
    """Where a workspace is needed, none, a short one and one that is not 16-byte aligned are refused."""
    code = ssm._STORAGE[dtype]
    for call, backward in ((fwd, False), (bwd, True)):
        need = ssm.decay_attention_workspace_size(1, 65536, 4, 8, 8, dtype, backward=backward)
        assert need > 0
        kw = dict(bt=1, L=65536, dtype=code)
        assert call(**kw) == INPUT and call(**kw, ws=P, n=need - 1) == INPUT and call(**kw, ws=ctypes.c_void_p(4104), n=need) == INPUT
    shared = ssm.decay_attention_workspace_size(1, 8, 4, 8, 8, dtype, backward=True, k_heads=1)
    assert shared >= 8 * 4 * 8 * 4
    assert bwd(bt=1, hk=1, dtype=code) == INPUT and bwd(bt=1, hk=1, dtype=code, ws=P, n=shared - 1) == INPUT
    assert ssm.decay_attention_workspace_size(8, 64, 64, 8, 8, dtype) == 0
    assert ssm.decay_attention_workspace_size(0, 64, 64, 8, 8, dtype) == 0 and ssm.decay_attention_workspace_size(4, 0, 64, 8, 8, dtype) == 0


def norm(rows=2, dim=8, dtype=0, x=P, ldx=8, ddtype=0, delta=None, ldd=8, weight=P, resid=None, ldr=8, out_dtype=2, y=P, ldy=8, scales=P):
    return _ffi.lib().hx_add_rmsnorm(rows, dim, dtype, x, ldx, ddtype, delta, ldd, weight, 1e-5, resid, ldr, out_dtype, y, ldy, scales, None)


def test_norm_refusals():
    assert norm(rows=-1) == DIM and norm(dim=-1) == DIM
    assert norm(dtype=2) == DTYPE and norm(dtype=-1) == DTYPE and norm(out_dtype=3) == DTYPE and norm(delta=P, ddtype=2) == DTYPE
    assert norm(rows=0) == 0 and norm(dim=0) == 0
    assert norm(x=None) == INPUT and norm(y=None) == INPUT and norm(scales=None) == INPUT
    assert norm(ldx=7) == INPUT and norm(ldy=7) == INPUT and norm(delta=P, ldd=7) == INPUT and norm(resid=P, ldr=7) == INPUT
    Q = ctypes.c_void_p(65536)
    assert norm(resid=P, ldr=9) == INPUT and norm(delta=Q, resid=Q, ldr=9) == INPUT  # in place with another stride
    assert norm(delta=Q, ddtype=1, resid=Q) == INPUT and norm(dtype=1, delta=Q, resid=Q) == INPUT  # or of another type
    assert norm(rows=1 << 40) == UNSUPPORTED and norm(rows=1 << 23, dim=4100, ldx=4100, ldy=4100) == UNSUPPORTED


def linear(M=2, N=8, K=8, X=P, ldx=8, sx=P, packed=P, scales=P, bias=None, act=0, out_dtype=0, Y=P, ldy=8):
    return _ffi.lib().hx_linear_i8(M, N, K, X, ldx, sx, packed, scales, bias, act, out_dtype, Y, ldy, None)


def test_linear_refusals():
    for k in ("M", "N", "K"):
        assert linear(**{k: -1}) == DIM
    assert linear(out_dtype=2) == DTYPE and linear(act=4) == INPUT and linear(act=-1) == INPUT
    assert linear(M=0) == 0 and linear(N=0) == 0
    for k in ("X", "sx", "packed", "scales", "Y"):
        assert linear(**{k: None}) == INPUT
    assert linear(ldx=7) == INPUT and linear(ldy=7) == INPUT and linear(packed=ctypes.c_void_p(4104)) == INPUT
    assert linear(K=1 << 17, ldx=1 << 17) == UNSUPPORTED and linear(N=1 << 28, ldy=1 << 28) == UNSUPPORTED and linear(M=1 << 30) == UNSUPPORTED


@pytest.mark.parametrize("n,k", [(1, 1), (16, 64), (17, 65), (5, 200), (33, 63)])
def test_quantize(n, k):
    """Codes are the nearest to 127 w / max|w|, ties to even; pieces hold them in the order of the header, zeros behind."""
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(n + k))
    w[0, 0] = 0
    if n > 2:
        w[1] = 0
        w[2, : min(k, 4)] = torch.tensor([2.0, 1.0, -1.0, 0.5])[:k]
        w[2, min(k, 4):] = 0
    packed, scales = ssm.i8_quantize(w, device="cpu")
    top = w.double().abs().amax(1, keepdim=True)
    want = torch.where(top > 0, torch.round(w.double() * 127 / torch.where(top > 0, top, 1.0)), 0.0)
    assert torch.equal(scales, (top / 127).float().squeeze(1))
    padded = torch.nn.functional.pad(want, (0, -k % 64, 0, -n % 16)).to(torch.int8)
    for i in range(padded.shape[0]):
        for j in range(padded.shape[1]):
            assert packed[i // 16, j // 64, j % 64 // 16, i % 16, j % 16] == padded[i, j]
    assert np.array_equal(ssm.i8_values(packed, scales, k), want.numpy().astype(np.float32) * scales.numpy()[:, None])


def test_quantize_refusals():
    for bad in (float("nan"), float("inf")):
        w = torch.ones(3, 4)
        w[1, 2] = bad
        with pytest.raises(_ffi.InvalidInput):
            ssm.i8_quantize(w, device="cpu")
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.i8_quantize(torch.ones(3))
    assert _ffi.lib().hx_i8_quantize(-1, 4, None, None, None) == DIM and _ffi.lib().hx_i8_quantize(2, 4, None, P, P) == INPUT
    assert _ffi.lib().hx_i8_quantize(0, 4, None, None, None) == 0


class Launch:
    device = torch.device("cuda:0")
    cuda_stream = 0


def test_wrappers_refuse_host_tensors_and_shapes():
    """The wrappers' own checks, reached without a device."""
    call = lambda f, *a, **kw: f.__wrapped__(*a, stream=Launch, **kw)  # noqa: E731
    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(_ffi.ShapeMismatch):
        call(ssm.decay_attention_fwd, x[0], x, x, torch.zeros(4))
    with pytest.raises(_ffi.ShapeMismatch):
        call(ssm.decay_attention_fwd, x, x, x, torch.zeros(4, 1))
    with pytest.raises(_ffi.DTypeMismatch):
        call(ssm.decay_attention_fwd, x.half(), x, x, torch.zeros(4))
    with pytest.raises(_ffi.InvalidInput):
        call(ssm.decay_attention_fwd, x, x, x, torch.zeros(4))  # host tensors
    with pytest.raises(_ffi.ShapeMismatch):
        call(lm.add_rmsnorm, x)
    with pytest.raises(_ffi.DTypeMismatch):
        call(lm.add_rmsnorm, torch.zeros(2, 3).half())
    with pytest.raises(_ffi.DTypeMismatch):
        call(lm.add_rmsnorm, torch.zeros(2, 3), out_dtype=torch.float16)
    with pytest.raises(_ffi.DTypeMismatch):
        call(ssm.linear_i8, torch.zeros(2, 3), torch.zeros(2), torch.zeros(1), torch.zeros(4))
    with pytest.raises(_ffi.ShapeMismatch):
        call(ssm.linear_i8, torch.zeros(3, dtype=torch.int8), torch.zeros(2), torch.zeros(1), torch.zeros(4))
