"""The gated recurrence's entry points refuse bad arguments on the host, and the wrappers' device check — no GPU needed."""
import ctypes
import types

import pytest
import torch

from helixml_amd import _ffi, ssm

P = ctypes.c_void_p(4096)


def fwd(bt=2, L=8, dim=4, dtype=0, x=P, f=P, z=None, init=None, out=P, last=None, states=None, ws=None, n=0):
    return _ffi.lib().hx_gated_scan_fwd(bt, L, dim, dtype, x, f, z, init, out, last, states, ws, n, None)


def bwd(bt=2, L=8, dim=4, dtype=0, x=P, f=P, z=None, states=P, dout=P, dlast=None, dx=P, df=P, dz=None, dinit=None, ws=None, n=0):
    return _ffi.lib().hx_gated_scan_bwd(bt, L, dim, dtype, x, f, z, states, dout, dlast, dx, df, dz, dinit, ws, n, None)


def step(bt=2, dim=4, dtype=0, state=P, x=P, f=P, z=None, out=P):
    return _ffi.lib().hx_gated_state_update(bt, dim, dtype, state, x, f, z, out, None)


def test_sizes_and_types():
    for call in (fwd, bwd, step):
        assert call(bt=-1) == _ffi.InvalidDimension.status
        assert call(dim=-1) == _ffi.InvalidDimension.status
        assert call(dtype=2) == _ffi.DTypeMismatch.status
        assert call(bt=2 ** 40, dim=2 ** 40) == _ffi.UnsupportedOperation.status
        assert call(bt=0) == 0 and call(dim=0) == 0
    for call in (fwd, bwd):
        assert call(L=-1) == _ffi.InvalidDimension.status
        assert call(L=2 ** 63 - 1) == _ffi.UnsupportedOperation.status
        assert call(dim=2 ** 63 - 1) == _ffi.UnsupportedOperation.status
        assert call(bt=2 ** 63 - 1) == _ffi.UnsupportedOperation.status
        assert call(L=2 ** 62) == _ffi.UnsupportedOperation.status
        assert call(L=0, x=None, f=None) == 0  # no steps, no state wanted: nothing to do


def test_missing_operands():
    for k in ("x", "f", "out"):
        assert fwd(**{k: None}) == _ffi.InvalidInput.status
    for k in ("x", "f", "states", "dout", "dx", "df"):
        assert bwd(**{k: None}) == _ffi.InvalidInput.status
    assert bwd(z=P) == _ffi.InvalidInput.status and bwd(dz=P) == _ffi.InvalidInput.status
    for k in ("state", "x", "f", "out"):
        assert step(**{k: None}) == _ffi.InvalidInput.status


@pytest.mark.parametrize("call,backward", [(fwd, False), (bwd, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_workspace(call, backward, dtype):
    """Where a workspace is needed, none, a short one and one that is not 16-byte aligned are refused."""
    sizes = [(1, 65536, 64), (1, 2048, 1536), (8, 2048, 1536), (1, 100, 64), (3, 1021, 1000)]
    for bt, L, dim in sizes:
        need = ssm.gated_scan_workspace_size(bt, L, dim, dtype, backward=backward)
        if need:
            kw = dict(bt=bt, L=L, dim=dim, dtype=ssm._STORAGE[dtype])
            assert call(**kw) == _ffi.InvalidInput.status
            assert call(**kw, ws=P, n=need - 1) == _ffi.InvalidInput.status
            assert call(**kw, ws=ctypes.c_void_p(4104), n=need) == _ffi.InvalidInput.status
    assert ssm.gated_scan_workspace_size(0, 5, 5, dtype, backward=backward) == 0
    assert ssm.gated_scan_workspace_size(5, 0, 5, dtype, backward=backward) == 0
    assert ssm.gated_scan_workspace_size(1, 1, 1 << 20, dtype, backward=backward) == 0


def test_tensors_of_another_device_are_refused():
    """A tensor's device has to be the launch stream's, whatever the current device is."""
    launch = types.SimpleNamespace(device=torch.device("cuda:0"))
    here = types.SimpleNamespace(device=torch.device("cuda:0"))
    there = types.SimpleNamespace(device=torch.device("cuda:1"))
    ssm._on_stream_device(launch, x=here, f=None)
    with pytest.raises(_ffi.DeviceMismatch):
        ssm._on_stream_device(launch, x=here, f=there)
