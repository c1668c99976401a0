"""linear_w4 with more rows than one call of the library takes."""
import types

import pytest
import torch

from helixml_amd import _ffi, ssm
from tests.test_w4_gpu import random_weights

LIMIT = 32 * 65535


def test_rows_are_cut_where_a_call_ends(monkeypatch):
    """Every row once, each call within what hx_linear_w4 takes, operands and strides those of the rows."""
    calls = []
    monkeypatch.setattr(_ffi, "call", lambda name, *a: calls.append((name, a)))
    here = types.SimpleNamespace(device=torch.device("cpu"), cuda_stream=0)
    for M, dtype in ((0, torch.float32), (1, torch.bfloat16), (LIMIT, torch.float32), (LIMIT + 1, torch.bfloat16), (2 * LIMIT + 7, torch.float32)):
        calls.clear()
        X = torch.empty(M, 5, dtype=torch.bfloat16)[:, :2]
        out = torch.empty(M, 3, dtype=dtype)[:, :1]
        packed, scales = random_weights(1, 2, 0)
        assert ssm.linear_w4.__wrapped__(X, packed, scales, out=out, stream=here) is out
        at = 0
        for name, (m, n, k, x, ldx, w, s, bias, act, od, y, ldy, stream) in calls:
            assert name == "hx_linear_w4" and (n, k) == (1, 2) and 0 <= m <= LIMIT
            assert x == X.data_ptr() + 10 * at and y == out.data_ptr() + 3 * out.element_size() * at
            assert m <= 1 or (ldx, ldy) == (5, 3)
            assert (w, s, bias, act, stream) == (packed.data_ptr(), scales.data_ptr(), None, 0, 0)
            at += m
        assert at == M and len(calls) == max(1, -(-M // LIMIT))


@pytest.mark.gpu
def test_more_rows_than_one_call_takes(dev):
    """2^21 rows, 64 of them again and again: each repetition has the bits of the 64."""
    packed, scales = (t.to(dev) for t in random_weights(5, 33, 7))
    X = torch.randn(64, 33, device=dev).to(torch.bfloat16)
    want = ssm.linear_w4(X, packed, scales, out_dtype=torch.float32)
    many = ssm.linear_w4(X.repeat(32768, 1), packed, scales, out_dtype=torch.float32).view(32768, 64, 5)
    assert (many == want).all()
