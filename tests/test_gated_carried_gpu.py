"""The gated recurrence's state carried in one buffer: last_state is init_state, dinit is dlast."""
import pytest
import torch

from helixml_amd import _ffi, ssm
from tests.test_gated_gpu import inputs, to

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@TYPES
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("bt,L,dim", [(2, 0, 5), (3, 1, 7), (2, 128, 64), (3, 129, 65), (2, 1021, 130), (1, 4111, 66), (9, 2200, 33)])
def test_one_buffer_for_both_ends(dev, bt, L, dim, gate, dtype):
    x = to(dev, inputs(bt, L, dim, seed=L + 1, dtype=dtype, gate=gate))
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    s = torch.cuda.current_stream().cuda_stream
    out, last, states = ssm.gated_scan_fwd(x["x"], x["f"], x["z"], x["init"], return_last_state=True, return_states=True)
    grads = ssm.gated_scan_bwd(x["x"], x["f"], x["dout"], states, z=x["z"], dlast=x["dlast"])
    n = max(ssm.gated_scan_workspace_size(bt, L, dim, dtype), ssm.gated_scan_workspace_size(bt, L, dim, dtype, backward=True))
    ws = torch.empty(n, device=dev, dtype=torch.uint8)
    for _ in range(3):
        state, y = x["init"].clone(), torch.empty_like(out)
        _ffi.call("hx_gated_scan_fwd", bt, L, dim, ssm._STORAGE[dtype], p(x["x"]), p(x["f"]), p(x["z"]), p(state), p(y), p(state),
                  None, p(ws), n, s)
        assert torch.equal(state, last) and torch.equal(y, out)
        carry = x["dlast"].clone()
        dx, df = torch.empty_like(out), torch.empty_like(out)
        dz = torch.empty_like(out) if gate else None
        _ffi.call("hx_gated_scan_bwd", bt, L, dim, ssm._STORAGE[dtype], p(x["x"]), p(x["f"]), p(x["z"]), p(states), p(x["dout"]),
                  p(carry), p(dx), p(df), p(dz), p(carry), p(ws), n, s)
        for a, b in zip((dx, df, dz, carry), grads):
            assert (a is None and b is None) or torch.equal(a, b)
