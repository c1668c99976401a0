"""ByteLM's 4-bit head stands for what w_head holds: new weights are never answered with the old ones' 4-bit form."""
import numpy as np
import pytest
import torch

from helixml_amd import lm, ssm
from tests.test_w4_gpu import expand

BF = torch.bfloat16


def model(dev="cpu", **kw):
    return lm.ByteLM(n_layers=1, d_model=64, device=dev, **kw)


def assign(m, w):
    m.w_head = w


def write(m, w):
    m.w_head.copy_(w)


def write_a_row(m, w):
    m.w_head[3] = w[3]


@pytest.mark.parametrize("change", [assign, write, write_a_row])
def test_new_weights_end_the_4_bit_form(change):
    m = model(seed=1)
    old = m.w_head.clone()
    m.quantize_head()
    assert m.w_head4 is not None and m.w_head4 is m.w_head4
    change(m, model(seed=2).w_head)
    assert not torch.equal(m.w_head, old)
    assert m.w_head4 is None
    assert np.array_equal(m.host_params()["w_head"], m.w_head.float().numpy())
    m.quantize_head()
    for a, b in zip(m.w_head4, ssm.w4_quantize(m.w_head)):
        assert torch.equal(a, b)


def test_a_head_in_use_ends_and_comes_back_by_hand():
    m = model(seed=1)
    pair = ssm.w4_quantize(m.w_head)
    m.w_head4 = pair
    assert m.w_head4 is pair
    m.w_head4 = None
    assert m.w_head4 is None


def test_weights_made_under_inference_mode():
    m = model(seed=1)
    with torch.inference_mode():
        m.w_head = m.w_head * 2
    m.quantize_head()
    assert m.w_head4 is not None
    m.w_head = m.w_head.clone()
    assert m.w_head4 is None


def test_host_params_are_the_weights_in_use():
    m = model(seed=3)
    m.quantize_head()
    assert np.array_equal(m.host_params()["w_head"], expand(*m.w_head4, 64))


def test_values_of_a_packed_pair():
    g = torch.Generator().manual_seed(0)
    for K in (1, 31, 32, 33, 100, 513):
        groups = -(-K // 32)
        packed = torch.randint(0, 256, (5, 16 * groups), generator=g, dtype=torch.uint8)
        scales = torch.randint(0, 250, (5, -(-groups // 16) * 16), generator=g, dtype=torch.uint8)
        # the least bytes' values are fp32 subnormals, exact too: one significant bit more than a power of two
        assert np.array_equal(ssm.w4_values(packed, scales, K).astype(np.float64), expand(packed, scales, K))
    scales[2, 0] = 255
    assert np.isnan(ssm.w4_values(packed, scales, K)[2, :32]).all()
    assert np.isfinite(ssm.w4_values(packed, scales, K)[:2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("change", [assign, write])
def test_logits_are_those_of_the_new_weights(dev, change):
    m, plain = model(dev, seed=1), model(dev, seed=1)
    m.quantize_head()
    w = model(dev, seed=2).w_head
    for t in (m, plain):
        change(t, w.clone())
    tokens = torch.randint(0, 256, (2, 30), dtype=torch.int32).to(dev)
    assert torch.equal(m.prefill(tokens)[0], plain.prefill(tokens)[0])
