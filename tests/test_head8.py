"""ByteLM's 8-bit head: it stands for what w_head holds, one rounded form is kept at a time, and its logits are those of the
rounded weights and the last norm's output in 8 bits, in prefill and decode alike."""
import numpy as np
import pytest
import torch

from helixml_amd import _ffi, lm, ssm
from tests.test_i8_gpu import HALF, product


def model(dev="cpu", **kw):
    return lm.ByteLM(n_layers=2, d_model=64, device=dev, **kw)


def test_new_weights_end_the_8_bit_form():
    for change in (lambda m, w: setattr(m, "w_head", w), lambda m, w: m.w_head.copy_(w)):
        m = model(seed=1)
        m.quantize_head(8)
        assert m.w_head8 is not None and m.w_head4 is None
        assert np.array_equal(m.host_params()["w_head"], ssm.i8_values(*m.w_head8, 64))
        change(m, model(seed=2).w_head)
        assert m.w_head8 is None and np.array_equal(m.host_params()["w_head"], m.w_head.float().numpy())


def test_one_form_at_a_time():
    m = model(seed=1)
    m.quantize_head()
    m.w_head8 = None  # there is none: the other stays
    assert m.w_head4 is not None
    m.quantize_head(8)
    assert m.w_head4 is None and m.w_head8 is not None
    m.w_head4 = None
    assert m.w_head8 is not None
    m.w_head8 = None
    assert m.w_head8 is None
    with pytest.raises(_ffi.InvalidInput):
        m.quantize_head(5)


@pytest.mark.gpu
def test_logits(dev):
    """The head's logits against the 8-bit product's definition on the codes that the last norm gives."""
    m = model(dev, seed=3)
    m.quantize_head(8)
    x = torch.randn(3, 40, 64, generator=torch.Generator().manual_seed(0)).to(dev)
    got = m._head(x, torch.cuda.current_stream()).cpu()
    codes, scales = lm.add_rmsnorm(x.view(120, 64), m.norm_f, eps=m.eps)
    packed, sw = m.w_head8
    w = torch.from_numpy(ssm.i8_values(packed, torch.ones_like(sw), 64)).to(torch.int8)
    want, bound = product(codes.cpu(), scales.cpu(), w, sw.cpu())
    assert (np.abs(got.double().numpy().reshape(120, -1) - want) <= bound + HALF[torch.float32] * (np.abs(want) + bound)).all()


@pytest.mark.gpu
def test_decode_agrees_with_prefill_and_replays(dev):
    """A decode step's logits are prefill's to the layers' own rounding, the head's rows bit for bit; a captured step replays
    to the eager one's bits, with eager work between the replays."""
    m = model(dev, seed=4)
    m.quantize_head(8)
    tokens = torch.randint(0, 256, (2, 21), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(dev)
    x = torch.randn(50, 64, device=dev)
    every = m._head(x, torch.cuda.current_stream())
    assert torch.equal(m._head(x[:3], torch.cuda.current_stream()), every[:3])
    _, state = m.prefill(tokens)
    copy = [(a.clone(), b.clone()) for a, b in state]
    step = m.decode_graph(state)
    for i in range(4):
        tok = torch.full((2,), 7 * i, dtype=torch.int32, device=dev)
        eager = m.decode_step(tok, copy)
        assert torch.equal(step(tok), eager), i
        torch.randn(1000, device=dev).sum()
    for (a, b), (c, d) in zip(state, copy):
        assert torch.equal(a, c) and torch.equal(b, d)
