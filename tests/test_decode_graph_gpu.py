"""A captured decode step owns what its launches read: the operands of ``adjust`` and the model's weights."""
import gc
import weakref

import pytest
import torch

from helixml_amd import lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantized", [False, True])
def test_a_step_keeps_what_it_was_captured_with(dev, quantized):
    """The caller's dict gets other tensors, the model is dropped and its memory written over: replays still give what
    decode_step gave with the captured ones."""
    bt, V = 3, 256
    g = torch.Generator().manual_seed(1)
    make = lambda: lm.ByteLM(n_layers=2, d_model=64, device=dev, seed=5)  # noqa: E731
    m, twin = make(), make()
    if quantized:
        m.quantize_head()
        twin.quantize_head()
    kw = dict(history=torch.randint(0, V, (bt, 20), generator=g, dtype=torch.int32).to(dev),
              lengths=torch.full((bt,), 20, device=dev, dtype=torch.int32),
              repetition=torch.full((bt,), 1.7, device=dev), bias=torch.randn(V, generator=g).to(dev),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (8,), generator=g, dtype=torch.int64).to(torch.int32).to(dev))
    own = {k: v.clone() for k, v in kw.items()}
    step = m.decode_graph(m.new_state(bt), adjust=kw)
    held = [weakref.ref(t) for t in (*kw.values(), m.embed, m.norm_f, m.w_head, *m.layers[1].values())]
    sizes = [t.numel() * t.element_size() for t in (r() for r in held)]
    m.layers[1].clear()
    for k in list(kw):
        kw[k] = torch.zeros_like(kw[k])
    kw.pop("bias")
    del m
    gc.collect()
    assert all(r() is not None for r in held)
    junk = [torch.full((n,), 255, device=dev, dtype=torch.uint8) for n in sizes for _ in range(8)]
    state = twin.new_state(bt)
    for n in range(4):
        tok = torch.randint(0, V, (bt,), generator=g, dtype=torch.int32).to(dev)
        got = step(tok)
        torch.cuda.synchronize()
        assert torch.equal(got, twin.decode_step(tok, state, adjust=own)), n
    del junk
