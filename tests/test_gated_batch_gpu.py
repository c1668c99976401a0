"""A sequence's bits do not depend on what else is in the batch: each alone against the same one among others."""
import pytest
import torch

from tests.test_gated_gpu import inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bt,L,dim", [(4, 1500, 96), (70, 700, 65), (3, 100, 200)])
def test_a_sequence_alone_has_the_bits_that_it_has_in_a_batch(dev, bt, L, dim, dtype):
    x = inputs(bt, L, dim, seed=6, dtype=dtype)
    whole = run(dev, x)
    for b in sorted({0, 1, bt // 2, bt - 1}):
        alone = run(dev, {k: v[b: b + 1].contiguous() for k, v in x.items()})
        for k in whole:
            assert torch.equal(alone[k], whole[k][b: b + 1]), (b, k)
