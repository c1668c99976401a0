"""The norm to 8 bits (hx_add_rmsnorm) where its arithmetic is at an end: rows of zeros without an eps."""
import pytest
import torch

from helixml_amd import lm, ssm
from tests.test_i8_gpu import F32

pytestmark = pytest.mark.gpu

DIMS = [100, 700, 2000, 6000, 20000]  # a wave, a block of either size and a block in passes to a row


@pytest.mark.parametrize("dim", DIMS)
def test_rows_of_zeros_without_eps(dev, dim):
    """Codes and scale are 0 where every product is, also with an eps of 0, and so is a product of such a row. The other rows are what
    they are alone."""
    x, w = torch.randn(5, dim, generator=torch.Generator().manual_seed(dim)).to(dev), torch.ones(dim, device=dev)
    x[1] = 0
    x[3], w[dim // 2] = 0, 0
    x[3, dim // 2] = 2.0  # a row that only its weight makes zero
    for weight in (w, None):
        codes, scales = lm.add_rmsnorm(x, weight, eps=0.0)
        zero = [1, 3] if weight is not None else [1]
        assert not scales[zero].any() and not codes[zero].any(), scales
        packed, sw = ssm.i8_quantize(torch.ones(3, dim), device=dev)
        assert not ssm.linear_i8(codes, scales, packed, sw, out_dtype=F32)[zero].any()
        for i in range(5):
            one, s = lm.add_rmsnorm(x[i: i + 1], weight, eps=0.0)
            assert torch.equal(codes[i], one[0]) and torch.equal(scales[i], s[0]) and (i in zero or s[0] > 0)
