"""8-bit products (hx_linear_i8) of few rows by many outputs against sums in 64 bits. Bounds as in test_i8_gpu: the sum is exact, its conversion, the
scales' product, their product and the bias round by 2^-24 each; SiLU's exponential errs by an ulp and |y| 2^-23 of its argument, its
reciprocal by an ulp; adding to Y rounds once more; storage adds half a step."""
import pytest
import torch

from helixml_amd import ssm
from tests.test_i8_gpu import F32, HALF, I8, pieces

pytestmark = pytest.mark.gpu


def operands(dev, m, n, k, ldx=None, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + m + n + k)
    whole = lambda *s: torch.randint(-127, 128, s, generator=g, device=dev, dtype=I8)  # noqa: E731
    x, w = whole(m, ldx or k)[:, :k], whole(n, k)
    rand = lambda n: torch.rand(n, generator=g, device=dev) + 0.5  # noqa: E731
    return x, rand(m), w, rand(n) / (5000.0 * k ** 0.5), torch.randn(n, generator=g, device=dev), g


def sums(x, w):
    """X . W^T in 64 bits, exact, some outputs at a time."""
    return torch.cat([x.double() @ part.double().t().contiguous() for part in w.split(1 << 14)], 1)


def check(got, acc, sx, sw, bias, act, y):
    by = sx.double()[:, None] * sw.double()
    v = acc * by
    e = v.abs() * 4 * 2.0 ** -24
    if bias is not None:
        v = v + bias.double()
        e = e + (v.abs() + bias.double().abs()) * 2.0 ** -24
    if act & 1:
        s = torch.sigmoid(v)
        e = e * 1.1 + (v * s).abs() * (v.abs() + 4) * 2.0 ** -22
        v = v * s
    if act & 2:
        v = v + y.double()
        e = e + (v.abs() + y.double().abs()) * 2.0 ** -24
    bad = ~((got.double() - v).abs() <= e + HALF[got.dtype] * (v.abs() + e) + 1e-30)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def test_few_rows_of_a_large_vocabulary(dev):
    """One token's and a serving batch's logits over 131072 entries."""
    x, sx, w, sw, _, _ = operands(dev, 300, 131072, 4096)
    acc, p = sums(x, w), pieces(w)
    for m in (1, 16, 17, 64, 128, 129, 300):
        check(ssm.linear_i8(x[:m], sx[:m], p, sw, out_dtype=F32), acc[:m], sx[:m], sw, None, 0, None)
