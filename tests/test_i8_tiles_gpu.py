"""8-bit products (hx_linear_i8) of many rows, which go through tiles of 128 x 128 or 256 x 256 outputs, and of few rows by many outputs: all
output types and epilogues, remainders of every size, against sums in 64 bits. Bounds as in test_i8_gpu: the sum is exact, its conversion, the
scales' product, their product and the bias round by 2^-24 each; SiLU's exponential errs by an ulp and |y| 2^-23 of its argument, its
reciprocal by an ulp; adding to Y rounds once more; storage adds half a step."""
import pytest
import torch

from helixml_amd import ssm
from tests.test_i8_gpu import BF16, F32, HALF, I8, pieces

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


# 153, 128, 144 and 256 tiles of 128, 289 and 272 of 256: K that ends inside a tile of columns, at its end and one before, rows and outputs that end anywhere
MANY = [(2100, 1100, 1040, None), (2048, 1024, 256, None), (1933, 1039, 1037, 1040), (129, 16290, 130, 144), (4097, 4100, 4112, None), (4111, 4090, 4223, 4224),
        (4352, 4096, 4096, None)]


@pytest.mark.parametrize("out_dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,ldx", MANY)
def test_many_rows(dev, m, n, k, ldx, out_dtype):
    x, sx, w, sw, b, g = operands(dev, m, n, k, ldx)
    acc, p = sums(x, w), pieces(w)
    for bias, act in ((None, 0), (b, 1), (b, 2), (None, 3)):
        wide = torch.full((m, n + 5), 7.0, device=dev, dtype=out_dtype)  # rows that start at any element
        y = wide[:, 3: 3 + n]
        if act & 2:
            y.copy_(torch.randn(m, n, generator=g, device=dev))
        before = y.clone()
        got = ssm.linear_i8(x, sx, p, sw, bias=bias, act=act, out=y)
        check(got, acc, sx, sw, bias, act, before)
        assert (wide[:, :3] == 7).all() and (wide[:, 3 + n:] == 7).all()
        if act == 1:
            assert torch.equal(ssm.linear_i8(x, sx, p, sw, bias=bias, act=act, out_dtype=out_dtype), got)


@pytest.mark.parametrize("m,n,k,few", [(2100, 1100, 1040, (1, 16, 17, 64, 127, 300, 1000)), (4097, 4100, 4112, (1, 5, 33, 100, 500, 2048, 4000))])
def test_rows_are_independent_of_tiles(dev, m, n, k, few):
    """A row's bits are the same from tiles and from the few rows' kernel."""
    x, sx, w, sw, b, _ = operands(dev, m, n, k)
    p = pieces(w)
    every = ssm.linear_i8(x, sx, p, sw, bias=b, act=1, out_dtype=F32)
    for i in few:
        assert torch.equal(ssm.linear_i8(x[:i], sx[:i], p, sw, bias=b, act=1, out_dtype=F32), every[:i]), i
        assert torch.equal(ssm.linear_i8(x[-i:], sx[-i:], p, sw, bias=b, act=1, out_dtype=F32), every[-i:]), i


def test_few_rows_of_a_large_vocabulary(dev):
    """One token's and a serving batch's logits over 131072 entries."""
    x, sx, w, sw, _, _ = operands(dev, 300, 131072, 4096)
    acc, p = sums(x, w), pieces(w)
    for m in (1, 16, 17, 64, 128, 129, 300):
        check(ssm.linear_i8(x[:m], sx[:m], p, sw, out_dtype=F32), acc[:m], sx[:m], sw, None, 0, None)
