"""The norm to 8 bits (hx_add_rmsnorm) where its arithmetic is at an end: rows of zeros without an eps, ties between products that fill
48 bits, factors that 32 bits do not hold. Codes are compared with the definition in whole numbers, outputs with float64."""
import numpy as np
import pytest
import torch

from helixml_amd import lm, ssm
from tests.test_i8_gpu import BF16, F32, HALF, I8, definition

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


def whole_codes(r, w):
    """round(127 p / max |p|), ties to even, of whole r and w of at most 24 bits: every step in whole numbers of at most 56 bits."""
    p = r.astype(np.int64) * w.astype(np.int64)
    top = np.abs(p).max(1, keepdims=True)
    code, rest = np.divmod(127 * np.abs(p), top)
    up = (2 * rest > top) | ((2 * rest == top) & (code % 2 == 1))
    return (np.sign(p) * (code + up)).astype(np.int8)


@pytest.mark.parametrize("dim", DIMS)
def test_ties_of_products_of_48_bits(dev, dim):
    """Ties go to the even code also where 127 p does not fit the 53 bits of a double: every border c + 1/2, both signs, and values
    next to one, in columns with one weight and with weights that make up for their halves."""
    g = np.random.default_rng(dim)
    rows = 64
    a = g.integers(1 << 15, 1 << 16, (rows, 1)) | 1
    c = np.arange(dim) % 127
    r = (2 * c + 1) * a * g.choice([-1, 1], (rows, dim))
    odd = g.random((rows, dim)) < 0.1
    r = np.where(odd, r + g.integers(-1, 2, r.shape), r)
    r[:, dim // 3] = 254 * a[:, 0]
    w = np.full(dim, int(g.integers(1 << 23, 1 << 24)) | 1)
    half = g.random(dim) < 0.3
    half[dim // 3] = False
    w2, r2 = np.where(half, w * 2, w).astype(np.float64) / 2, r  # p / 2 of the others: ties at other borders
    for weight, x, whole_w in ((w.astype(np.float64), r, w), (w2, r2, np.where(half, 2 * w, w))):
        want = whole_codes(x, whole_w)
        for scale in (1.0, 2.0 ** -30, 2.0 ** 60):
            X, W = torch.from_numpy(x.astype(np.float32) * np.float32(scale)), torch.from_numpy(weight.astype(np.float32))
            assert np.array_equal(W.double().numpy(), weight) and np.array_equal(X.double().numpy() / scale, x)
            codes, _ = lm.add_rmsnorm(X.to(dev), W.to(dev))
            assert np.array_equal(codes.cpu().numpy(), want), int((codes.cpu().numpy() != want).sum())


@pytest.mark.parametrize("out_dtype", [BF16, F32, I8], ids=["bf16", "f32", "i8"])
@pytest.mark.parametrize("dim", DIMS)
def test_factors_past_32_bits(dev, dim, out_dtype):
    """Rows so small or large that 1 / rms leaves what 32 bits hold (with an eps of 0), and products that do while the outputs do not."""
    g = torch.Generator().manual_seed(dim)
    n = lambda: torch.randn(4, dim, generator=g)  # noqa: E731
    spread = 10.0 ** (torch.rand(dim, generator=g) * 16 - 13)
    spread[0] = 1e3
    for x, w in ((n() * 1e-42, torch.full((dim,), 1e30)), (torch.sign(n()) * 3e38, torch.full((dim,), 1e-30)), (n() * 1e-32, spread),
                 (n() * 1e30, 1e-6 / spread)):
        _, p, inv = definition(x, w, None, eps=0.0)
        y = lm.add_rmsnorm(x.to(dev), w.to(dev), eps=0.0, out_dtype=out_dtype)
        if out_dtype == I8:
            top = np.abs(p).max(1)
            assert np.array_equal(y[0].cpu().numpy(), np.rint(p * 127.0 / top[:, None]).astype(np.int8))
            got, want, half = y[1], top * inv / 127.0, 2.0 ** -24
        else:
            got, want, half = y, p * inv[:, None], HALF[out_dtype]
        # bf16's products may be formed in 32 bits, whose subnormals are off by 2^-150 before a factor of up to 2^9
        assert (np.abs(got.double().cpu().numpy() - want) <= half * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -134 + 2.0 ** -141).all()
