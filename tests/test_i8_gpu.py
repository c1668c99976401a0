"""The norm to 8 bits (hx_add_rmsnorm) and 8-bit products (hx_linear_i8) against their definitions in float64.

Bounds. hx_add_rmsnorm forms codes in 64 bits: they are the definition's own. A scale or an output is rounded once, half a step of
its type (bf16 through fp32: 2^-24 more). hx_linear_i8 sums exactly and rounds four times (the sum to fp32, the scales'
product, their product, the bias), 2^-24 each, of the magnitudes that it joins; SiLU's exponential errs by an ulp (2^-23) and |y| 2^-23 of its
argument, its reciprocal by an ulp; adding to Y rounds once more.
"""
import numpy as np
import pytest
import torch

from helixml_amd import _ffi, lm, ssm

pytestmark = pytest.mark.gpu

F32, BF16, I8 = torch.float32, torch.bfloat16, torch.int8
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8 * (1 + 2.0 ** -8)}
EPS = 1e-5


def definition(x, weight, delta, eps=EPS):
    """(r, p, 1 / rms) in float64."""
    r = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    d = r.double().numpy()
    inv = np.ones(d.shape[0]) if weight is None else 1.0 / np.sqrt((d * d).mean(1) + eps)
    return r, d if weight is None else d * weight.double().numpy(), inv


def codes_of(p, inv):
    top = np.abs(p).max(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(top[:, None] > 0, np.rint(p * 127.0 / top[:, None]), 0.0)
    return q.astype(np.int8), top * inv / 127.0


def check_norm(dev, x, weight, delta, out_dtype, resid=True):
    d = lambda t: None if t is None else t.to(dev)  # noqa: E731
    r, p, inv = definition(x, weight, delta)
    kept = torch.empty_like(d(x)) if resid else None
    y = lm.add_rmsnorm(d(x), d(weight), delta=d(delta), eps=EPS, out_dtype=out_dtype, resid=kept)
    if resid:
        assert torch.equal(kept.cpu(), r)
    if out_dtype == I8:
        q, s = codes_of(p, inv)
        assert np.array_equal(y[0].cpu().numpy(), q)
        assert (np.abs(y[1].double().cpu().numpy() - s) <= 2.0 ** -24 * s + 2.0 ** -150).all()
    else:
        want = p * inv[:, None]
        assert (np.abs(y.double().cpu().numpy() - want) <= HALF[out_dtype] * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -134).all()


@pytest.mark.parametrize("out_dtype", [I8, F32, BF16], ids=["i8", "f32", "bf16"])
@pytest.mark.parametrize("dim", [1, 3, 4, 63, 64, 255, 512, 513, 1023, 1024, 1500, 2048, 2049, 4096, 4099, 8192, 8195, 16384, 16385, 40001])
def test_norm(dev, dim, out_dtype):
    g = torch.Generator().manual_seed(dim)
    rows = 5 if dim > 2048 else 9
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    weight = 1 + 0.2 * n(dim)
    for xt, dt, w in ((F32, BF16, weight), (F32, F32, None), (BF16, F32, weight), (BF16, BF16, None), (F32, None, weight), (BF16, None, None)):
        check_norm(dev, (3 * n(rows, dim)).to(xt), w, None if dt is None else n(rows, dim).to(dt), out_dtype, resid=dt is not None)


def test_ties(dev):
    """x half of the largest is a tie (63.5) however the norm rounds: to the even code, with and without a norm."""
    x = torch.tensor([[2.0, 1.0, -1.0, 0.5], [3.0, 1.5, -1.5, 3.0], [254.0, 1.0, 3.0, -5.0], [1.0, 0.5, -0.5, 0.25], [254.0 * 0.3, 0.3, -127 * 0.3, 0.9]])
    for xt in (F32, BF16):
        for w in (None, torch.ones(4), torch.full((4,), 0.7), torch.full((4,), 3e-20)):
            check_norm(dev, x.to(xt), w, None, I8)
    q, _ = lm.add_rmsnorm(x.to(dev), torch.ones(4, device=dev))
    assert q[:4].cpu().tolist() == [[127, 64, -64, 32], [127, 64, -64, 127], [127, 0, 2, -2], [127, 64, -64, 32]]


def test_rows_of_zeros_and_not_finite(dev):
    x = torch.randn(6, 100)
    x[1] = 0
    x[2, 7], x[3, 99], x[4, 0] = float("nan"), float("inf"), -float("inf")
    x[5] = 1e-42  # denormal
    for w in (None, torch.ones(100), torch.cat((torch.zeros(1), torch.ones(99)))):
        q, s = lm.add_rmsnorm(x.to(dev), None if w is None else w.to(dev))
        assert torch.isnan(s[2:5]).all() and not q[1:5].any() and s[1] == 0 and torch.isfinite(s[[0, 1, 5]]).all()
        check_norm(dev, x[[0, 1, 5]], w, None, I8)
    y = lm.add_rmsnorm(x.to(dev), torch.ones(100, device=dev), out_dtype=F32)
    assert torch.isfinite(y[[0, 1, 5]]).all() and torch.isnan(y[2]).all() and not y[1].any()
    w = torch.ones(100)
    w[3] = float("inf")
    q, s = lm.add_rmsnorm(x[:1].to(dev), w.to(dev))
    assert torch.isnan(s).all() and not q.any()


@pytest.mark.parametrize("dim", [100, 3000, 20000])
def test_norm_in_place_and_strided(dev, dim):
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, delta, w = n(4, dim), n(4, dim).to(BF16), n(dim)
    r, p, inv = definition(x, w, delta)
    want, s = codes_of(p, inv)
    wide = lambda t, pad: torch.full((4, dim + pad), float("nan") if t.is_floating_point() else 99, dtype=t.dtype, device=dev)  # noqa: E731
    X, D, R, Y = wide(x, 3), wide(delta, 5), wide(x, 1), wide(torch.zeros(1, dtype=I8), 7)
    X[:, 1: 1 + dim], D[:, 3: 3 + dim] = x.to(dev), delta.to(dev)
    q, sc = lm.add_rmsnorm(X[:, 1: 1 + dim], w.to(dev), delta=D[:, 3: 3 + dim], resid=R[:, :dim], out=Y[:, 5: 5 + dim])
    assert np.array_equal(q.cpu().numpy(), want) and torch.equal(R[:, :dim].cpu(), r) and torch.isnan(R[:, dim:]).all()
    assert (Y[:, :5] == 99).all() and (Y[:, 5 + dim:] == 99).all()
    stream = x.to(dev)
    q, sc = lm.add_rmsnorm(stream, w.to(dev), delta=delta.to(dev), resid=stream)
    assert np.array_equal(q.cpu().numpy(), want) and torch.equal(stream.cpu(), r)
    assert (np.abs(sc.double().cpu().numpy() - s) <= 2.0 ** -24 * s).all()


# ------------------------------------------------------------------ products
def pieces(w):
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % 64, 0, -n % 16))
    return w.view(w.shape[0] // 16, 16, w.shape[1] // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous()


def whole(g, *s):
    return torch.randint(-127, 128, s, generator=g, dtype=I8)


def product(x, sx, w, sw, bias=None, act=0, y=None):
    """(result, bound of everything but its storage)."""
    acc = x.double().numpy() @ w.double().numpy().T
    by = sx.double().numpy()[:, None] * sw.double().numpy()
    v, e = acc * by, np.abs(acc * by) * 4 * 2.0 ** -24
    if bias is not None:
        v = v + bias.double().numpy()
        e = e + (np.abs(v) + np.abs(bias.double().numpy())) * 2.0 ** -24
    if act & 1:
        with np.errstate(over="ignore"):
            sg = 1.0 / (1.0 + np.exp(-v))
        e = e * (1.1 + 0.0 * sg) + np.abs(v * sg) * (np.abs(v) + 4) * 2.0 ** -22
        v = v * sg
    if act & 2:
        old = y.double().numpy()
        v = v + old
        e = e + (np.abs(v) + np.abs(old)) * 2.0 ** -24
    return v, e


def check_product(dev, m, n, k, out_dtype, bias=False, act=0, seed=0):
    g = torch.Generator().manual_seed(seed + m + n + k)
    x, w = whole(g, m, k), whole(g, n, k)
    sx, sw = torch.rand(m, generator=g) + 0.5, (torch.rand(n, generator=g) + 0.5) / (5000.0 * max(k, 1) ** 0.5)
    b = torch.randn(n, generator=g) if bias else None
    y = torch.randn(m, n, generator=g).to(out_dtype) if act & 2 else None
    want, bound = product(x, sx, w, sw, b, act, y)
    d = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = ssm.linear_i8(d(x), d(sx), d(pieces(w)), d(sw), bias=d(b), act=act, out_dtype=out_dtype, out=d(y))
    assert got.dtype == out_dtype and got.shape == (m, n)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound + HALF[out_dtype] * (np.abs(want) + bound) + 1e-30).all(), (float((err / (bound + HALF[out_dtype] * np.abs(want) + 1e-30)).max()))


SIZES = [(1, 1, 1), (1, 16, 64), (2, 17, 65), (3, 15, 63), (16, 64, 128), (17, 100, 130), (31, 48, 16), (33, 65, 1000), (48, 256, 512), (64, 128, 64),
         (65, 129, 192), (100, 300, 77), (128, 128, 256), (129, 257, 320), (255, 512, 1024), (300, 400, 1111), (512, 768, 640), (1000, 1030, 513)]


@pytest.mark.parametrize("out_dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(dev, m, n, k, out_dtype):
    for bias, act in ((False, 0), (True, 1), (True, 2), (False, 3)):
        check_product(dev, m, n, k, out_dtype, bias, act)


@pytest.mark.parametrize("m,n,k", [(1, 8192, 2048), (4, 4096, 8192), (48, 2048, 8192), (9, 32768, 4096), (2048, 1024, 2048), (4097, 2050, 272)])
def test_product_of_models_sizes(dev, m, n, k):
    check_product(dev, m, n, k, BF16, bias=True, act=1)


def test_largest_sums(dev):
    """K of 2^17 - 1 codes of -128 in X and 127 in W: the sums fill 32 bits."""
    k = (1 << 17) - 1
    for m in (1, 70):
        x, w = torch.full((m, k), -128, dtype=I8), torch.full((20, k), 127, dtype=I8)
        w[3] = -127
        got = ssm.linear_i8(x.to(dev), torch.ones(m, device=dev), pieces(w).to(dev), torch.ones(20, device=dev), out_dtype=F32)
        want = torch.full((m, 20), -128.0 * 127 * k, dtype=torch.float64)
        want[:, 3] *= -1
        assert torch.equal(got.cpu(), want.float())


def test_rows_are_independent(dev):
    """A row's bits do not depend on how many rows there are, whichever kernel takes them."""
    g = torch.Generator().manual_seed(5)
    x, w = whole(g, 700, 1040), whole(g, 515, 1040)
    sx, sw = torch.rand(700, generator=g).to(dev), torch.rand(515, generator=g).to(dev)
    b = torch.randn(515, generator=g).to(dev)
    d, p = x.to(dev), pieces(w).to(dev)
    every = ssm.linear_i8(d, sx, p, sw, bias=b, act=1, out_dtype=F32)
    for m in (1, 2, 5, 16, 17, 33, 64, 65, 130, 257, 699):
        assert torch.equal(ssm.linear_i8(d[:m], sx[:m], p, sw, bias=b, act=1, out_dtype=F32), every[:m]), m


@pytest.mark.parametrize("m", [1, 20, 300])
def test_strided_operands(dev, m):
    """Rows of X and Y from any byte and element on; what lies beside them stays as it was."""
    g = torch.Generator().manual_seed(m)
    n, k = 70, 200
    x, w = whole(g, m, k), whole(g, n, k)
    sx, sw = torch.rand(m, generator=g).to(dev), torch.rand(n, generator=g).to(dev)
    p = pieces(w).to(dev)
    for out_dtype in (F32, BF16):
        want = ssm.linear_i8(x.to(dev), sx, p, sw, out_dtype=out_dtype)
        for left, pad in ((1, 3), (5, 8), (0, 13)):
            X = torch.full((m, left + k + pad), 111, dtype=I8, device=dev)
            X[:, left: left + k] = x.to(dev)
            Y = torch.full((m, left + n + pad), 7.0, dtype=out_dtype, device=dev)
            ssm.linear_i8(X[:, left: left + k], sx, p, sw, out=Y[:, left: left + n])
            assert torch.equal(Y[:, left: left + n], want) and (Y[:, :left] == 7).all() and (Y[:, left + n:] == 7).all()


def test_scales_that_are_not_finite(dev):
    """A row of X whose scale is NaN becomes NaN throughout, the others stay."""
    g = torch.Generator().manual_seed(3)
    for m in (3, 200):
        x, w = whole(g, m, 100), whole(g, 40, 100)
        sx, sw = torch.rand(m, generator=g), torch.rand(40, generator=g)
        good = ssm.linear_i8(x.to(dev), sx.to(dev), pieces(w).to(dev), sw.to(dev), out_dtype=F32)
        sx[1] = float("nan")
        got = ssm.linear_i8(x.to(dev), sx.to(dev), pieces(w).to(dev), sw.to(dev), out_dtype=F32)
        assert torch.isnan(got[1]).all()
        keep = [i for i in range(m) if i != 1]
        assert torch.equal(got[keep], good[keep])


def test_empty(dev):
    p, s = ssm.i8_quantize(torch.randn(5, 7), device=dev)
    assert ssm.linear_i8(torch.empty(0, 7, dtype=I8, device=dev), torch.empty(0, device=dev), p, s).shape == (0, 5)
    p0, s0 = ssm.i8_quantize(torch.empty(5, 0), device=dev)
    y = ssm.linear_i8(torch.empty(3, 0, dtype=I8, device=dev), torch.ones(3, device=dev), p0, s0, bias=torch.arange(5.0, device=dev), out_dtype=F32)
    assert torch.equal(y.cpu(), torch.arange(5.0).repeat(3, 1))
    q, sc = lm.add_rmsnorm(torch.empty(0, 8, device=dev), torch.ones(8, device=dev))
    assert q.shape == (0, 8) and sc.shape == (0,)
