"""4-bit weights with group scales: hx_w4_quantize (host) and hx_linear_w4 (device).

Two kinds of comparison. Whole-number activations and scales of one make every product and partial sum a multiple of
1/2 below 2^23, exact in fp32 in any order: outputs are equal bit for bit. With any values, K products summed in fp32 in
any order are off by at most K 2^-24 of the sum of their magnitudes, counted twice (2^-23) for accumulators that cut
instead of rounding; the epilogue adds 2^-22 of what it joins (silu: (|y| + 2) 2^-23 relative), storage half a step."""
import ctypes

import numpy as np
import pytest
import torch

from helixml_amd import _ffi, ssm

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def rows(K):
    g = -(-K // 32)
    return 16 * g, 16 * -(-g // 16)


def expand(packed, scales, K):
    """The weights that a packed pair stands for, in float64."""
    packed, scales = np.asarray(packed), np.asarray(scales)
    code = np.stack((packed & 15, packed >> 4), -1).reshape(packed.shape[0], -1)
    power = 2.0 ** (scales.astype(np.float64) - 127)
    return (VALUES[code] * np.repeat(power, 32, 1)[:, : code.shape[1]])[:, :K]


# ------------------------------------------------------------------ rounding (host)
def test_quantize_takes_the_nearest_code():
    """Every weight becomes the code nearest to it at its group's scale (ties to the even code), the scale puts the
    group's largest magnitude into [4, 8), and what has a code already comes back unchanged."""
    rng = np.random.default_rng(0)
    for K in (1, 2, 31, 32, 33, 64, 100, 512, 513):
        w = torch.from_numpy((rng.standard_normal((5, K)) * 10.0 ** rng.uniform(-3, 3, (5, 1))).astype(np.float32))
        packed, scales = ssm.w4_quantize(w)
        assert packed.shape == (5, rows(K)[0]) and scales.shape == (5, rows(K)[1])
        got = expand(packed, scales, K)
        for n in range(5):
            for g in range(-(-K // 32)):
                v = w[n, 32 * g: 32 * g + 32].double().numpy()
                power = 2.0 ** (int(scales[n, g]) - 127)
                assert 4 * power <= np.abs(v).max() < 8 * power
                d = np.abs(np.abs(v)[:, None] / power - VALUES[:8])
                assert (np.abs(np.abs(got[n, 32 * g: 32 * g + 32]) / power - np.abs(v) / power) == d.min(1)).all()
        assert (np.signbit(got) == np.signbit(w.numpy())).all()
        again = ssm.w4_quantize(torch.from_numpy(got.astype(np.float32)))
        assert np.array_equal(expand(*again, K), got)
        unused = np.stack((packed.numpy() & 15, packed.numpy() >> 4), -1).reshape(5, -1)[:, K:]
        assert (unused == 0).all() and (scales.numpy()[:, -(-K // 32):] == 127).all()


def test_quantize_ties_and_borders():
    mid = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.999]
    want = [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0]
    w = torch.tensor([mid + [-m for m in mid] + [4.0]])
    assert expand(*ssm.w4_quantize(w), w.shape[1])[0].tolist() == want + [-v for v in want] + [4.0]
    for top, code in ((0.0, 2), (1e-45, 2), (2.0 ** -123, 2), (2.0 ** -122, 3), (1.0, 125), (3.4e38, 252)):
        s = ssm.w4_quantize(torch.tensor([[top, 0.0]]))[1]
        assert int(s[0, 0]) == code, top


def test_quantize_refusals():
    for bad in (float("nan"), float("inf")):
        with pytest.raises(_ffi.InvalidInput):
            ssm.w4_quantize(torch.tensor([[1.0, bad]]))
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.w4_quantize(torch.zeros(3))
    assert _ffi.lib().hx_w4_quantize(-1, 4, None, None, None) == _ffi.InvalidDimension.status
    assert _ffi.lib().hx_w4_quantize(1, 4, None, None, None) == _ffi.InvalidInput.status
    assert _ffi.lib().hx_w4_quantize(0, 4, None, None, None) == 0


def test_linear_refusals():
    L, p = _ffi.lib(), ctypes.c_void_p(4096)
    call = lambda M=1, N=4, K=32, X=p, ldx=32, W=p, S=p, act=0, od=0, Y=p, ldy=4: L.hx_linear_w4(  # noqa: E731
        M, N, K, X, ldx, W, S, None, act, od, Y, ldy, None)
    assert call(M=-1) == _ffi.InvalidDimension.status
    assert call(od=2) == _ffi.DTypeMismatch.status
    assert call(act=4) == _ffi.InvalidInput.status
    assert call(X=None) == _ffi.InvalidInput.status
    assert call(Y=None) == _ffi.InvalidInput.status
    assert call(ldx=31) == _ffi.InvalidInput.status
    assert call(ldy=3) == _ffi.InvalidInput.status
    assert call(W=ctypes.c_void_p(4104)) == _ffi.InvalidInput.status
    assert call(S=ctypes.c_void_p(4097)) == _ffi.InvalidInput.status
    assert call(M=0) == 0 and call(N=0) == 0
    for big in (dict(N=2 ** 30, ldy=2 ** 30), dict(M=32 * 65535 + 1), dict(K=2 ** 26, ldx=2 ** 26), dict(ldx=2 ** 26)):
        assert call(**big) == _ffi.UnsupportedOperation.status


# ------------------------------------------------------------------ products (device)
SIZES = [(1, 1, 1), (1, 16, 32), (1, 17, 33), (2, 5, 64), (3, 100, 31), (1, 256, 512), (5, 160, 4096), (16, 64, 128), (17, 48, 96),
         (33, 70, 1000), (64, 130, 544), (65, 33, 256), (130, 40, 160), (1, 1000, 2080), (7, 4100, 512), (4, 300, 777),
         (2, 16400, 160), (6, 16390, 288), (16, 16400, 1100), (40, 16500, 640), (33, 16384, 96), (3, 32770, 264), (9, 4113, 1056), (20, 48, 4100), (31, 4120, 2500)]


def random_weights(N, K, seed, lo=120, hi=130):
    """Every code and padding nibble random, group exponents random, padding scale bytes NaN."""
    g = torch.Generator().manual_seed(seed)
    pr, sr = rows(K)
    packed = torch.randint(0, 256, (N, pr), generator=g, dtype=torch.uint8)
    scales = torch.full((N, sr), 255, dtype=torch.uint8)
    groups = -(-K // 32)
    scales[:, :groups] = torch.randint(lo, hi, (N, groups), generator=g, dtype=torch.uint8)
    return packed, scales


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", SIZES)
def test_whole_numbers_are_exact(dev, M, N, K):
    g = torch.Generator().manual_seed(M * N + K)
    packed, scales = random_weights(N, K, K)
    scales[:, : -(-K // 32)] = 127
    X = torch.randint(-8, 9, (M, K), generator=g).to(torch.bfloat16)
    want = X.double().numpy() @ expand(packed, scales, K).T
    got = ssm.linear_w4(X.to(dev), packed.to(dev), scales.to(dev), out_dtype=torch.float32)
    assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias,act", [(False, 0), (True, 1), (True, 2), (False, 3)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_and_epilogue(dev, M, N, K, bias, act, dtype):
    g = torch.Generator().manual_seed(N + K)
    packed, scales = random_weights(N, K, K + 1, 118, 127)
    X = torch.randn(M, K, generator=g).to(torch.bfloat16)
    b = torch.randn(N, generator=g) if bias else None
    y0 = torch.randn(M, N, generator=g).to(dtype)
    w = expand(packed, scales, K)
    want = X.double().numpy() @ w.T
    E = K * 2.0 ** -23 * (np.abs(X.double().numpy()) @ np.abs(w).T)
    if bias:
        want = want + b.double().numpy()
        E = E + 2.0 ** -23 * np.abs(want)
    if act & 1:
        s = 1 / (1 + np.exp(-want))
        E = 1.1 * E + np.abs(want * s) * (np.abs(want) + 2) * 2.0 ** -22  # |silu'| <= 1.0998
        want = want * s
    if act & 2:
        want = want + y0.double().numpy()
        E = E + 2.0 ** -23 * np.abs(want)
    # rows of X and Y strided, the columns around Y's left alone
    Xd = torch.zeros(M, K + 8, device=dev, dtype=torch.bfloat16)
    Xd[:, :K] = X.to(dev)
    Yd = torch.full((M, N + 3), 7.0, device=dev, dtype=dtype)
    Yd[:, :N] = y0.to(dev)
    ssm.linear_w4(Xd[:, :K], packed.to(dev), scales.to(dev), bias=None if b is None else b.to(dev), act=act, out=Yd[:, :N])
    got = Yd[:, :N].double().cpu().numpy()
    tol = E + HALF[dtype] * (np.abs(want) + E)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())
    assert (Yd[:, N:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(3, 40, 100), (20, 64, 512), (1, 33, 2048)])
def test_every_scale_byte(dev, M, N, K):
    """Scale bytes 0..252 are exact powers of two (one nonzero activation a row: each output is one product)."""
    packed, scales = random_weights(N, K, 5, 0, 253)
    X = torch.zeros(M, K, dtype=torch.bfloat16)
    at = torch.arange(M) * 31 % K
    X[torch.arange(M), at] = 1.0
    want = expand(packed, scales, K).T[at.numpy()]
    got = ssm.linear_w4(X.to(dev), packed.to(dev), scales.to(dev), out_dtype=torch.float32)
    assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("byte", [253, 254])
def test_scales_past_the_range_of_bf16(dev, byte):
    """What bf16 cannot hold becomes an infinity of its sign."""
    packed = torch.zeros(16, 16, dtype=torch.uint8)
    packed[:, 0] = torch.arange(16, dtype=torch.uint8)
    scales = torch.full((16, 16), 127, dtype=torch.uint8)
    scales[:, 0] = byte
    X = torch.zeros(1, 32, dtype=torch.bfloat16)
    X[0, 0] = 2.0 ** -10
    want = VALUES * 2.0 ** (byte - 127)
    want = np.where(np.abs(want) < 2.0 ** 128, want, np.copysign(np.inf, want)) * 2.0 ** -10
    got = ssm.linear_w4(X.to(dev), packed.to(dev), scales.to(dev), out_dtype=torch.float32)[0]
    assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.gpu
def test_subnormal_activations(dev):
    """A product of a subnormal activation is that number's, not nought's."""
    packed = torch.full((1, 16), 0x22, dtype=torch.uint8)  # ones
    scales = torch.full((1, 16), 227, dtype=torch.uint8)  # 2^100
    for e in (-126, -127, -130, -133):
        X = torch.zeros(1, 32, dtype=torch.bfloat16)
        X[0, 3] = 2.0 ** e
        assert ssm.linear_w4(X.to(dev), packed.to(dev), scales.to(dev), out_dtype=torch.float32).item() == 2.0 ** (e + 100)


@pytest.mark.gpu
def test_no_inner_elements(dev):
    """K = 0: the bias alone, or nothing."""
    packed, scales = torch.empty(5, 0, device=dev, dtype=torch.uint8), torch.empty(5, 0, device=dev, dtype=torch.uint8)
    X = torch.empty(3, 0, device=dev, dtype=torch.bfloat16)
    b = torch.randn(5, device=dev)
    assert torch.equal(ssm.linear_w4(X, packed, scales, bias=b, out_dtype=torch.float32), b.expand(3, 5))
    assert (ssm.linear_w4(X, packed, scales, out_dtype=torch.float32) == 0).all()


@pytest.mark.gpu
def test_unaligned_rows_of_x(dev):
    """Rows of X that start at any element, in a buffer whose other elements are NaN."""
    M, N, K = 7, 60, 300
    packed, scales = random_weights(N, K, 4)
    scales[:, : -(-K // 32)] = 127
    X = torch.randint(-8, 9, (M, K)).to(torch.bfloat16)
    want = X.double().numpy() @ expand(packed, scales, K).T
    for left, right in ((1, 0), (3, 2), (5, 8)):
        buf = torch.full((M, K + left + right), float("nan"), device=dev, dtype=torch.bfloat16)
        buf[:, left: left + K] = X.to(dev)
        got = ssm.linear_w4(buf[:, left: left + K], packed.to(dev), scales.to(dev), out_dtype=torch.float32)
        assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.gpu
def test_not_a_number(dev):
    """A NaN activation reaches its row alone, a NaN scale its column alone; what lies behind K, in X's rows and in the
    padding of the weights, reaches nothing."""
    M, N, K = 6, 50, 70
    packed, scales = random_weights(N, K, 3)
    X = torch.full((M, 96), float("nan"))
    X[:, :K] = torch.randn(M, K)
    X[2, 5] = float("nan")
    scales[9, 1] = 255
    got = ssm.linear_w4(X.to(dev, torch.bfloat16)[:, :K], packed.to(dev), scales.to(dev), out_dtype=torch.float32).cpu()
    nan = torch.isnan(got)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[2], want[:, 9] = True, True
    assert torch.equal(nan, want)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(160, 4096), (1000, 512), (4100, 2048), (33, 77), (16400, 544)])
def test_a_row_does_not_depend_on_the_batch(dev, N, K):
    packed, scales = (t.to(dev) for t in random_weights(N, K, 9))
    X = torch.randn(80, K).to(dev, torch.bfloat16)
    whole = ssm.linear_w4(X, packed, scales, out_dtype=torch.float32)
    for m in (1, 2, 4, 5, 16, 17, 33, 64, 79):
        assert torch.equal(ssm.linear_w4(X[:m], packed, scales, out_dtype=torch.float32), whole[:m]), m


@pytest.mark.gpu
def test_wrapper_refusals(dev):
    packed, scales = (t.to(dev) for t in random_weights(8, 64, 1))
    X = torch.zeros(2, 64, device=dev, dtype=torch.bfloat16)
    with pytest.raises(_ffi.DTypeMismatch):
        ssm.linear_w4(X.float(), packed, scales)
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.linear_w4(X[:, :32], packed, scales)
    with pytest.raises(_ffi.InvalidInput):
        ssm.linear_w4(X, packed, scales, act=2)
    with pytest.raises(_ffi.InvalidInput):
        ssm.linear_w4(torch.zeros(64, 2, device=dev, dtype=torch.bfloat16).t(), packed, scales)
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.linear_w4(X, packed, scales, out=torch.zeros(2, 9, device=dev))
    with pytest.raises(_ffi.DTypeMismatch):
        ssm.linear_w4(X, packed, scales, out_dtype=torch.float16)
    with pytest.raises(_ffi.InvalidInput):
        ssm.linear_w4(X, packed.cpu(), scales)


# ------------------------------------------------------------------ many outputs, many rows (device)
LARGE = [(13, 8250, 4200), (40, 9000, 2100), (9000, 40, 1100), (64, 16390, 1030)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", LARGE)
def test_large_products(dev, M, N, K):
    g = torch.Generator().manual_seed(M + N)
    packed, scales = random_weights(N, K, K)
    W = packed.to(dev)
    ones = scales.clone()
    ones[:, : -(-K // 32)] = 127
    X = torch.randint(-8, 9, (M, K), generator=g).to(torch.bfloat16)
    got = ssm.linear_w4(X.to(dev), W, ones.to(dev), out_dtype=torch.float32)
    assert np.array_equal(got.double().cpu().numpy(), X.double().numpy() @ expand(packed, ones, K).T)

    X = torch.randn(M, K, generator=g).to(torch.bfloat16)
    y0 = torch.randn(M, N, generator=g).to(torch.bfloat16)
    Y = torch.full((M, N + 3), 7.0, device=dev, dtype=torch.bfloat16)
    Y[:, :N] = y0.to(dev)
    ssm.linear_w4(X.to(dev), W, scales.to(dev), act=2, out=Y[:, :N])
    w = expand(packed, scales, K)
    want = X.double().numpy() @ w.T
    E = K * 2.0 ** -23 * (np.abs(X.double().numpy()) @ np.abs(w).T)
    want = want + y0.double().numpy()
    E = E + 2.0 ** -23 * np.abs(want)
    tol = E + 2.0 ** -8 * (np.abs(want) + E)
    bad = np.abs(Y[:, :N].double().cpu().numpy() - want) > tol
    assert not bad.any(), np.argwhere(bad)[:4].tolist()
    assert (Y[:, N:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(8250, 4200), (9000, 2100), (32780, 4096)])
def test_a_row_of_a_large_product_does_not_depend_on_the_batch(dev, N, K):
    packed, scales = (t.to(dev) for t in random_weights(N, K, 9))
    X = torch.randn(100, K).to(dev, torch.bfloat16)
    whole = ssm.linear_w4(X, packed, scales, out_dtype=torch.float32)
    for m in (1, 4, 5, 8, 9, 16, 17, 32, 40, 64):
        assert torch.equal(ssm.linear_w4(X[:m], packed, scales, out_dtype=torch.float32), whole[:m]), m


@pytest.mark.gpu
@pytest.mark.parametrize("byte", [252, 253, 254])
@pytest.mark.parametrize("M,N,K", [(1, 16, 33), (5, 40, 70), (20, 33, 1), (9, 50, 127), (3, 20, 555), (17, 64, 4107)])
def test_unused_codes_reach_nothing_at_any_scale(dev, M, N, K, byte):
    """Codes from K on are unused: random ones change no output, also where the last group's scale makes an infinity of
    them. Its own weights are zero, so what the row gives is the other groups' products, equal bit for bit."""
    packed, scales = random_weights(N, K, K + byte)
    groups = -(-K // 32)
    scales[:, :groups] = 127
    scales[:, groups - 1] = byte
    code = torch.stack((packed & 15, packed >> 4), -1).view(N, -1)
    code[:, 32 * (groups - 1): K] = 0
    code[:, K:] |= 4  # 2 and more: past bf16's range at scale bytes 253 and 254 for most
    packed = code[:, 0::2] | code[:, 1::2] << 4
    X = torch.randint(-8, 9, (M, K)).to(torch.bfloat16)
    want = X.double().numpy() @ expand(packed, scales, K).T
    got = ssm.linear_w4(X.to(dev), packed.to(dev), scales.to(dev), out_dtype=torch.float32)
    assert np.array_equal(got.double().cpu().numpy(), want)
