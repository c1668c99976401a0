"""hx_logits_adjust against its definition in float64, row by row. Tolerance: the repetition penalty, the two
subtractions and the bias are at most five roundings of 2^-24 of the magnitudes that they join (the division is IEEE's),
storage adds half a step (2^-24 fp32, 2^-8 bf16) of the value. Masked places are -inf exactly, untouched rows keep their
bits."""
import ctypes

import numpy as np
import pytest
import torch

from helixml_amd import _ffi, lm

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def oracle(logits, history=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
           bias=None, allowed=None):
    l = logits.double().numpy().copy()
    E = np.zeros_like(l)
    bt, V = l.shape
    for b in range(bt):
        n = 0 if history is None else history.shape[1]
        n = n if lengths is None else min(max(int(lengths[b]), 0), n)
        p = 0 if prompt_lengths is None else int(prompt_lengths[b])
        h = np.empty(0, np.int64) if history is None else history[b, :n].numpy().astype(np.int64)
        ok = (h >= 0) & (h < V)
        seen = np.zeros(V, bool)
        seen[h[ok]] = True
        late = ok & (np.arange(n) >= p)
        count = np.bincount(h[late], minlength=V).astype(np.float64)
        r = 1.0 if repetition is None else float(repetition[b])
        with np.errstate(invalid="ignore", divide="ignore"):
            l[b] = np.where(seen, np.where(l[b] > 0, l[b] / r, l[b] * r), l[b])
            fc = 0.0 if frequency is None else float(frequency[b]) * count
            pc = 0.0 if presence is None else float(presence[b]) * (count > 0)
            bb = 0.0 if bias is None else (bias if bias.dim() == 1 else bias[b]).double().numpy()
            E[b] = 5 * 2.0 ** -24 * (np.abs(l[b]) + np.abs(fc) + np.abs(pc) + np.abs(bb))
            l[b] = l[b] - fc - pc + bb
        if allowed is not None:
            w = (allowed if allowed.dim() == 1 else allowed[b]).numpy().astype(np.int64)
            v = np.arange(V)
            l[b] = np.where((w[v // 32] >> (v % 32)) & 1, l[b], -np.inf)
    return l, E


def compare(got, want, E, dtype):
    got = got.double().cpu().numpy()
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
    tol = E[fin] + HALF[dtype] * (np.abs(want[fin]) + E[fin])
    assert (np.abs(got[fin] - want[fin]) <= tol).all(), float((np.abs(got[fin] - want[fin]) / np.maximum(tol, 1e-300)).max())


def make(bt, V, H, seed, dtype, **flags):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    i = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, dtype=torch.int32)  # noqa: E731
    x = dict(logits=(3 * n(bt, V)).to(dtype))
    if H is not None:
        few = torch.where(i(0, 2, bt, H) > 0, i(0, max(1, V // 16), bt, H), i(-2, V + 2, bt, H))
        x.update(history=few, lengths=i(0, H + 1, bt), repetition=1 + n(bt).abs(), frequency=n(bt), presence=n(bt))
    if flags.get("prompt"):
        x["prompt_lengths"] = i(-1, H + 2, bt)
    if flags.get("bias"):
        x["bias"] = n(bt, V) if flags["bias"] == 2 else n(V)
    if flags.get("mask"):
        words = -(-V // 32)
        shape = (bt, words) if flags["mask"] == 2 else (words,)
        x["allowed"] = torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, dtype=torch.int64).to(torch.int32)
    return x


SIZES = [(1, 1, 1), (3, 256, 0), (2, 256, 700), (5, 31, 64), (2, 33, 1000), (1, 4096, 300), (3, 4097, 5000), (2, 10007, 129), (1, 70001, 2500),
         (300, 50, 3), (4, 32768, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("flags", [dict(), dict(prompt=True, bias=1, mask=2), dict(bias=2, mask=1), dict(prompt=True, mask=2)], ids=str)
@pytest.mark.parametrize("bt,V,H", SIZES)
def test_against_definition(dev, bt, V, H, flags, dtype):
    x = make(bt, V, H, seed=V + H, dtype=dtype, **flags)
    d = {k: v.to(dev) for k, v in x.items()}
    keep = d["logits"].clone()
    got = lm.adjust_logits(**d)
    assert torch.equal(d["logits"], keep)
    compare(got, *oracle(**x), dtype)
    # in place, the same bits
    assert lm.adjust_logits(**d, out=d["logits"]) is d["logits"]
    assert torch.equal(d["logits"].view(torch.uint8), got.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strided_rows(dev, dtype):
    """Every operand a view into wider rows, none of them 16-byte aligned; what lies beside the output stays."""
    bt, V, H = 3, 300, 50
    x = make(bt, V, H, seed=1, dtype=dtype, prompt=True, bias=2, mask=2)

    def wide(t, left, right):
        w = torch.full((t.shape[0], t.shape[1] + left + right), 5, device=dev, dtype=t.dtype)
        w[:, left: left + t.shape[1]] = t.to(dev)
        return w[:, left: left + t.shape[1]], w

    d = {k: wide(v, 1, 2)[0] if v.dim() == 2 else v.to(dev) for k, v in x.items()}
    out, whole = wide(torch.zeros(bt, V, dtype=dtype), 3, 4)
    lm.adjust_logits(**d, out=out)
    compare(out, *oracle(**x), dtype)
    assert (whole[:, :3] == 5).all() and (whole[:, 3 + V:] == 5).all()


@pytest.mark.gpu
def test_nothing_asked_for_keeps_the_bits(dev):
    x = torch.randn(4, 5000, device=dev)
    x[0, 7], x[1, 8], x[2, 9] = float("nan"), float("inf"), float("-inf")
    assert torch.equal(lm.adjust_logits(x).view(torch.int32), x.view(torch.int32))
    # penalties of one and nought change nothing either
    h = torch.randint(0, 5000, (4, 100), device=dev, dtype=torch.int32)
    one, nought = torch.ones(4, device=dev), torch.zeros(4, device=dev)
    got = lm.adjust_logits(x, h, repetition=one, frequency=nought, presence=nought)
    assert torch.equal(torch.nan_to_num(got, nan=1.5), torch.nan_to_num(x, nan=1.5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_without_allowed_tokens_and_values_without_a_number(dev, dtype):
    """A row that allows nothing is -inf throughout; masked NaN and infinities become -inf, unmasked ones follow the
    formula (a type's lowest value among them)."""
    V = 1000
    x = make(4, V, 60, seed=2, dtype=dtype, mask=2)
    x["allowed"][1] = 0
    x["allowed"][2] = -1
    x["lengths"][:] = 60
    low = torch.finfo(dtype).min
    for n, v in enumerate((float("nan"), float("inf"), float("-inf"), low)):
        x["logits"][:, n::7] = v
    got = lm.adjust_logits(**{k: v.to(dev) for k, v in x.items()})
    assert (got[1] == float("-inf")).all()
    want, E = oracle(**x)
    # past the type's range a value is an infinity of its sign; fp32 sums reach that range before float64's
    top = torch.finfo(dtype).max
    g = got.double().cpu().numpy()
    plain = np.isfinite(want) & (np.abs(want) < 0.9 * float(top))
    compare(torch.from_numpy(g[plain]).to(dtype), want[plain], E[plain], dtype)
    rest = ~plain & ~np.isnan(want)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert (np.sign(g[rest]) == np.sign(want[rest])).all() and (np.abs(g[rest]) >= 0.5 * float(top)).all()


@pytest.mark.gpu
def test_long_history_counts_every_entry(dev):
    """One token a hundred thousand times, another once at the very end, the rest of the row untouched."""
    V, H = 257, 100001
    h = torch.full((1, H), 3, dtype=torch.int32, device=dev)
    h[0, -1] = 256
    x = torch.zeros(1, V, device=dev)
    got = lm.adjust_logits(x, h, frequency=torch.tensor([0.5], device=dev), presence=torch.tensor([2.0], device=dev)).cpu()
    assert got[0, 3] == -50002.0 and got[0, 256] == -2.5
    got[0, 3] = got[0, 256] = 0
    assert (got == 0).all()


@pytest.mark.gpu
def test_captured_and_replayed(dev):
    x = {k: v.to(dev) for k, v in make(3, 9000, 400, seed=1, dtype=torch.float32, prompt=True, bias=1, mask=2).items()}
    lm.adjust_logits(**x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = lm.adjust_logits(**x)
    for seed in (2, 3, 4):
        for k, v in make(3, 9000, 400, seed=seed, dtype=torch.float32, prompt=True, bias=1, mask=2).items():
            x[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        held = out.clone()
        assert torch.equal(held, lm.adjust_logits(**x))


def test_refusals():
    L, p = _ffi.lib(), ctypes.c_void_p(4096)

    def call(batch=2, vocab=64, dtype=0, logits=p, ldl=64, history=p, ldh=8, hist=8, bias=None, ldb=0, allowed=None, lda=0,
             out=ctypes.c_void_p(8192), ldo=64):
        return L.hx_logits_adjust(batch, vocab, dtype, logits, ldl, history, ldh, hist, None, None, None, None, None, bias, ldb,
                                  allowed, lda, out, ldo, None)

    assert call(batch=-1) == _ffi.InvalidDimension.status
    assert call(hist=-1) == _ffi.InvalidDimension.status
    assert call(dtype=2) == _ffi.DTypeMismatch.status
    assert call(batch=65536) == _ffi.UnsupportedOperation.status
    assert call(vocab=2 ** 31, ldl=2 ** 31, ldo=2 ** 31) == _ffi.UnsupportedOperation.status
    assert call(logits=None) == _ffi.InvalidInput.status
    assert call(out=None) == _ffi.InvalidInput.status
    assert call(ldl=63) == _ffi.InvalidInput.status
    assert call(ldo=63) == _ffi.InvalidInput.status
    assert call(out=p, ldl=65) == _ffi.InvalidInput.status
    assert call(history=None) == _ffi.InvalidInput.status
    assert call(ldh=7) == _ffi.InvalidInput.status
    assert call(bias=p, ldb=63) == _ffi.InvalidInput.status
    assert call(allowed=p, lda=1) == _ffi.InvalidInput.status
    assert call(batch=0) == 0 and call(vocab=0) == 0


@pytest.mark.gpu
def test_wrapper_refusals(dev):
    x = torch.zeros(2, 64, device=dev)
    h = torch.zeros(2, 8, device=dev, dtype=torch.int32)
    with pytest.raises(_ffi.ShapeMismatch):
        lm.adjust_logits(x[0])
    with pytest.raises(_ffi.DTypeMismatch):
        lm.adjust_logits(x.half())
    with pytest.raises(_ffi.DTypeMismatch):
        lm.adjust_logits(x, h.long())
    with pytest.raises(_ffi.ShapeMismatch):
        lm.adjust_logits(x, h[:1])
    with pytest.raises(_ffi.ShapeMismatch):
        lm.adjust_logits(x, h, repetition=torch.ones(3, device=dev))
    with pytest.raises(_ffi.ShapeMismatch):
        lm.adjust_logits(x, allowed=torch.zeros(2, 3, device=dev, dtype=torch.int32))
    with pytest.raises(_ffi.InvalidInput):
        lm.adjust_logits(x, bias=torch.zeros(64))
    with pytest.raises(_ffi.InvalidInput):
        lm.adjust_logits(torch.zeros(64, 2, device=dev).t())
    with pytest.raises(_ffi.DTypeMismatch):
        lm.adjust_logits(x, out=x.bfloat16())
