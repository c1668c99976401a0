"""Linear attention with one decay a head (hx_decay_attention_fwd / _bwd / _step) against its definition in float64, with
componentwise error bounds.

Bounds. Every output is a sum of products of magnitudes that the same recurrence over absolute values gives, A. The kernels
form it in 32 bits: a product over dk or dv channels and one over a chunk's tokens (at most 64) add at most that many roundings of
2^-24 of A, whatever their order; a chunk passes its state on with at most four more, so do segments. A power w^x over x <= 64
tokens errs by 2^-23 from the exponential and |x log2 w| 2^-23 from its argument. In bf16 the scores and the state are
split into two parts where an output is formed, each off by at most 2^-17 of its value, and weighted operands into three, which is
2^-24. Shared heads' sums add a rounding a head. Storage adds half a step of the value.
"""
import numpy as np
import pytest
import torch

from helixml_amd import _ffi, ssm

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def inputs(bt, L, heads, dk, dv, seed, dtype, hq=None, hk=None, hv=None, chunk=True, lengths=None, decay=None, scale=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if decay is None:
        decay = -torch.exp(torch.rand(heads, generator=g) * 7.0 - 7.5)
    return dict(q=n(bt, L, hq or heads, dk).to(dtype), k=n(bt, L, hk or heads, dk).to(dtype), v=n(bt, L, hv or heads, dv).to(dtype),
                log_decay=torch.as_tensor(decay, dtype=F32), scale=dk ** -0.5 if scale is None else scale,
                lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32),
                init=n(bt, heads, dk, dv) if chunk else None, dout=n(bt, L, heads, dv).to(dtype), dlast=n(bt, heads, dk, dv) if chunk else None)


def f64(t):
    return None if t is None else t.double().numpy()


def oracle(x):
    """The definition, token by token: outputs, gradients, and the magnitudes A that each is a sum of."""
    heads = x["log_decay"].shape[0]
    wide = lambda t: np.repeat(f64(t), heads // t.shape[2], 2)  # noqa: E731
    q, k, v, do = wide(x["q"]), wide(x["k"]), wide(x["v"]), f64(x["dout"])
    bt, L, _, dk = q.shape
    dv = v.shape[-1]
    w = np.exp(f64(x["log_decay"]))[:, None, None]
    s = x["scale"]
    o = {n: np.zeros((bt, L, heads, d)) for n, d in (("out", dv), ("dq", dk), ("dk", dk), ("dv", dv))}
    A = {n: np.zeros_like(t) for n, t in o.items()}
    o["last"], o["dinit"], A["last"], A["dinit"] = (np.zeros((bt, heads, dk, dv)) for _ in range(4))
    outer = lambda a, b: a[:, :, None] * b[:, None, :]  # noqa: E731
    for b in range(bt):
        n = L if x["lengths"] is None else min(max(int(x["lengths"][b]), 0), L)
        S = np.zeros((heads, dk, dv)) if x["init"] is None else f64(x["init"])[b].copy()
        M = np.abs(S)
        for t in range(n):
            S = w * S + outer(k[b, t], v[b, t])
            M = w * M + outer(np.abs(k[b, t]), np.abs(v[b, t]))
            o["out"][b, t], A["out"][b, t] = s * np.einsum("hk,hkv->hv", q[b, t], S), s * np.einsum("hk,hkv->hv", np.abs(q[b, t]), M)
            o["dq"][b, t], A["dq"][b, t] = s * np.einsum("hkv,hv->hk", S, do[b, t]), s * np.einsum("hkv,hv->hk", M, np.abs(do[b, t]))
        o["last"][b], A["last"][b] = S, M
        G = np.zeros((heads, dk, dv)) if x["dlast"] is None else f64(x["dlast"])[b].copy()
        M = np.abs(G)
        for t in reversed(range(n)):
            G = G + s * outer(q[b, t], do[b, t])
            M = M + s * outer(np.abs(q[b, t]), np.abs(do[b, t]))
            o["dk"][b, t], A["dk"][b, t] = np.einsum("hkv,hv->hk", G, v[b, t]), np.einsum("hkv,hv->hk", M, np.abs(v[b, t]))
            o["dv"][b, t], A["dv"][b, t] = np.einsum("hkv,hk->hv", G, k[b, t]), np.einsum("hkv,hk->hv", M, np.abs(k[b, t]))
            G, M = w * G, w * M
        o["dinit"][b], A["dinit"][b] = G, M
    for n, of in (("dq", "q"), ("dk", "k"), ("dv", "v")):
        each = x[of].shape[2]
        o[n], A[n] = (t.reshape(bt, L, each, heads // each, -1).sum(3) for t in (o[n], A[n]))
    return o, A


def unit(x):
    """The relative error of a sum of magnitudes A (head by head, the largest): see above."""
    bt, L, _, dk = x["q"].shape
    heads, dv = x["log_decay"].shape[0], x["v"].shape[-1]
    steps = min(L, 64)
    l2 = np.abs(f64(x["log_decay"])) / np.log(2.0)
    l2 = np.where(np.isfinite(l2), l2, 0.0).max() if heads else 0.0
    n = max(dk, dv) + 64 + 4 * (L // 32 + 2) + heads + 8
    two = 2.0 * 2.0 ** -17 if x["q"].dtype == BF16 else 0.0
    return n * 2.0 ** -24 + (2.0 + min(l2 * steps, 150.0)) * 2.0 ** -23 + two


def check(name, got, want, A, u, half):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got = got.double().cpu().numpy()
    tol = u * A + half * (np.abs(want) + u * A) + 1e-30
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (name, int(bad.sum()), float(np.nanmax(np.abs(got - want) / tol)), np.argwhere(bad)[:4].tolist())


def on(dev, x):
    return {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in x.items()}


def run(dev, x, **kw):
    d = on(dev, x)
    out, last = ssm.decay_attention_fwd(d["q"], d["k"], d["v"], d["log_decay"], scale=d["scale"], lengths=d["lengths"], init_state=d["init"],
                                        return_last_state=True, **kw)
    dq, dk, dv, dinit = ssm.decay_attention_bwd(d["q"], d["k"], d["v"], d["log_decay"], d["dout"], scale=d["scale"], lengths=d["lengths"],
                                                init_state=d["init"], dlast=d["dlast"], **kw)
    torch.cuda.synchronize()
    return dict(out=out, last=last, dq=dq, dk=dk, dv=dv, dinit=dinit)


def check_all(dev, x):
    got, (want, A) = run(dev, x), oracle(x)
    u, half = unit(x), HALF[x["q"].dtype]
    for n in ("out", "last", "dq", "dk", "dv", "dinit"):
        check(n, got[n], want[n], A[n], u, HALF[F32] if n in ("last", "dinit") else half)
    return got


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 3, 3, 5), (1, 31, 2, 16, 16), (1, 32, 1, 64, 64), (2, 33, 2, 17, 40), (1, 63, 1, 40, 72), (1, 64, 3, 64, 64),
          (3, 65, 2, 65, 63), (1, 127, 2, 128, 64), (1, 128, 1, 129, 130), (1, 129, 2, 64, 128), (2, 100, 1, 200, 256), (1, 70, 1, 256, 256), (1, 257, 1, 33, 9)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_against_float64(dev, shape, dtype):
    check_all(dev, inputs(*shape, seed=sum(shape), dtype=dtype, chunk=shape[1] % 2 == 1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bt,L,heads,dk,dv", [(1, 1100, 2, 24, 40), (2, 777, 1, 64, 64), (1, 512, 1, 128, 16), (1, 2049, 1, 8, 8)])
def test_segments(dev, bt, L, heads, dk, dv, dtype):
    assert ssm.decay_attention_workspace_size(bt, L, heads, dk, dv, dtype) > 0
    check_all(dev, inputs(bt, L, heads, dk, dv, seed=L, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("hq,hk,hv", [(6, 2, 2), (1, 1, 6), (6, 3, 6), (2, 6, 3), (3, 2, 1)])
def test_shared_heads(dev, hq, hk, hv, dtype):
    check_all(dev, inputs(2, 130, 6, 20, 24, seed=hq + 10 * hk, dtype=dtype, hq=hq, hk=hk, hv=hv))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("L", [70, 1030])
def test_lengths(dev, L, dtype):
    """Sequences of no, one, some and all tokens; lengths outside [0, L] are clamped. What lies behind them is not read."""
    lengths = [0, 1, 33, L - 1, L, 64, -5, L + 100]
    x = inputs(len(lengths), L, 2, 24, 20, seed=L, dtype=dtype, lengths=lengths)
    for n in ("q", "k", "v", "dout"):
        for b, m in enumerate(lengths):
            x[n][b, min(max(m, 0), L):] = float("nan")
    clean = {k: torch.nan_to_num(v) if isinstance(v, torch.Tensor) and v.dim() == 4 else v for k, v in x.items()}
    got, (want, A) = run(dev, x), oracle(clean)
    for n in got:
        check(n, got[n], want[n], A[n], unit(x), HALF[F32] if n in ("last", "dinit") else HALF[dtype])
    for b, m in enumerate(lengths):
        for n in ("out", "dq", "dk", "dv"):
            assert not got[n][b, min(max(m, 0), L):].any()
    for b in (0, 6):
        assert torch.equal(got["last"][b].cpu(), x["init"][b]) and torch.equal(got["dinit"][b].cpu(), x["dlast"][b])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decays(dev, dtype):
    """Nothing kept, hardly anything, nearly all, all, and a state that grows."""
    decay = [-float("inf"), -100.0, -20.0, -2.0, -1e-6, 0.0, 0.01]
    check_all(dev, inputs(2, 300, len(decay), 16, 16, seed=9, dtype=dtype, decay=decay))


def test_slow_decay_over_many_tokens(dev):
    """A state that lives for tens of thousands of tokens, each of them 1, so that S has a closed form. What may be lost: the state
    is rounded once a chunk of 32 tokens, 2^-24 of a state that never passes the last one, plus a chunk's own sums and powers (64 roundings
    of its magnitude, which is in turn a part of the state)."""
    L, g = 60000, -1e-5
    one = torch.ones(1, L, 1, 1, device=dev)
    out, last = ssm.decay_attention_fwd(one, one, one, torch.tensor([g], device=dev), return_last_state=True)
    g32 = float(torch.tensor(g))
    want = np.expm1(g32 * np.arange(1, L + 1)) / np.expm1(g32)
    got = out.double().cpu().numpy().ravel()
    bound = (L / 32 + 64) * 2.0 ** -24 * want[-1]
    assert np.abs(got - want).max() <= bound and abs(float(last) - want[-1]) <= bound


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strided_tokens(dev, dtype):
    """q, k and v as slices of one projection's output, from an odd element on: the same bits as from copies."""
    x = inputs(2, 150, 3, 20, 12, seed=4, dtype=dtype)
    wide = torch.full((2, 150, 3 * 52 + 7), float("nan"), dtype=dtype)
    at = 1
    parts = {}
    for n in ("q", "k", "v"):
        w = x[n].shape[2] * x[n].shape[3]
        wide[:, :, at: at + w] = x[n].flatten(2)
        parts[n] = (at, w)
        at += w + 2
    d = wide.to(dev)
    views = {n: d[:, :, a: a + w].unflatten(2, x[n].shape[2:]) for n, (a, w) in parts.items()}
    want, y = run(dev, x), on(dev, x)
    out, last = ssm.decay_attention_fwd(views["q"], views["k"], views["v"], y["log_decay"], scale=x["scale"], init_state=y["init"], return_last_state=True)
    grads = ssm.decay_attention_bwd(views["q"], views["k"], views["v"], y["log_decay"], y["dout"], scale=x["scale"], init_state=y["init"], dlast=y["dlast"])
    for n, t in zip(("out", "last", "dq", "dk", "dv", "dinit"), (out, last, *grads)):
        assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite_stays_behind(dev, what, value, dtype):
    """A token that is not finite reaches no token before it (forward) or after it (its own gradients aside)."""
    x = inputs(1, 150, 2, 16, 16, seed=6, dtype=dtype)
    want = run(dev, x)
    at = 85
    x[what][0, at, 0, 3] = value
    got = run(dev, x)
    assert torch.equal(got["out"][:, :at], want["out"][:, :at]) and torch.equal(got["out"][:, :, 1], want["out"][:, :, 1])
    assert not torch.isfinite(got["out"][0, at, 0].float()).all()
    # dk and dv of later tokens are formed from q and dout of tokens from them on
    if what == "q":
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:, at + 1:], want[n][:, at + 1:]), n
            assert not torch.isfinite(got[n][0, : at + 1, 0].float()).all(), n
    else:
        assert torch.equal(got["dq"][:, :at], want["dq"][:, :at])


WIDTHS = [(1, 600, 1, 168, 58), (1, 700, 1, 5, 140), (2, 300, 2, 3, 7), (1, 1000, 2, 190, 190), (1, 330, 2, 193, 70), (1, 520, 1, 6, 2), (2, 200, 1, 256, 193),
          (1, 1100, 1, 128, 65), (1, 90, 2, 256, 4)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", WIDTHS, ids=lambda s: "x".join(map(str, s)))
def test_widths_in_segments(dev, shape, dtype):
    """Rows that end anywhere, narrower than one load among them, in tiles of every width, with lengths, cut and not."""
    bt, L = shape[:2]
    check_all(dev, inputs(*shape, seed=sum(shape), dtype=dtype, lengths=[L - 1, L // 2][:bt]))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_carried_in_place(dev, dtype):
    """One buffer for the state before and after; one for its gradient."""
    x = inputs(2, 700, 1, 24, 24, seed=8, dtype=dtype)
    want, d = run(dev, x), on(dev, x)
    code = ssm._STORAGE[dtype]
    out = torch.empty_like(d["dout"])
    sizes = (2, 700, 1, 1, 1, 1, 24, 24, code)
    ws = torch.empty(ssm.decay_attention_workspace_size(2, 700, 1, 24, 24, dtype, backward=True), device=dev, dtype=torch.uint8)
    ld = 24
    qkv = (d["q"].data_ptr(), ld, d["k"].data_ptr(), ld, d["v"].data_ptr(), ld, d["log_decay"].data_ptr(), float(x["scale"]), None)
    state, grad = d["init"].clone(), d["dlast"].clone()
    _ffi.call("hx_decay_attention_fwd", *sizes, *qkv, state.data_ptr(), out.data_ptr(), state.data_ptr(), ws.data_ptr(), ws.numel(), None)
    assert torch.equal(out, want["out"]) and torch.equal(state, want["last"])
    g = [torch.empty_like(d[n]) for n in ("q", "k", "v")]
    _ffi.call("hx_decay_attention_bwd", *sizes, *qkv, d["init"].data_ptr(), d["dout"].data_ptr(), grad.data_ptr(), *(t.data_ptr() for t in g),
              grad.data_ptr(), ws.data_ptr(), ws.numel(), None)
    for t, n in zip((*g, grad), ("dq", "dk", "dv", "dinit")):
        assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("L", [40, 700], ids=["one segment", "segments"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_gradient_in_the_states_place(dev, dtype, L):
    """dinit may take init_state's buffer, which dq's pass reads."""
    x = inputs(3, L, 2, 160, 160, seed=9, dtype=dtype)
    want, d = run(dev, x), on(dev, x)
    code, ld = ssm._STORAGE[dtype], 2 * 160
    nbytes = ssm.decay_attention_workspace_size(3, L, 2, 160, 160, dtype, backward=True)
    ws = torch.empty(max(nbytes, 1), device=dev, dtype=torch.uint8)
    state, g = d["init"].clone(), [torch.empty_like(d[n]) for n in ("q", "k", "v")]
    _ffi.call("hx_decay_attention_bwd", 3, L, 2, 2, 2, 2, 160, 160, code, d["q"].data_ptr(), ld, d["k"].data_ptr(), ld, d["v"].data_ptr(), ld,
              d["log_decay"].data_ptr(), float(x["scale"]), None, state.data_ptr(), d["dout"].data_ptr(), d["dlast"].data_ptr(),
              *(t.data_ptr() for t in g), state.data_ptr(), ws.data_ptr(), nbytes, None)
    for t, n in zip((*g, state), ("dq", "dk", "dv", "dinit")):
        assert torch.equal(t, want[n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_pieces_and_tokens_agree(dev, dtype):
    """A sequence in pieces of any length, each from the last one's state, and token by token: the whole sequence's result."""
    x = inputs(2, 200, 2, 24, 40, seed=3, dtype=dtype)
    want, A = oracle(x)
    d = on(dev, x)
    state, outs = d["init"], []
    for a, b in ((0, 1), (1, 65), (65, 65), (65, 197), (197, 200)):
        out, state = ssm.decay_attention_fwd(d["q"][:, a:b].contiguous(), d["k"][:, a:b].contiguous(), d["v"][:, a:b].contiguous(), d["log_decay"],
                                             scale=x["scale"], init_state=state, return_last_state=True)
        outs.append(out)
    u = unit(x)
    check("out", torch.cat(outs, 1), want["out"], A["out"], u, HALF[dtype])
    check("last", state, want["last"], A["last"], u, HALF[F32])
    state = d["init"].clone()
    for t in range(200):  # rows of a batch are strided here
        out = ssm.decay_attention_step(state, d["q"][:, t], d["k"][:, t], d["v"][:, t], d["log_decay"], scale=x["scale"])
        check(f"token {t}", out, want["out"][:, t], A["out"][:, t], u + 200 * 2.0 ** -23, HALF[dtype])
    check("state", state, want["last"], A["last"], u + 200 * 2.0 ** -23, HALF[F32])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bt,heads,hq,hk,hv,dk,dv", [(1, 1, 1, 1, 1, 1, 1), (3, 4, 4, 2, 2, 17, 5), (2, 6, 1, 1, 6, 128, 64), (2, 2, 2, 2, 2, 63, 255), (1, 2, 2, 2, 2, 256, 256),
                                                     (5, 1, 1, 1, 1, 64, 66)])
def test_step(dev, bt, heads, hq, hk, hv, dk, dv, dtype):
    x = inputs(bt, 1, heads, dk, dv, seed=dk, dtype=dtype, hq=hq, hk=hk, hv=hv)
    want, A = oracle(x)
    d = on(dev, x)
    state = d["init"].clone()
    out = ssm.decay_attention_step(state, d["q"][:, 0], d["k"][:, 0], d["v"][:, 0], d["log_decay"], scale=x["scale"])
    u = (dk + 8) * 2.0 ** -24
    check("out", out, want["out"][:, 0], A["out"][:, 0], u, HALF[dtype])
    check("state", state, want["last"], A["last"], 4 * 2.0 ** -24, HALF[F32])


@pytest.mark.parametrize("what", ["q", "k", "v", "init"])
def test_gradients_are_differences(dev, what):
    """The loss sum(dout out) + sum(dlast last) is linear in each operand alone, so its difference between two of them is the
    gradient's product with theirs; the loss is formed in float64."""
    x = inputs(2, 90, 2, 8, 12, seed=11, dtype=F32, hk=1, lengths=[90, 57])
    got = run(dev, x)
    name = {"q": "dq", "k": "dk", "v": "dv", "init": "dinit"}[what]
    g = torch.Generator().manual_seed(1)
    by = torch.randn(x[what].shape, generator=g)
    y = dict(x)
    y[what] = x[what] + by
    by = (y[what].double() - x[what].double()).numpy()
    loss = lambda z: sum((o * f64(x[w])).sum() for o, w in ((oracle(z)[0]["out"], "dout"), (oracle(z)[0]["last"], "dlast")))  # noqa: E731
    A = oracle(x)[1][name]
    want, bound = loss(y) - loss(x), (A * np.abs(by)).sum() * (unit(x) + HALF[F32])
    assert abs((got[name].double().cpu().numpy() * by).sum() - want) <= bound


def test_same_bits(dev):
    for dtype in (F32, BF16):
        x = inputs(1, 2500, 2, 64, 64, seed=2, dtype=dtype)
        a, b = run(dev, x), run(dev, x)
        for n in a:
            assert torch.equal(a[n], b[n]), n


def test_empty(dev):
    z = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
    for bt, L, heads in ((0, 5, 2), (2, 5, 0), (2, 0, 2)):
        h = max(heads, 0)
        init = torch.randn(bt, h, 4, 4, device=dev)
        out, last = ssm.decay_attention_fwd(z(bt, L, h, 4), z(bt, L, h, 4), z(bt, L, h, 4), torch.zeros(h, device=dev), init_state=init, return_last_state=True)
        assert out.shape == (bt, L, h, 4) and torch.equal(last, init)
        *_, dinit = ssm.decay_attention_bwd(z(bt, L, h, 4), z(bt, L, h, 4), z(bt, L, h, 4), torch.zeros(h, device=dev), z(bt, L, h, 4), dlast=init)
        assert torch.equal(dinit, init)
