"""The gated linear recurrence (hx_gated_scan_fwd / _bwd, hx_gated_state_update) against its definition in
float64, with componentwise error bounds that are carried along the recurrence.

Bounds. The kernels form a = sigmoid(f) and i = sigmoid(-f) from e = exp2(-|f| log2 e): the argument's rounding
(2^-24 of |f| log2 e, and as much for the constant) is a relative error of at most |f| 2^-23 in e, the exponential
and the reciprocal add an ulp (2^-23) each. With d = (|f| + 2) 2^-23 that is |da|, |di| <= a i d + 2^-22 of the value.
Every product and sum of the recurrence adds at most 2^-24 of the magnitudes that it joins, whichever way the steps are
grouped (a group's decay is a product of a's, whose relative errors add); four such roundings are counted a step, 2^-22.
    E_t = a E_{t-1} + (da + 2^-22 a) H_{t-1} + (di + 2^-22 i) |x|,   H_t = a H_{t-1} + i |x|
bounds the state's error, and the same recurrence run backwards the adjoint's. Storage adds half a step, 2^-8 (bf16) or
2^-24 (fp32) of the value.
"""
import numpy as np
import pytest
import torch

from helixml_amd import _ffi, ssm

pytestmark = pytest.mark.gpu

U = 2.0 ** -22
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
CHUNK = ssm.GATED_CHUNK


def sig(v):
    with np.errstate(over="ignore"):
        return 1.0 / (1.0 + np.exp(-v))


def inputs(bt, L, dim, seed, dtype, gate=True, chunk=True):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    f = n(bt, L, dim) + 1.5 * n(dim) + 2.5
    return dict(x=n(bt, L, dim).to(dtype), f=f.to(dtype), z=n(bt, L, dim).to(dtype) if gate else None,
                init=n(bt, dim) if chunk else None, dout=n(bt, L, dim).to(dtype), dlast=n(bt, dim) if chunk else None)


def f64(t):
    return None if t is None else t.double().numpy()


def oracle_fwd(x, f, z=None, init=None, **_):
    """(out, last, before [bt, L, dim], bounds of out and last)."""
    bt, L, dim = x.shape
    a, i = sig(f), sig(-f)
    da = a * i * (np.abs(f) + 2) * 2.0 ** -23
    h = np.zeros((bt, dim)) if init is None else init.copy()
    H, E = np.abs(h), np.zeros((bt, dim))
    before, bE, hs, hE, hH = (np.empty_like(x) for _ in range(5))
    for t in range(L):
        before[:, t], bE[:, t] = h, E
        E = a[:, t] * E + (da[:, t] + U * a[:, t]) * H + (da[:, t] + U * i[:, t]) * np.abs(x[:, t])
        h = a[:, t] * h + i[:, t] * x[:, t]
        H = a[:, t] * H + i[:, t] * np.abs(x[:, t])
        hs[:, t], hE[:, t], hH[:, t] = h, E, H
    out, oE = hs, hE + U * hH
    if z is not None:
        s = sig(z)
        v = z * s
        out = hs * v
        oE = hE * np.abs(v) + hH * np.abs(v) * ((np.abs(z) + 2) * 2.0 ** -23 + 2 * U)
    return dict(out=out, last=h, before=before, hs=hs, out_E=oE, last_E=E + U * H, bE=bE, hE=hE, hH=hH)


def oracle_bwd(x, f, dout, z=None, init=None, dlast=None):
    o = oracle_fwd(x, f, z, init)
    bt, L, dim = x.shape
    a, i = sig(f), sig(-f)
    dg = (np.abs(f) + 2) * 2.0 ** -23
    da = a * i * dg
    carry = np.zeros((bt, dim)) if dlast is None else dlast.copy()
    C, E = np.abs(carry), np.zeros((bt, dim))
    dh, dhE = dout, np.zeros_like(dout)
    r = {}
    if z is not None:
        s, t = sig(z), sig(-z)
        v, d = z * s, s * (1 + z * t)
        zr = (np.abs(z) + 2) * 2.0 ** -23 + 2 * U
        dh = dout * v
        dhE = np.abs(dh) * zr
        r["dz"] = dout * o["hs"] * d
        r["dz_E"] = np.abs(dout) * ((o["hE"] + U * o["hH"]) * np.abs(d) + o["hH"] * s * (1 + np.abs(z) * t) * 2 * zr)
    dx, dxE, df, dfE = (np.empty_like(x) for _ in range(4))
    for t in reversed(range(L)):
        g, G, gE = dh[:, t] + carry, np.abs(dh[:, t]) + C, dhE[:, t] + E
        gE = gE + U * G
        dx[:, t] = g * i[:, t]
        dxE[:, t] = gE * i[:, t] + G * (da[:, t] + U * i[:, t])
        m = np.abs(o["before"][:, t]) + np.abs(x[:, t])
        df[:, t] = g * i[:, t] * a[:, t] * (o["before"][:, t] - x[:, t])
        ai = a[:, t] * i[:, t]
        dfE[:, t] = gE * ai * m + G * ai * (m * (2 * dg[:, t] + 4 * U) + o["bE"][:, t])
        carry, E = g * a[:, t], gE * a[:, t] + G * (da[:, t] + U * a[:, t])
        C = G * a[:, t]
    r.update(dx=dx, dx_E=dxE, df=df, df_E=dfE, dinit=carry, dinit_E=E + U * C)
    return r


def check(name, got, want, bound, half):
    got = got.double().cpu().numpy()
    tol = bound + half * (np.abs(want) + bound) + 1e-37
    bad = np.abs(got - want) > tol
    assert not bad.any(), (name, int(bad.sum()), float((np.abs(got - want) / tol).max()), np.argwhere(bad)[:4].tolist())
    assert np.isfinite(got).all()


def to(dev, x):
    return {k: None if v is None else v.to(dev) for k, v in x.items()}


def run(dev, x, **kw):
    d = to(dev, x)
    out, last, states = ssm.gated_scan_fwd(d["x"], d["f"], d["z"], d["init"], return_last_state=True, return_states=True, **kw)
    dx, df, dz, dinit = ssm.gated_scan_bwd(d["x"], d["f"], d["dout"], states, z=d["z"], dlast=d["dlast"], **kw)
    torch.cuda.synchronize()
    return dict(out=out, last=last, states=states, dx=dx, df=df, dz=dz, dinit=dinit)


SHAPES = [(1, 1, 1), (2, 2, 3), (1, 127, 64), (2, 128, 63), (1, 129, 65), (3, 255, 2), (1, 256, 130), (2, 257, 66),
          (1, 1000, 7), (1, 2500, 36), (5, 1021, 40), (2, 700, 200), (1, 513, 256), (1, 4111, 128), (16, 3, 31)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate,chunk", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("bt,L,dim", SHAPES)
def test_forward_and_gradients(dev, bt, L, dim, gate, chunk, dtype):
    x = inputs(bt, L, dim, seed=L + dim, dtype=dtype, gate=gate, chunk=chunk)
    got = run(dev, x)
    ref = {k: f64(v) for k, v in x.items()}
    o = oracle_fwd(**ref)
    check("out", got["out"], o["out"], o["out_E"], HALF[dtype])
    check("last", got["last"], o["last"], o["last_E"], 2.0 ** -24)
    check("states", got["states"], o["before"][:, ::CHUNK], o["bE"][:, ::CHUNK] + U * np.abs(o["before"][:, ::CHUNK]), 2.0 ** -24)
    b = oracle_bwd(**ref)
    for k in ("dx", "df", "dz"):
        if k in b:
            check(k, got[k], b[k], b[k + "_E"], HALF[dtype])
    check("dinit", got["dinit"], b["dinit"], b["dinit_E"], 2.0 ** -24)


@pytest.mark.parametrize("bt,L,dim,dtype", [(1, 70001, 2, torch.float32), (2, 40000, 5, torch.bfloat16), (12, 2300, 700, torch.bfloat16),
                                            (1, 16384, 3, torch.float32), (1, 16385, 3, torch.float32)])
def test_long_chains(dev, bt, L, dim, dtype):
    """Sequences of many groups of tiles, and more tiles than fit the GPU at once."""
    x = inputs(bt, L, dim, seed=L, dtype=dtype)
    got = run(dev, x)
    ref = {k: f64(v) for k, v in x.items()}
    o = oracle_fwd(**ref)
    check("out", got["out"], o["out"], o["out_E"], HALF[dtype])
    check("last", got["last"], o["last"], o["last_E"], 2.0 ** -24)
    check("states", got["states"], o["before"][:, ::CHUNK], o["bE"][:, ::CHUNK] + U * np.abs(o["before"][:, ::CHUNK]), 2.0 ** -24)
    b = oracle_bwd(**ref)
    for k in ("dx", "df", "dz"):
        check(k, got[k], b[k], b[k + "_E"], HALF[dtype])
    check("dinit", got["dinit"], b["dinit"], b["dinit_E"], 2.0 ** -24)


@pytest.mark.parametrize("bt,L,dim,dtype", [(3, 260, 192, torch.float32), (67, 300, 513, torch.bfloat16), (601, 131, 65, torch.float32)])
def test_many_columns(dev, bt, L, dim, dtype):
    """9, 603 and 1202 columns of 64 channels: several ticket counters, in the larger two the last with fewer columns."""
    x = inputs(bt, L, dim, seed=bt, dtype=dtype)
    got = run(dev, x)
    ref = {k: f64(v) for k, v in x.items()}
    o = oracle_fwd(**ref)
    check("out", got["out"], o["out"], o["out_E"], HALF[dtype])
    check("last", got["last"], o["last"], o["last_E"], 2.0 ** -24)
    b = oracle_bwd(**ref)
    for k in ("dx", "df", "dz"):
        check(k, got[k], b[k], b[k + "_E"], HALF[dtype])
    check("dinit", got["dinit"], b["dinit"], b["dinit_E"], 2.0 ** -24)


@pytest.mark.parametrize("fill", [0, 255, None], ids=["zeros", "ones", "numbers"])
def test_a_workspace_may_hold_anything(dev, fill):
    """What an earlier call left, zeros, or numbers: a workspace is cleared by the call that uses it."""
    x = inputs(2, 3000, 70, seed=11, dtype=torch.float32)
    d = to(dev, x)
    want = run(dev, x)
    n = max(ssm.gated_scan_workspace_size(2, 3000, 70, backward=b) for b in (False, True))
    ws = torch.randn(n // 4 + 4, device=dev).view(torch.uint8)[:n].contiguous()
    if fill is not None:
        ws.fill_(fill)
    out, last, states = ssm.gated_scan_fwd(d["x"], d["f"], d["z"], d["init"], return_last_state=True, return_states=True, workspace=ws)
    if fill is not None:
        ws.fill_(fill)
    got = ssm.gated_scan_bwd(d["x"], d["f"], d["dout"], states, z=d["z"], dlast=d["dlast"], workspace=ws)
    for k, v in zip(("out", "last", "states", "dx", "df", "dz", "dinit"), (out, last, states) + got):
        assert torch.equal(v, want[k]), k


def test_operands_may_be_dropped_while_their_work_is_queued(dev):
    """A call on a side stream that is still busy: the inputs are released and their memory is written again by the main
    stream before the kernels run."""
    x = inputs(1, 2000, 64, seed=12, dtype=torch.float32)
    want = run(dev, x)["out"]
    side = torch.cuda.Stream()
    d = to(dev, x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
    out = ssm.gated_scan_fwd(d["x"], d["f"], d["z"], d["init"], stream=side)
    shapes = {k: v.shape for k, v in d.items()}
    d.clear()
    again = [torch.full(s, float("nan"), device=dev) for s in shapes.values() for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and len(again) > 0


def test_in_place(dev):
    """out may be x, f or z: every element is read before its place is written, by the same lane."""
    x = inputs(2, 700, 66, seed=13, dtype=torch.bfloat16)
    want = run(dev, x)["out"]
    for k in ("x", "f", "z"):
        d = to(dev, x)
        assert torch.equal(ssm.gated_scan_fwd(d["x"], d["f"], d["z"], d["init"], out=d[k]), want), k


def test_gradients_against_differences():
    """The oracle's gradients against central differences of the float64 forward (step 1e-5: the difference's own
    error is about 1e-10 of the loss's third derivative, and 1e-16 / 1e-5 of its value)."""
    x = {k: f64(v) for k, v in inputs(2, 9, 3, seed=3, dtype=torch.float32).items()}
    rng = np.random.default_rng(0)
    b = oracle_bwd(**x)

    def loss(**kw):
        o = oracle_fwd(**{**x, **kw})
        return float((o["out"] * x["dout"]).sum() + (o["last"] * x["dlast"]).sum())

    for name, grad in (("x", "dx"), ("f", "df"), ("z", "dz"), ("init", "dinit")):
        for _ in range(12):
            at = tuple(int(rng.integers(n)) for n in x[name].shape)
            up, dn = x[name].copy(), x[name].copy()
            up[at] += 1e-5
            dn[at] -= 1e-5
            num = (loss(**{name: up}) - loss(**{name: dn})) / 2e-5
            assert abs(num - b[grad][at]) <= 1e-7 * max(1.0, abs(num)), (name, at, num, b[grad][at])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_chunks_continue_a_sequence(dev, dtype):
    """Two calls, the second from the first's last state, are one call's rows to the bounds' rounding; so are the
    gradients, the second's dinit handed to the first as dlast."""
    x = inputs(2, 700, 70, seed=8, dtype=dtype)
    d, cut = to(dev, x), 301
    first = {k: (v[:, :cut].contiguous() if v is not None and v.dim() == 3 else v) for k, v in d.items()}
    second = {k: (v[:, cut:].contiguous() if v is not None and v.dim() == 3 else v) for k, v in d.items()}
    o1, l1, s1 = ssm.gated_scan_fwd(first["x"], first["f"], first["z"], d["init"], return_last_state=True, return_states=True)
    o2, l2, s2 = ssm.gated_scan_fwd(second["x"], second["f"], second["z"], l1, return_last_state=True, return_states=True)
    g2 = ssm.gated_scan_bwd(second["x"], second["f"], second["dout"], s2, z=second["z"], dlast=d["dlast"])
    g1 = ssm.gated_scan_bwd(first["x"], first["f"], first["dout"], s1, z=first["z"], dlast=g2[3])
    ref = {k: f64(v) for k, v in x.items()}
    o, b = oracle_fwd(**ref), oracle_bwd(**ref)
    check("out", torch.cat((o1, o2), 1), o["out"], 2 * o["out_E"], HALF[dtype])
    check("last", l2, o["last"], 2 * o["last_E"], 2.0 ** -24)
    for n, k in enumerate(("dx", "df", "dz")):
        check(k, torch.cat((g1[n], g2[n]), 1), b[k], 2 * b[k + "_E"], HALF[dtype])
    check("dinit", g1[3], b["dinit"], 2 * b["dinit_E"], 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("bt,dim", [(1, 1), (1, 1024), (3, 333), (256, 70), (7, 4096)])
def test_step(dev, bt, dim, gate, dtype):
    x = inputs(bt, 1, dim, seed=dim, dtype=dtype, gate=gate)
    state = x["init"].to(dev)
    z = x["z"][:, 0].to(dev) if gate else None
    out = ssm.gated_state_update(state, x["x"][:, 0].to(dev), x["f"][:, 0].to(dev), z)
    o = oracle_fwd(**{k: f64(v) for k, v in x.items()})
    check("out", out, o["out"][:, 0], o["out_E"][:, 0], HALF[dtype])
    check("state", state, o["last"], o["last_E"], 2.0 ** -24)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_closed_and_open_gates(dev, dtype):
    """f = +inf keeps the state and lets no gradient through to x, f = -inf takes x and forgets what came before
    (nothing before it gets a gradient through h), |f| = 200 does the same without infinities."""
    bt, L, dim = 1, 600, 4
    x = inputs(bt, L, dim, seed=4, dtype=dtype)
    x["f"][:, 100:400, 0] = float("inf")
    x["f"][:, 300, 1] = float("-inf")
    x["f"][:, 100:400, 2] = 200.0
    x["f"][:, 300, 3] = -200.0
    x["z"] = None
    got = {k: None if v is None else v.float().cpu() for k, v in run(dev, x).items()}
    for v in got.values():
        assert v is None or torch.isfinite(v).all()
    # Through the held steps the true state is one number h, that of step 99. Steps with a = 1 and i x = 0 multiply by
    # one and add nothing, exactly, alone or grouped, so each output there is some grouping of the steps up to 99: within
    # that step's bound of h (as step 99's own output is), plus half a step of storage each.
    ref = {k: f64(x[k]) for k in ("x", "f", "z", "init")}
    o = oracle_fwd(**{k: v if v is None or v.ndim < 3 else v[:, :100] for k, v in ref.items()})
    for c in (0, 2):
        h = float(o["out"][0, 99, c])
        tol = 2 * float(o["out_E"][0, 99, c]) + 2 * HALF[dtype] * abs(h)
        assert (got["out"][0, 100:400, c] - got["out"][0, 99, c]).abs().max() <= tol
        assert (got["dx"][0, 100:400, c] == 0).all() and (got["df"][0, 100:400, c] == 0).all()
    for c in (1, 3):
        assert got["out"][0, 300, c] == x["x"][0, 300, c].float()
        assert got["df"][0, 300, c] == 0


def test_not_a_number_stays_in_its_channel(dev):
    """A NaN input reaches its channel's later outputs and nothing else; the gradients that depend on it are NaN,
    those of other channels are not."""
    x = inputs(2, 900, 66, seed=5, dtype=torch.float32)
    x["x"][1, 333, 40] = float("nan")
    got = {k: v.cpu() for k, v in run(dev, x).items()}
    nan = torch.isnan(got["out"])
    assert nan[1, 333:, 40].all() and int(nan.sum()) == 900 - 333
    assert torch.isnan(got["last"][1, 40]) and int(torch.isnan(got["last"]).sum()) == 1
    for k in ("dx", "df", "dz"):
        n = torch.isnan(got[k])
        n[1, :, 40] = False
        assert not n.any(), k
    assert torch.isnan(got["df"][1, 333:, 40]).all()


def test_no_steps_and_no_rows(dev):
    init = torch.randn(3, 5, device=dev)
    e = torch.empty(3, 0, 5, device=dev)
    out, last, states = ssm.gated_scan_fwd(e, e, None, init, return_last_state=True, return_states=True)
    assert out.shape == (3, 0, 5) and torch.equal(last, init) and states.shape == (3, 0, 5)
    assert (ssm.gated_scan_fwd(e, e, return_last_state=True)[1] == 0).all()
    assert torch.equal(ssm.gated_scan_bwd(e, e, e, states, dlast=init)[3], init)
    assert (ssm.gated_scan_bwd(e, e, e, states)[3] == 0).all()
    for shape in ((0, 4, 5), (2, 4, 0)):
        e = torch.empty(shape, device=dev)
        assert ssm.gated_scan_fwd(e, e).shape == shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_same_bits_every_time_and_for_every_batch(dev, dtype):
    """Equal calls give equal bits, and a sequence's do not depend on what else is in the batch."""
    x = inputs(4, 1500, 96, seed=6, dtype=dtype)
    one, two = run(dev, x), run(dev, x)
    for k in one:
        assert torch.equal(one[k], two[k]), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_unaligned_rows(dev, dtype):
    """Operands that start one element off a wide load's alignment."""
    x = inputs(2, 300, 64, seed=7, dtype=dtype)
    d = to(dev, x)

    def off(t):
        if t is None:
            return None
        buf = torch.empty(t.numel() + 1, device=dev, dtype=t.dtype)
        v = buf[1:].view(t.shape)
        v.copy_(t)
        return v

    out, last, states = ssm.gated_scan_fwd(off(d["x"]), off(d["f"]), off(d["z"]), off(d["init"]), out=off(d["x"]),
                                           return_last_state=True, return_states=True)
    dx, df, dz, dinit = ssm.gated_scan_bwd(off(d["x"]), off(d["f"]), off(d["dout"]), off(states), z=off(d["z"]), dlast=off(d["dlast"]))
    ref = {k: f64(v) for k, v in x.items()}
    o, b = oracle_fwd(**ref), oracle_bwd(**ref)
    check("out", out, o["out"], o["out_E"], HALF[dtype])
    for k, v in (("dx", dx), ("df", df), ("dz", dz)):
        check(k, v, b[k], b[k + "_E"], HALF[dtype])


def test_captured_and_replayed(dev):
    """Forward and backward in one graph, replayed with new inputs and eager work in between: every replay gives the
    eager call's bits."""
    x = to(dev, inputs(1, 3000, 64, seed=9, dtype=torch.bfloat16))

    def step():
        out, last, states = ssm.gated_scan_fwd(x["x"], x["f"], x["z"], x["init"], return_last_state=True, return_states=True)
        return (out, last) + ssm.gated_scan_bwd(x["x"], x["f"], x["dout"], states, z=x["z"], dlast=x["dlast"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for seed in (21, 22, 23):
        new = to(dev, inputs(1, 3000, 64, seed=seed, dtype=torch.bfloat16))
        for k, v in new.items():
            x[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(kept, eager)):
            assert torch.equal(a, b), (seed, n)


def test_two_graphs_share_a_workspace(dev):
    """A forward and a backward captured apart on one workspace, of different sizes, replayed in turn on one stream."""
    xa, xb = (to(dev, inputs(1, L, d, seed=s, dtype=torch.float32)) for L, d, s in ((2500, 70, 41), (900, 200, 42)))
    n = max(ssm.gated_scan_workspace_size(1, 2500, 70), ssm.gated_scan_workspace_size(1, 900, 200, backward=True))
    ws = torch.empty(n, device=dev, dtype=torch.uint8)
    st = ssm.gated_scan_fwd(xb["x"], xb["f"], xb["z"], xb["init"], return_states=True)[1]
    calls = (lambda: (ssm.gated_scan_fwd(xa["x"], xa["f"], xa["z"], xa["init"], workspace=ws),),
             lambda: ssm.gated_scan_bwd(xb["x"], xb["f"], xb["dout"], st, z=xb["z"], dlast=xb["dlast"], workspace=ws))
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    graphs, held = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(c())
        graphs.append(g)
    for _ in range(3):
        for n in (0, 1, 1, 0):
            for t in held[n]:
                t.zero_()
            graphs[n].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held[n], want[n])), n


def test_two_streams_at_once(dev):
    """Calls on two streams, each with its own inputs, give what they give alone."""
    xs = [to(dev, inputs(1, 4000, 96, seed=s, dtype=torch.float32)) for s in (31, 32)]
    alone = [ssm.gated_scan_fwd(x["x"], x["f"], x["z"], x["init"], return_last_state=True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(4):
        got.append([ssm.gated_scan_fwd(x["x"], x["f"], x["z"], x["init"], return_last_state=True, stream=s) for x, s in zip(xs, streams)])
    torch.cuda.synchronize()
    for pair in got:
        for (o, l), (ro, rl) in zip(pair, alone):
            assert torch.equal(o, ro) and torch.equal(l, rl)
    # a raw handle works the same way
    raw = ssm.gated_scan_fwd(xs[0]["x"], xs[0]["f"], xs[0]["z"], xs[0]["init"], stream=streams[0].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(raw, alone[0][0])


def test_refusals(dev):
    x = torch.zeros(2, 8, 4, device=dev)
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.gated_scan_fwd(x, x[:, :4].contiguous())
    with pytest.raises(_ffi.DTypeMismatch):
        ssm.gated_scan_fwd(x, x.bfloat16())
    with pytest.raises(_ffi.DTypeMismatch):
        ssm.gated_scan_fwd(x.half(), x.half())
    with pytest.raises(_ffi.InvalidInput):
        ssm.gated_scan_fwd(x, x.cpu())
    with pytest.raises(_ffi.InvalidInput):
        ssm.gated_scan_fwd(x, x.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.gated_scan_bwd(x, x, x, torch.zeros(2, 2, 4, device=dev))
    with pytest.raises(_ffi.ShapeMismatch):
        ssm.gated_state_update(torch.zeros(2, 5, device=dev), x[:, 0].contiguous(), x[:, 0].contiguous())
    need = ssm.gated_scan_workspace_size(1, 100000, 4)
    assert need > 0
    big = torch.zeros(1, 100000, 4, device=dev)
    for ws in (torch.empty(need - 1, device=dev, dtype=torch.uint8), torch.empty(1, device=dev, dtype=torch.uint8).expand(need)):
        with pytest.raises(_ffi.InvalidInput):
            ssm.gated_scan_fwd(big, big, workspace=ws)
        with pytest.raises(_ffi.InvalidInput):
            ssm.gated_scan_bwd(big, big, big, torch.zeros(1, 782, 4, device=dev), workspace=ws)
    with pytest.raises(_ffi.DeviceMismatch):
        ssm.gated_scan_fwd(big, big, workspace=torch.empty(need, dtype=torch.uint8))
