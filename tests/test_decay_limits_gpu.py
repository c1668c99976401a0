"""Linear attention with a decay a head at the ends of what it takes: more blocks than one launch holds, no tokens at all, states that
grow, and states that live for hundreds of chunks."""
import numpy as np
import pytest
import torch

from helixml_amd import ssm
from tests.test_decay_gpu import check_all, inputs, on

F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}


@pytest.mark.gpu
@pytest.mark.parametrize("bt,heads,hq,dk,dv", [(1 << 20, 12, 12, 8, 128), (1 << 20, 12, 1, 256, 72)], ids=["two slices", "eight waves"])
def test_more_blocks_than_a_launch_holds(dev, bt, heads, hq, dk, dv):
    """batch * heads below 2^24 is taken whatever the heads' widths. One token from no state: out = scale (q . k) v."""
    g = torch.Generator(device=dev).manual_seed(dk)
    n = lambda *s: torch.randn(*s, generator=g, device=dev).to(BF16)  # noqa: E731
    q, k, v = n(bt, 1, hq, dk), n(bt, 1, hq, dk), n(bt, 1, heads, dv)
    out = ssm.decay_attention_fwd(q, k, v, torch.full((heads,), -0.5, device=dev), scale=0.25)
    for i in range(0, bt, bt // 16):  # every sequence, a sixteenth of them at a time
        at = slice(i, i + bt // 16)
        qk = q[at].float() * k[at].float()
        s, a = (t.sum(-1, keepdim=True).repeat_interleave(heads // hq, 2) for t in (qk, qk.abs()))
        want = 0.25 * s * v[at].float()
        # dk roundings of the sum here and there, a score in two bf16 parts, the output's own
        bound = 0.25 * a * v[at].float().abs() * (2 * (dk + 8) * 2.0 ** -24 + 2.0 ** -17)
        assert ((out[at].float() - want).abs() <= bound + HALF[BF16] * (want.abs() + bound) + 1e-30).all(), i


@pytest.mark.gpu
def test_more_gradients_than_a_launch_holds(dev):
    """The same for the three gradients' passes, which go out side by side: one token, so that each is one product of three."""
    bt, heads, d = 700001, 8, 8
    g = torch.Generator(device=dev).manual_seed(1)
    n = lambda: torch.randn(bt, 1, heads, d, generator=g, device=dev)  # noqa: E731
    q, k, v, do = n(), n(), n(), n()
    got = dict(zip(("dq", "dk", "dv"), ssm.decay_attention_bwd(q, k, v, torch.full((heads,), -0.5, device=dev), do, scale=0.25)))
    for name, a, b, c in (("dq", do, v, k), ("dk", do, v, q), ("dv", q, k, do)):
        s, m = (a * b).sum(-1, keepdim=True), (a * b).abs().sum(-1, keepdim=True)
        bound = 0.25 * m * c.abs() * 2 * (d + 8) * 2.0 ** -24
        assert ((got[name] - 0.25 * s * c).abs() <= bound + 1e-30).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("L,decay", [(1, [1.2, 1.0]), (3, [1.2, 0.0]), (65, [1.2, 0.5, -0.1]), (70, [1.0, 0.3]), (200, [0.4, 0.1, -0.4])])
def test_states_that_grow(dev, L, decay, dtype):
    """A growth is carried as a decay is, as long as that of 64 tokens and of the sequence fits 32 bits: in one chunk that is not whole, over
    several, over segments."""
    check_all(dev, inputs(2, L, len(decay), 24, 20, seed=L, dtype=dtype, decay=decay))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_no_tokens_and_no_sequences(dev, dtype):
    """The states pass through unchanged, of shared heads too; nothing is launched for a batch or a head count of none."""
    x = on(dev, inputs(3, 0, 4, 24, 40, seed=0, dtype=dtype, hk=2, hv=1))
    args = (x["q"], x["k"], x["v"], x["log_decay"])
    out, last = ssm.decay_attention_fwd(*args, init_state=x["init"], return_last_state=True)
    assert out.shape == (3, 0, 4, 40) and torch.equal(last, x["init"])
    dq, dk, dv, dinit = ssm.decay_attention_bwd(*args, x["dout"], init_state=x["init"], dlast=x["dlast"])
    assert dq.shape == x["q"].shape and dk.shape == x["k"].shape and dv.shape == x["v"].shape and torch.equal(dinit, x["dlast"])
    assert not ssm.decay_attention_fwd(*args, return_last_state=True)[1].any() and not ssm.decay_attention_bwd(*args, x["dout"])[3].any()
    for bt, heads in ((0, 4), (3, 0)):
        x = on(dev, inputs(bt, 7, max(heads, 1), 24, 40, seed=0, dtype=dtype))
        q, k, v, do = (x[n][:, :, :heads].contiguous() for n in ("q", "k", "v", "dout"))
        g = x["log_decay"][:heads]
        out, last = ssm.decay_attention_fwd(q, k, v, g, return_last_state=True)
        assert out.shape == (bt, 7, heads, 40) and last.shape == (bt, heads, 24, 40)
        assert [t.shape for t in ssm.decay_attention_bwd(q, k, v, g, do)] == [q.shape, k.shape, v.shape, last.shape]
        assert ssm.decay_attention_step(last, q[:, 0], k[:, 0], v[:, 0], g).shape == (bt, heads, 40)


# ------------------------------------------------------------------ states that live long
# A state of random elements decays over L tokens of zeros to e^(g L) of itself, and the mean of its elements' relative errors tells a
# factor's own error, which every element has alike and which comes again with every step, from their roundings, which have no
# common sign. With N steps (chunks, or segments) of a state:
#   the roundings of one element add up to N errors of at most 2^-24 without a mean, two each where the state is read again: over M elements
#   their mean passes 10 * 2^-24 * sqrt(2 N / M) in none of 10^20 runs (Hoeffding);
#   expm1 is off by a few units in the last place of a difference from 1 of |g| L / N, and so are the argument and the product with it: 8 * 2^-24
#   |g| L in all;
#   the last state is stored once more, and the definition is in 64 bits: 2^-24.
# A factor that is rounded to 24 bits errs by up to 2^-25 a step. The decays are chosen so that it errs by nearly that.
def mean_bound(g, L, steps, M):
    return 2.0 ** -24 * (10 * np.sqrt(2 * steps / M) + 8 * abs(g) * L + 1)


def hard_decay(tokens, about):
    """The decay next to `about` whose factor over so many tokens lies furthest from 32 bits' numbers."""
    g = np.float32(about) * (1 + np.arange(4096, dtype=np.float32) * np.float32(2.0 ** -14))
    f = np.exp(g.astype(np.float64) * tokens)
    off = f - f.astype(np.float32)
    i = int(np.abs(off).argmax())
    assert abs(off[i]) > 0.95 * 2.0 ** -25
    return float(g[i])


def test_the_bound_tells_a_rounded_factor():
    """On the CPU: a factor rounded to 32 bits passes the bound several times over, one kept as its difference from 1 does not reach it."""
    for tokens, L, M in ((32, 16384, 16384), (64, 16384, 16384), (64, 65536, 4096), (128, 65536, 4096)):
        g, steps = hard_decay(tokens, -1.0 / L), L // tokens
        s = 1 + np.random.default_rng(tokens).random(M, dtype=np.float32)
        want = s.astype(np.float64) * np.exp(g * L)
        rounded, kept = s.copy(), s.copy()
        f, d = np.float32(np.exp(g * tokens)), np.float32(np.expm1(g * tokens))
        for _ in range(steps):
            rounded = rounded * f
            kept = kept + kept * d
        bound = mean_bound(g, L, steps, M)
        assert abs(np.mean(rounded / want - 1)) > 4 * bound and abs(np.mean(kept / want - 1)) < bound, tokens


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bt,heads,L,d", [(64, 16, 16384, 16), (1, 1, 65536, 64)], ids=["whole", "cut"])
def test_states_that_live_long(dev, bt, heads, L, d, dtype):
    """Carried from chunk to chunk inside one block, and from segment to segment; the state, and its gradient the other way."""
    cut = ssm.decay_attention_workspace_size(bt, L, heads, d, d, dtype) > 0
    assert cut == (bt == 1)
    chunk = 32 if dtype == F32 else 64
    gs = [hard_decay(2 * chunk if cut else chunk, -(1.0 + i / 16) / L) for i in range(heads)]
    z = torch.zeros(bt, L, 1, d, device=dev, dtype=dtype)
    state = 1 + torch.rand(bt, heads, d, d, generator=torch.Generator(device=dev).manual_seed(3), device=dev)
    decay = torch.tensor(gs, device=dev)
    out, last = ssm.decay_attention_fwd(z, z, z, decay, init_state=state, return_last_state=True)
    assert not out.any()
    del out
    dinit = ssm.decay_attention_bwd(z, z, z, decay, torch.zeros(bt, L, heads, d, device=dev, dtype=dtype), init_state=state, dlast=state)[3]
    M = bt * d * d
    for i, g in enumerate(gs):
        want = state[:, i].double() * np.exp(g * L)
        for name, t in (("last", last), ("dinit", dinit)):
            err = float((t[:, i].double() / want - 1).mean())
            assert abs(err) <= mean_bound(g, L, L // chunk, M), (name, i, err / mean_bound(g, L, L // chunk, M))
