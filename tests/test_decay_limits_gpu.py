"""Linear attention with a decay a head at the ends of what it takes: more blocks than one launch holds, and states that live for
hundreds of chunks."""
import numpy as np
import pytest
import torch

from helixml_amd import ssm

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
