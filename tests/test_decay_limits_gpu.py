"""Linear attention with a decay a head at the ends of what it takes: more blocks than one launch holds."""
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
