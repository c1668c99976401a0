"""The gated recurrence, 4-bit weights and logit adjustment together, as a recurrent byte LM uses them: prefill, decode
token by token from its state, a captured decode step, a training pass; and in the byte LM that is here.

Every stage of a run is held to its own float64 definition on the inputs that it had on the device, with the bounds of the
stages' own tests, so nothing is compared through another stage's rounding."""
import numpy as np
import pytest
import torch

from helixml_amd import lm, ssm
from tests.test_gated_gpu import HALF, check, f64, oracle_bwd, oracle_fwd
from tests.test_logits_gpu import compare, oracle as logits_oracle
from tests.test_w4_gpu import expand

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class RecurrentLM:
    """embed -> n x (RMSNorm -> [x | f | z] = W_in -> recurrence -> residual += W_out) -> RMSNorm -> head, weights in 4 bits."""

    def __init__(self, dev, layers=2, dim=96, vocab=300, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda n, k: ssm.w4_quantize(torch.randn(n, k, generator=g) * (2.0 / k) ** 0.5, device=dev)  # noqa: E731
        self.dim, self.vocab, self.dev = dim, vocab, dev
        self.embed = torch.randn(vocab, dim, generator=g).to(dev)
        self.norm = torch.ones(dim, device=dev)
        self.layers = [dict(x=w(dim, dim), f=w(dim, dim), z=w(dim, dim), out=w(dim, dim), bias=torch.full((dim,), 2.0, device=dev))
                       for _ in range(layers)]
        self.head = w(vocab, dim)
        self.seen = []

    def _linear(self, x, w, **kw):
        before = kw["out"].clone() if kw.get("act", 0) & 2 else None
        y = ssm.linear_w4(x, *w, **kw)
        self.seen.append(("w4", x, w, kw, before, y.clone()))
        return y

    def _mix(self, p, xn, shape):
        f = self._linear(xn, p["f"], bias=p["bias"])
        return [t.view(shape) for t in (self._linear(xn, p["x"]), f, self._linear(xn, p["z"]))]

    def run(self, tokens, states=None):
        """tokens [batch, length] -> (logits of every position, the layers' states)."""
        bt, L = tokens.shape
        r = lm.embedding(tokens, self.embed).view(bt * L, self.dim)
        last = []
        for n, p in enumerate(self.layers):
            x, f, z = self._mix(p, lm.rmsnorm(r, self.norm, out_dtype=BF), (bt, L, self.dim))
            init = None if states is None else states[n]
            y, h = ssm.gated_scan_fwd(x, f, z, init, return_last_state=True)
            self.seen.append(("scan", x, f, z, init, y, h))
            last.append(h)
            self._linear(y.view(bt * L, self.dim), p["out"], act=2, out=r)
        return self._linear(lm.rmsnorm(r, self.norm, out_dtype=BF), self.head, out_dtype=torch.float32), last

    def step(self, tokens, states, **adjust):
        """tokens [batch] -> adjusted logits; the states are advanced in place."""
        r = lm.embedding(tokens, self.embed)
        for h, p in zip(states, self.layers):
            x, f, z = self._mix(p, lm.rmsnorm(r, self.norm, out_dtype=BF), r.shape)
            before = h.clone()
            y = ssm.gated_state_update(h, x, f, z)
            self.seen.append(("step", x, f, z, before, y, h.clone()))
            self._linear(y, p["out"], act=2, out=r)
        logits = self._linear(lm.rmsnorm(r, self.norm, out_dtype=BF), self.head, out_dtype=torch.float32)
        out = lm.adjust_logits(logits, **adjust)
        self.seen.append(("logits", logits, {k: v.clone() for k, v in adjust.items()}, out.clone()))
        return out

    def hold(self):
        """Every call since the last time against its definition."""
        for s in self.seen:
            if s[0] == "w4":
                _, x, (packed, scales), kw, before, y = s
                X, w = f64(x.cpu()), expand(packed.cpu(), scales.cpu(), x.shape[1])
                want = X @ w.T
                E = x.shape[1] * 2.0 ** -23 * (np.abs(X) @ np.abs(w).T)
                for add in (kw.get("bias"), before):
                    if add is not None:
                        want = want + f64(add.cpu())
                        E = E + 2.0 ** -23 * np.abs(want)
                check("w4", y, want, E, HALF[y.dtype])
            elif s[0] in ("scan", "step"):
                x, f, z, init, y, h = [None if t is None else f64(t.cpu()) for t in s[1:]]
                if s[0] == "step":
                    x, f, z = x[:, None], f[:, None], z[:, None]
                o = oracle_fwd(x, f, z, init)
                pick = (lambda v: v[:, 0]) if s[0] == "step" else (lambda v: v)
                check("y", s[5], pick(o["out"]), pick(o["out_E"]), HALF[BF])
                check("h", s[6], o["last"], o["last_E"], 2.0 ** -24)
            else:
                compare(s[3], *logits_oracle(s[1].cpu(), **{k: v.cpu() for k, v in s[2].items()}), torch.float32)
        self.seen = []


def test_prefill_then_decode(dev):
    m = RecurrentLM(dev)
    g = torch.Generator().manual_seed(1)
    bt, L, room = 3, 150, 170
    tokens = torch.randint(0, m.vocab, (bt, L), generator=g, dtype=torch.int32).to(dev)
    logits, states = m.run(tokens)
    m.hold()
    history = torch.zeros(bt, room, device=dev, dtype=torch.int32)
    history[:, :L] = tokens
    lengths = torch.full((bt,), L, device=dev, dtype=torch.int32)
    prompts = lengths.clone()
    allowed = torch.randint(-2 ** 31, 2 ** 31, (bt, -(-m.vocab // 32)), generator=g, dtype=torch.int64).to(torch.int32).to(dev)
    flat = torch.full((bt,), 1.3, device=dev)
    kw = dict(history=history, lengths=lengths, prompt_lengths=prompts, repetition=flat, frequency=0.1 * flat, presence=0.2 * flat,
              allowed=allowed)
    token = lm.adjust_logits(logits.view(bt, L, -1)[:, -1], **kw).argmax(-1).int()
    bits = lambda t: (allowed.gather(1, (t // 32).long()[:, None])[:, 0] >> (t % 32)) & 1  # noqa: E731
    for n in range(8):
        assert bits(token).all()
        history[:, L + n] = token
        lengths += 1
        token = m.step(token, states, **kw).argmax(-1).int()
    m.hold()


def test_decode_step_in_a_graph(dev):
    m = RecurrentLM(dev, seed=2)
    g = torch.Generator().manual_seed(3)
    bt = 5
    states = [torch.randn(bt, m.dim, generator=g).to(dev) for _ in m.layers]
    token = torch.zeros(bt, device=dev, dtype=torch.int32)
    history = torch.zeros(bt, 64, device=dev, dtype=torch.int32)
    lengths = torch.zeros(bt, device=dev, dtype=torch.int32)
    kw = dict(history=history, lengths=lengths, repetition=torch.full((bt,), 1.5, device=dev))

    class Silent(list):  # nothing is kept, so nothing is copied while the graph is captured
        def append(self, _):
            pass

    m.seen = Silent()
    m.step(token, [h.clone() for h in states], **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    own = [h.clone() for h in states]
    with torch.cuda.graph(graph):
        out = m.step(token, own, **kw)
    for h, s in zip(own, states):
        h.copy_(s)
    eager = [h.clone() for h in states]
    for n in range(6):
        token.copy_(torch.randint(0, m.vocab, (bt,), generator=g, dtype=torch.int32))
        history[:, n] = token
        lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        held = out.clone()
        assert torch.equal(held, m.step(token, eager, **kw)), n
        assert all(torch.equal(a, b) for a, b in zip(own, eager)), n


def test_training_pass(dev):
    """A layer's recurrence in training: projections of a batch, the forward with its states, the backward; gradients of
    everything that went in."""
    m = RecurrentLM(dev, layers=1, seed=4)
    g = torch.Generator().manual_seed(5)
    bt, L = 2, 333
    xn = torch.randn(bt * L, m.dim, generator=g).to(dev, BF)
    x, f, z = m._mix(m.layers[0], xn, (bt, L, m.dim))
    init, dlast = (torch.randn(bt, m.dim, generator=g).to(dev) for _ in range(2))
    y, last, states = ssm.gated_scan_fwd(x, f, z, init, return_last_state=True, return_states=True)
    dout = torch.randn(bt, L, m.dim, generator=g).to(dev, BF)
    dx, df, dz, dinit = ssm.gated_scan_bwd(x, f, dout, states, z=z, dlast=dlast)
    m.hold()
    r = [f64(t.cpu()) for t in (x, f, dout, z, init, dlast)]
    b = oracle_bwd(*r)
    for k, v in (("dx", dx), ("df", df), ("dz", dz)):
        check(k, v, b[k], b[k + "_E"], HALF[BF])
    check("dinit", dinit, b["dinit"], b["dinit_E"], 2.0 ** -24)


def test_byte_lm_with_a_4_bit_head_and_adjusted_logits(dev):
    """quantize_head: logits are those of a head that holds the expanded weights in bf16 (which holds them exactly), up to
    the order of an fp32 sum of d_model products on each side: 2 K 2^-23 of sum |x w| <= |x| |w|, where the normed row has
    |x| <= sqrt(K) (1 + 2^-8). Decode with ``adjust`` is adjust_logits of the plain decode's logits, eager and captured."""
    K, bt = 64, 3
    m = lm.ByteLM(n_layers=2, d_model=K, device=dev, seed=7)
    plain = lm.ByteLM(n_layers=2, d_model=K, device=dev, seed=7)
    packed, scales = ssm.w4_quantize(m.w_head)
    w = expand(packed.cpu(), scales.cpu(), K)
    plain.w_head = torch.from_numpy(w).to(dev, BF)
    assert np.array_equal(plain.w_head.double().cpu().numpy(), w)
    m.quantize_head()
    g = torch.Generator().manual_seed(8)
    tokens = torch.randint(0, 256, (bt, 40), generator=g, dtype=torch.int32).to(dev)
    a, sa = m.prefill(tokens)
    b, sb = plain.prefill(tokens)
    tol = 2 * K * 2.0 ** -23 * np.sqrt(K) * (1 + 2.0 ** -8) * np.linalg.norm(w, axis=1)
    assert (np.abs(a.double().cpu().numpy() - b.double().cpu().numpy()) <= tol).all()
    history = torch.zeros(bt, 64, device=dev, dtype=torch.int32)
    history[:, :40] = tokens
    lengths = torch.full((bt,), 40, device=dev, dtype=torch.int32)
    kw = dict(history=history, lengths=lengths, repetition=torch.full((bt,), 1.2, device=dev), presence=torch.full((bt,), 0.5, device=dev),
              allowed=torch.randint(-2 ** 31, 2 ** 31, (8,), generator=g, dtype=torch.int64).to(torch.int32).to(dev))
    copy = lambda st: [(s.clone(), c.clone()) for s, c in st]  # noqa: E731
    s1, s2, s3 = copy(sa), copy(sa), copy(sa)
    step = m.decode_graph(s3, adjust=kw)
    for n in range(4):
        tok = torch.randint(0, 256, (bt,), generator=g, dtype=torch.int32).to(dev)
        history[:, 40 + n] = tok
        lengths += 1
        raw = m.decode_step(tok, s1)
        got = m.decode_step(tok, s2, adjust=kw)
        assert torch.equal(got, lm.adjust_logits(raw, **kw))
        assert torch.equal(step(tok), got), n
