"""The decayed attention, the norm to 8 bits and 8-bit products together, as a linear-attention LM uses them: a prompt, decode
token by token from its state, a captured decode step, a training pass. Every stage is held to its own float64 definition on the
inputs that it had on the device. Then what a user's program may do around the calls: streams, graphs, workspaces, far offsets."""
import numpy as np
import pytest
import torch

from helixml_amd import _ffi, lm, ssm
from tests import test_decay_gpu as attn
from tests import test_i8_gpu as i8

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


class LinearLM:
    """embed -> n x (norm to 8 bits -> [q | k | v] = W_in -> attention -> 8 bits -> residual += W_out) -> norm to 8 bits -> head."""

    def __init__(self, dev, layers=2, dim=96, heads=3, dk=16, dv=24, vocab=300, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda n, k: ssm.i8_quantize(torch.randn(n, k, generator=g) * (2.0 / k) ** 0.5, device=dev)  # noqa: E731
        self.dim, self.heads, self.dk, self.dv, self.dev = dim, heads, dk, dv, dev
        self.embed = torch.randn(vocab, dim, generator=g).to(dev)
        self.norms = [(1 + 0.1 * torch.randn(dim, generator=g)).to(dev) for _ in range(layers + 1)]
        self.layers = [dict(qkv=w(heads * (2 * dk + dv), dim), out=w(dim, heads * dv)) for _ in range(layers)]
        self.decay = -torch.exp(torch.rand(heads, generator=g) * 4 - 5).to(dev)
        self.head = w(vocab, dim)
        self.seen = []

    def _norm(self, x, weight, delta=None, resid=None):
        before = x.clone()
        y = lm.add_rmsnorm(x, weight, delta=delta, resid=resid)
        self.seen.append(("norm", before, weight, delta, resid, y))
        return y

    def _linear(self, x, w, **kw):
        y = ssm.linear_i8(*x, *w, **kw)
        self.seen.append(("linear", x, w, y))
        return y

    def _split(self, t):
        h, dk, dv = self.heads, self.dk, self.dv
        q, k, v = t.split((h * dk, h * dk, h * dv), -1)  # strided views of the projection's output
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv))

    def run(self, tokens, states=None, lengths=None):
        bt, L = tokens.shape
        r, delta, last = lm.embedding(tokens, self.embed).view(bt * L, self.dim), None, []
        for n, p in enumerate(self.layers):
            qkv = self._linear(self._norm(r, self.norms[n], delta, r), p["qkv"])
            q, k, v = self._split(qkv.view(bt, L, -1))
            init = None if states is None else states[n]
            out, h = ssm.decay_attention_fwd(q, k, v, self.decay, scale=0.25, lengths=lengths, init_state=init, return_last_state=True)
            self.seen.append(("attn", q, k, v, init, lengths, out, h))
            last.append(h)
            delta = self._linear(self._norm(out.view(bt * L, -1), None), p["out"])
        return self._linear(self._norm(r, self.norms[-1], delta, r), self.head, out_dtype=F32), last

    def step(self, tokens, states):
        r, delta = lm.embedding(tokens, self.embed), None
        for n, p in enumerate(self.layers):
            q, k, v = self._split(self._linear(self._norm(r, self.norms[n], delta, r), p["qkv"]))
            before = states[n].clone()
            out = ssm.decay_attention_step(states[n], q, k, v, self.decay, scale=0.25)
            self.seen.append(("step", q, k, v, before, out, states[n].clone()))
            delta = self._linear(self._norm(out.flatten(1), None), p["out"])
        return self._linear(self._norm(r, self.norms[-1], delta, r), self.head, out_dtype=F32)

    def hold(self):
        """Every call since the last time against its definition."""
        c = lambda t: None if t is None else t.detach().cpu().contiguous()  # noqa: E731
        for s in self.seen:
            if s[0] == "norm":
                _, x, weight, delta, resid, (q, sc) = s
                r, p, inv = i8.definition(c(x), c(weight), c(delta))
                want, scale = i8.codes_of(p, inv)
                assert np.array_equal(q.cpu().numpy(), want)
                assert (np.abs(sc.double().cpu().numpy() - scale) <= 2.0 ** -24 * scale + 2.0 ** -150).all()
            elif s[0] == "linear":
                _, (q, sc), (packed, sw), y = s
                w = torch.from_numpy(ssm.i8_values(packed, torch.ones_like(sw), q.shape[1])).to(torch.int8)
                want, bound = i8.product(c(q), c(sc), w, c(sw))
                assert (np.abs(y.double().cpu().numpy() - want) <= bound + i8.HALF[y.dtype] * (np.abs(want) + bound) + 1e-30).all()
            else:
                q, k, v, init, *_ = s[1:]
                lengths = s[5] if s[0] == "attn" else None
                if s[0] == "step":
                    q, k, v = (t.unsqueeze(1) for t in (q, k, v))
                out, last = s[-2:]
                x = dict(q=c(q), k=c(k), v=c(v), log_decay=c(self.decay), scale=0.25, lengths=c(lengths), init=c(init),
                         dout=torch.zeros(*q.shape[:2], self.heads, self.dv), dlast=None)
                want, A = attn.oracle(x)
                u = attn.unit(x)
                attn.check("out", out.view(want["out"].shape), want["out"], A["out"], u, attn.HALF[out.dtype])
                attn.check("last", last, want["last"], A["last"], u, attn.HALF[F32])
        self.seen.clear()


def test_prompt_then_tokens(dev):
    m = LinearLM(dev)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 300, (3, 75), generator=g, dtype=torch.int32).to(dev)
    _, states = m.run(tokens)
    m.hold()
    for i in range(3):
        m.step(tokens[:, i], states)
    m.hold()


def test_padded_prompts(dev):
    """A batch of prompts of unequal lengths leaves every sequence's own state."""
    m = LinearLM(dev, layers=1)
    g = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 300, (4, 130), generator=g, dtype=torch.int32).to(dev)
    lengths = torch.tensor([130, 0, 1, 66], dtype=torch.int32, device=dev)
    _, (states,) = m.run(tokens, lengths=lengths)
    m.hold()
    for b, n in enumerate(lengths.tolist()):
        if n:
            alone = m.run(tokens[b: b + 1, :n])[1][0]
            assert (states[b] - alone[0]).abs().max() <= 2.0 ** -18 * states[b].abs().max()
        else:
            assert not states[b].any()


def test_captured_step_replays(dev):
    """A captured decode step, replayed with eager work and synchronizations between, gives the eager steps' bits."""
    m = LinearLM(dev)
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 300, (2, 40), generator=g, dtype=torch.int32).to(dev)
    _, states = m.run(tokens)
    mine, tok = [s.clone() for s in states], tokens[:, 0].clone()
    scratch = [s.clone() for s in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(tok, scratch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = m.step(tok, mine)
    kept = list(m.seen)
    for i in range(5):
        tok.copy_(tokens[:, i])
        graph.replay()
        m.seen.clear()
        want = m.step(tokens[:, i], states)
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and all(torch.equal(a, b) for a, b in zip(mine, states)), i
    del kept


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("L", [100, 1300])
def test_captured_training_replays(dev, dtype, L):
    """Forward and backward captured, with and without segments, while eager tensors of the same inputs live."""
    x = attn.inputs(1, L, 2, 24, 32, seed=L, dtype=dtype)
    d = attn.on(dev, x)
    qkv = [d[n] for n in ("q", "k", "v")]

    def both():
        out, last = ssm.decay_attention_fwd(*qkv, d["log_decay"], scale=0.2, init_state=d["init"], return_last_state=True)
        return (out, last, *ssm.decay_attention_bwd(*qkv, d["log_decay"], d["dout"], scale=0.2, init_state=d["init"], dlast=d["dlast"]))

    eager = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for i in range(4):
        for t in (*qkv, d["dout"]):
            t.copy_(torch.roll(t, 1, 1))
        graph.replay()
        for a, b in zip(held, both()):
            assert torch.equal(a, b), i
    for t in (*qkv, d["dout"]):
        t.copy_(torch.roll(t, -4, 1))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_two_graphs_share_a_workspace(dev):
    """Two captured calls with one workspace, replayed in turn on one stream."""
    xs = [attn.on(dev, attn.inputs(1, 1400, 2, 16, 16, seed=s, dtype=F32)) for s in (1, 2)]
    ws = torch.empty(ssm.decay_attention_workspace_size(1, 1400, 2, 16, 16), device=dev, dtype=torch.uint8)
    assert ws.numel() > 0
    call = lambda d: ssm.decay_attention_fwd(d["q"], d["k"], d["v"], d["log_decay"], init_state=d["init"], return_last_state=True, workspace=ws)  # noqa: E731
    want = [call(d) for d in xs]
    graphs, held = [], []
    for d in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(call(d))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1):
        ws.fill_(255)
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(held[i], want[i])), i


def test_streams(dev):
    """On a stream that is given, as torch's object or as a raw handle, also where the operands are dropped right after the call;
    two streams at once, each with a workspace of its own."""
    x = attn.inputs(1, 1500, 2, 32, 32, seed=5, dtype=BF16)
    d = attn.on(dev, x)
    args = lambda: (d["q"].clone(), d["k"].clone(), d["v"].clone(), d["log_decay"])  # noqa: E731
    want = ssm.decay_attention_fwd(*args(), init_state=d["init"], return_last_state=True)
    grads = ssm.decay_attention_bwd(*args(), d["dout"], init_state=d["init"], dlast=d["dlast"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        s = streams[i % 2]
        given = s if i < 3 else s.cuda_stream
        got.append((ssm.decay_attention_fwd(*args(), init_state=d["init"], return_last_state=True, stream=given),
                    ssm.decay_attention_bwd(*args(), d["dout"], init_state=d["init"], dlast=d["dlast"], stream=given)))
        torch.empty(1 << 20, device=dev).fill_(float("nan"))
    torch.cuda.synchronize()
    for fwd, bwd in got:
        assert all(torch.equal(a, b) for a, b in zip((*fwd, *bwd), (*want, *grads)))
    p = torch.randn(40, 200, device=dev)
    q, sc = lm.add_rmsnorm(p, None)
    w = ssm.i8_quantize(torch.randn(30, 200), device=dev)
    y = ssm.linear_i8(q, sc, *w)
    torch.cuda.synchronize()
    for given in (streams[0], streams[0].cuda_stream):
        q2, sc2 = lm.add_rmsnorm(p.clone(), None, stream=given)
        y2 = ssm.linear_i8(q2, sc2, *w, stream=given)
        streams[0].synchronize()
        assert torch.equal(q, q2) and torch.equal(sc, sc2) and torch.equal(y, y2)


def test_a_dirty_and_a_larger_workspace(dev):
    for dtype in (F32, BF16):
        x = attn.inputs(1, 1300, 3, 24, 24, seed=6, dtype=dtype, hk=1, hv=1)
        d = attn.on(dev, x)
        args = (d["q"], d["k"], d["v"], d["log_decay"])
        need = ssm.decay_attention_workspace_size(1, 1300, 3, 24, 24, dtype, backward=True, k_heads=1, v_heads=1)
        want = ssm.decay_attention_bwd(*args, d["dout"], init_state=d["init"], dlast=d["dlast"])
        for more in (0, 4096):
            ws = torch.full((need + more,), 255, device=dev, dtype=torch.uint8)
            got = ssm.decay_attention_bwd(*args, d["dout"], init_state=d["init"], dlast=d["dlast"], workspace=ws)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert (ws[need:] == 255).all()
        with pytest.raises(_ffi.InvalidInput):
            ssm.decay_attention_bwd(*args, d["dout"], workspace=torch.empty(need - 1, device=dev, dtype=torch.uint8))
        with pytest.raises(_ffi.InvalidInput):
            ssm.decay_attention_bwd(*args, d["dout"], workspace=torch.empty(2 * need, device=dev, dtype=torch.uint8)[::2])


def test_refused_on_the_device(dev):
    z = lambda *s, t=F32: torch.zeros(*s, device=dev, dtype=t)  # noqa: E731
    q, g = z(2, 8, 4, 16), z(4)
    for bad in (dict(k=z(2, 8, 3, 16)), dict(k=z(2, 7, 4, 16)), dict(v=z(2, 8, 0, 16)), dict(q=z(2, 8, 4, 16).to(BF16)), dict(log_decay=z(4, t=BF16)),
                dict(q=z(2, 8, 4, 32)[..., ::2]), dict(q=z(2, 8, 4, 20)[..., :16]), dict(q=z(2, 16, 4, 16)[:, ::2].transpose(0, 1).contiguous().transpose(0, 1)),
                dict(lengths=z(2)), dict(init_state=z(2, 4, 16, 15)), dict(out=z(2, 8, 4, 15)), dict(q=z(2, 8, 4, 300), k=z(2, 8, 4, 300))):
        kw = dict(dict(q=q, k=q, v=q, log_decay=g), **bad)
        with pytest.raises(_ffi.TensorError):
            ssm.decay_attention_fwd(**kw)
    with pytest.raises(_ffi.TensorError):
        ssm.decay_attention_bwd(q, q, q, g, z(2, 8, 3, 16))
    with pytest.raises(_ffi.TensorError):
        ssm.decay_attention_step(z(2, 4, 16, 16, t=BF16), q[:, 0], q[:, 0], q[:, 0], g)
    x = z(4, 64, t=torch.int8)
    p, s = ssm.i8_quantize(torch.randn(8, 64), device=dev)
    for bad in (dict(x_scales=z(3)), dict(packed=p[:, :, :, :, :8].contiguous()), dict(scales=z(17)), dict(X=z(4, 64)), dict(X=z(4, 128, t=torch.int8)[:, ::2]),
                dict(act=2), dict(act=2, out=z(4, 9)), dict(out=z(4, 8, t=torch.float16)), dict(out_dtype=torch.int8), dict(bias=z(7))):
        kw = dict(dict(X=x, x_scales=z(4), packed=p, scales=s), **bad)
        with pytest.raises(_ffi.TensorError):
            ssm.linear_i8(**kw)
    for bad in (dict(weight=z(63)), dict(delta=z(4, 63)), dict(delta=z(4, 64, t=torch.float16)), dict(resid=z(4, 64, t=BF16)), dict(out=z(4, 128)[:, ::2]),
                dict(out=z(3, 64))):
        with pytest.raises(_ffi.TensorError):
            lm.add_rmsnorm(z(4, 64), **bad)


def test_offsets_past_32_bits(dev):
    """Operands whose far rows lie more than 2^32 bytes (and 2^31 elements) from the first: the same bits as from copies."""
    W = 1 << 22
    wide = torch.zeros(2, 300, W, device=dev, dtype=BF16)  # 2.5e9 elements
    x = attn.inputs(2, 300, 2, 32, 16, seed=9, dtype=BF16)
    d = attn.on(dev, x)
    view = wide[:, :, 5:69].unflatten(2, (2, 32))
    view.copy_(d["q"])
    assert torch.equal(ssm.decay_attention_fwd(view, d["k"], d["v"], d["log_decay"]), ssm.decay_attention_fwd(d["q"], d["k"], d["v"], d["log_decay"]))
    for a, b in zip(ssm.decay_attention_bwd(view, d["k"], d["v"], d["log_decay"], d["dout"]), ssm.decay_attention_bwd(d["q"], d["k"], d["v"], d["log_decay"], d["dout"])):
        assert torch.equal(a, b)
    rows = wide.view(600, W)[:, 100:164]
    y = torch.randn(600, 64, device=dev).to(BF16)
    rows.copy_(y)
    (q, s), (q2, s2) = lm.add_rmsnorm(rows, None), lm.add_rmsnorm(y, None)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    del rows, view, wide
    for ld in (W - 16, W + 16):  # the tiled kernel's rows and, beyond its offsets, the others'
        wide = torch.zeros(1040, ld, device=dev, dtype=torch.int8)  # 4.4e9 bytes
        X = wide[:, 16: 16 + 256]
        X.copy_(torch.randint(-127, 128, (1040, 256), device=dev, dtype=torch.int8))
        p, sw = ssm.i8_quantize(torch.randn(4096, 256), device=dev)
        sx = torch.rand(1040, device=dev)
        assert torch.equal(ssm.linear_i8(X, sx, p, sw), ssm.linear_i8(X.contiguous(), sx, p, sw))
        del wide, X
