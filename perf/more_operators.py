"""The operators of a linear-attention language model served in 8 bits, as cases whose time and outputs can be measured.

Five kinds, each through a public entry point of ``helixml_amd`` where ``own`` is true and in plain torch operations
(32 bits; 64 where values lie next to a rounding border) where it is false:

  attn   linear attention with one decay a head over whole sequences or one chunk of longer ones
         (``ssm.decay_attention_fwd``): S_t = e^g S_{t-1} + k_t v_t^T, out_t = scale q_t S_t
  train  the same with its backward pass (``ssm.decay_attention_fwd`` and ``ssm.decay_attention_bwd``)
  step   one token of it for every sequence of a batch (``ssm.decay_attention_step``)
  norm   a root-mean-square norm with the residual's addition, its output in 8 bits with a scale a row, or as
         fp32 or bf16 (``lm.add_rmsnorm``)
  i8     activations in 8 bits with a scale a row times weights in 8 bits with a scale an output channel
         (``ssm.linear_i8``)
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "i8": 1}
SPAN = 128  # tokens that the plain form of the attention takes at a time
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one prompt continued by a chunk of odd length, its state handed in and out
        dict(name="attn_chunk", kind="attn", batch=1, seqlen=1999, heads=12, hq=12, hk=12, hv=12, dk=64, dv=64, dtype="bf16", chunk=True, ragged=False),
        # one long document in 32 bits: the time axis holds most of the parallelism
        dict(name="attn_long", kind="attn", batch=1, seqlen=65536, heads=16, hq=16, hk=16, hv=16, dk=64, dv=64, dtype="f32", chunk=False, ragged=False),
        # a training batch of ordinary size
        dict(name="train_batch", kind="train", batch=8, seqlen=2048, heads=16, hq=16, hk=16, hv=16, dk=64, dv=64, dtype="bf16", chunk=False, ragged=False),
        # a padded batch cut in the middle: unequal lengths, keys and values shared by groups of heads, odd channels
        dict(name="train_ragged", kind="train", batch=3, seqlen=1021, heads=6, hq=6, hk=2, hv=2, dk=40, dv=72, dtype="f32", chunk=True, ragged=True),
        # a long document in training, queries and keys shared by all heads as a state-space block shares B and C: the largest call
        dict(name="train_long", kind="train", batch=1, seqlen=65536, heads=16, hq=1, hk=1, hv=16, dk=128, dv=64, dtype="bf16", chunk=False, ragged=False),
        # one token of one sequence: latency alone
        dict(name="step_one", kind="step", batch=1, heads=8, hq=8, hk=8, hv=8, dk=64, dv=64, dtype="bf16"),
        # one token for a full batch: every state read and written
        dict(name="step_batch", kind="step", batch=256, heads=16, hq=1, hk=1, hv=16, dk=128, dv=64, dtype="f32"),
        # one token between two blocks of a layer stack: the smallest call
        dict(name="norm_token", kind="norm", rows=1, dim=1024, dtype="f32", delta="bf16", norm=True, out="i8"),
        # a prompt's residual stream
        dict(name="norm_prompt", kind="norm", rows=32768, dim=2048, dtype="f32", delta="bf16", norm=True, out="i8"),
        # one token through a block's input projection
        dict(name="i8_token", kind="i8", rows=1, out=8192, inner=2048, out_type="bf16", bias=False, silu=False, add=False),
        # a serving batch through its output projection, added to the residual stream
        dict(name="i8_batch", kind="i8", rows=48, out=2048, inner=8192, out_type="f32", bias=True, silu=False, add=True),
        # a prompt of odd length through a wide projection
        dict(name="i8_prompt", kind="i8", rows=8191, out=8192, inner=2048, out_type="bf16", bias=False, silu=True, add=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "train", "step", "norm", "i8"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    dtype = rng.choice(["f32", "bf16"])
    # sizes of channels are multiples of 8 three times in four, any number else
    width = lambda lo, hi: _log(rng, lo, hi) if rng.random() < 0.25 else max(8, _log(rng, lo, hi) // 8 * 8)  # noqa: E731
    if kind in ("attn", "train", "step"):
        heads, dk, dv = _log(rng, 1, 24), width(16, 256), width(16, 256)
        of = [h for h in range(1, heads + 1) if heads % h == 0]
        shared = rng.choice(["none", "qk", "kv"])
        g = rng.choice(of)
        case = dict(kind=kind, heads=heads, hq=g if shared == "qk" else heads, hk=heads if shared == "none" else g,
                    hv=g if shared == "kv" else heads, dk=dk, dv=dv, dtype=dtype)
        if kind == "step":
            return dict(case, batch=_log(rng, 1, max(1, min(512, 256 * 16 * 128 * 64 // (heads * dk * dv)))))
        batch = _log(rng, 1, 16)
        # at most the work of the listed training case; 32 bits cost a tenth of the rate
        top = 65536 * 16 * 128 * 64 // (batch * heads * max(dk, 64) * max(dv, 64) * (1 if dtype == "bf16" else 8))
        top = max(2, min(65536, top, 65536 * 16 * 128 // (batch * heads * max(dk, dv))))
        return dict(case, batch=batch, seqlen=_log(rng, 1 if flag() else min(64, top), top), chunk=flag(), ragged=flag())
    if kind == "norm":
        dim = width(64, 16384)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(65536, 32768 * 2048 // dim))), dim=dim, dtype=rng.choice(["f32", "f32", "bf16"]),
                    delta=rng.choice(["none", "f32", "bf16"]), norm=rng.random() < 0.75, out=rng.choice(["i8", "i8", "bf16", "f32"]))
    out, inner = width(64, 16384), width(64, 16384)
    most = min(16384, 8192 * 8192 * 2048 // (out * inner))
    return dict(kind=kind, rows=_log(rng, 1, max(1, min(most, 64) if flag() else most)), out=out, inner=inner, out_type=dtype, bias=flag(), silu=flag(), add=flag())


# ------------------------------------------------------------------ inputs
def _pieces(w):
    """A weight in 8 bits [N, K] as pieces of 16 rows by 64 columns, [ceil(N / 16), ceil(K / 64), 4, 16, 16]: within a piece
    sixteen columns of every row follow each other, rows before columns; zeros behind N and K."""
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % 64, 0, -n % 16))
    return w.view(w.shape[0] // 16, 16, w.shape[1] // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo

    kind = case["kind"]
    if kind in ("attn", "train", "step"):
        b, h, dk, dv, t = case["batch"], case["heads"], case["dk"], case["dv"], TYPES[case["dtype"]]
        # memories of two to some thousand tokens
        decay = -torch.exp(uniform(math.log(2e-4), math.log(0.5), h))
        token = (b,) if kind == "step" else (b, case["seqlen"])
        s = dict(kind=kind, q=normal(*token, case["hq"], dk, dtype=t), k=normal(*token, case["hk"], dk, dtype=t),
                 v=normal(*token, case["hv"], dv, dtype=t), decay=decay, scale=dk ** -0.5)
        # a state's elements after many tokens, as large as its memory is long
        state = lambda: normal(b, h, dk, dv) * torch.rsqrt(-2.0 * decay).view(1, h, 1, 1)  # noqa: E731
        if kind == "step":
            return dict(s, state=state())
        lengths = None
        if case["ragged"]:
            lengths = torch.randint(0, case["seqlen"] + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
            lengths[0] = case["seqlen"]
        s.update(lengths=lengths, init_state=state() if case["chunk"] else None)
        if kind == "train":
            s.update(dout=normal(*token, h, dv, dtype=t), dlast=normal(b, h, dk, dv) if case["chunk"] else None)
        return s
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        # a residual stream has channels that are far larger than others
        x = normal(rows, dim) * torch.exp(normal(dim, std=0.7))
        return dict(kind=kind, x=x.to(TYPES[case["dtype"]]), delta=None if case["delta"] == "none" else normal(rows, dim, dtype=TYPES[case["delta"]]),
                    weight=1.0 + normal(dim, std=0.2) if case["norm"] else None, out_type=TYPES[case["out"]])
    m, n, k = case["rows"], case["out"], case["inner"]
    whole = lambda *shape: torch.clamp(torch.round(normal(*shape, std=36.0)), -127, 127).to(torch.int8)  # noqa: E731
    w = whole(n, k)
    return dict(kind=kind, x=whole(m, k), x_scales=uniform(0.01, 0.05, m), w=w, packed=_pieces(w), scales=uniform(0.5, 1.5, n) / (36.0 * math.sqrt(k)),
                bias=normal(n) if case["bias"] else None, silu=case["silu"],
                add=normal(m, n, dtype=TYPES[case["out_type"]]) if case["add"] else None, out_type=TYPES[case["out_type"]])


# ------------------------------------------------------------------ the plain form
def _heads(t, heads):
    return t.float().repeat_interleave(heads // t.shape[-2], -2)


def _shared(t, heads):
    """The gradient of an operand that groups of heads share: the sum over each group."""
    return t.view(*t.shape[:2], heads, t.shape[2] // heads, t.shape[3]).sum(3)


def _power(decay, n):
    """e^(n decay) for whole numbers n, none of them negative, [heads, *n.shape]; zero where n is negative."""
    p = torch.exp(decay.double().view(-1, *[1] * n.dim()) * n.clamp(min=0)).float()
    return torch.where(n < 0, torch.zeros_like(p), p)


def _mix(a, b, c, decay):
    """sum over j <= i of e^((i - j) decay) (a_i . b_j) c_j, from a zero state: spans of SPAN tokens, the states between them
    by one product with the powers of a span's decay. a, b [batch, L, heads, m], c [batch, L, heads, n]."""
    length, heads = a.shape[1], a.shape[2]
    spans = -(-length // SPAN)
    cut = lambda t: torch.nn.functional.pad(t, (0, 0, 0, 0, 0, spans * SPAN - length)).view(t.shape[0], spans, SPAN, heads, -1).permute(0, 3, 1, 2, 4)  # noqa: E731
    a, b, c = cut(a), cut(b), cut(c)  # [batch, heads, spans, SPAN, channels]
    at = torch.arange(SPAN, device=a.device)
    near = _power(decay, at.unsqueeze(1) - at).unsqueeze(1)
    out = torch.matmul(torch.matmul(a, b.transpose(-1, -2).contiguous()) * near, c)
    if spans > 1:
        to_end = _power(decay, SPAN - 1 - at).view(1, heads, 1, SPAN, 1)
        ends = torch.matmul((b * to_end).transpose(-1, -2).contiguous(), c)
        span = torch.arange(spans, device=a.device)
        far = _power(decay, (span.unsqueeze(1) - 1 - span) * SPAN)
        entry = torch.matmul(far, ends.flatten(3)).view_as(ends)
        out = out + torch.matmul(a, entry) * _power(decay, at + 1).view(1, heads, 1, SPAN, 1)
    return out.permute(0, 2, 3, 1, 4).reshape(a.shape[0], spans * SPAN, heads, -1)[:, :length]


def _plain_attention(s, train):
    h, scale, decay, lengths = s["decay"].shape[0], s["scale"], s["decay"], s["lengths"]
    q, k, v = (_heads(s[n], h) for n in ("q", "k", "v"))
    batch, length = q.shape[:2]
    at = torch.arange(length, device=q.device)
    n = torch.full((batch,), length, device=q.device) if lengths is None else lengths.long()
    there = (at < n.unsqueeze(1)).view(batch, length, 1, 1)
    q, k, v = (torch.where(there, t, torch.zeros_like(t)) for t in (q, k, v))
    since = _power(decay, at + 1).t().view(1, length, h, 1)
    left = _power(decay, n.unsqueeze(1) - 1 - at).permute(1, 2, 0).unsqueeze(-1)  # [batch, length, heads, 1], 0 behind the end
    every = _power(decay, n).t().view(batch, h, 1, 1)
    first, dlast = s["init_state"], s.get("dlast")
    rows = lambda t: t.permute(0, 2, 1, 3).contiguous()  # noqa: E731  [batch, heads, length, channels]
    times = lambda t, state: torch.matmul(rows(t), state).permute(0, 2, 1, 3)  # noqa: E731
    outer = lambda a, b: torch.matmul(rows(a).transpose(-1, -2).contiguous(), rows(b))  # noqa: E731
    out, last = _mix(q, k, v, decay), outer(k * left, v)
    if first is not None:
        out, last = out + since * times(q, first), last + every * first
    found = dict(out=out * scale, last=last)
    if not train:
        return found
    do = torch.where(there, s["dout"].float(), torch.zeros_like(out))
    back = lambda a, b, c: _mix(a.flip(1), b.flip(1), c.flip(1), decay).flip(1) * scale  # noqa: E731
    dq, dk, dv = _mix(do, v, k, decay), back(v, do, q), back(k, q, do)
    dinit = outer(q * since, do) * scale
    if first is not None:
        dq = dq + since * times(do, first.transpose(-1, -2).contiguous())
    if dlast is not None:
        dk = dk + left * times(v, dlast.transpose(-1, -2).contiguous())
        dv = dv + left * times(k, dlast)
        dinit = dinit + every * dlast
    return dict(found, dq=_shared(dq * scale, s["q"].shape[2]), dk=_shared(dk, s["k"].shape[2]), dv=_shared(dv, s["v"].shape[2]), dinit=dinit)


def _plain_norm(s):
    r = s["x"] if s["delta"] is None else (s["x"].float() + s["delta"].float()).to(s["x"].dtype)
    y, power = r.double(), 1.0
    if s["weight"] is not None:
        y, power = y * s["weight"].double(), torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    found = {} if s["delta"] is None else dict(resid=r)
    if s["out_type"] != torch.int8:
        return dict(found, y=(y * power).to(s["out_type"]))
    # a row's codes do not depend on its norm: what is rounded is y * 127 over the row's largest, ties to the even code
    top = y.abs().amax(1, keepdim=True)
    code = torch.where(top > 0, torch.round(y * 127.0 / top), torch.zeros_like(y))
    return dict(found, y=code.float() * (top * power / 127.0).float())


def _plain_product(s):
    y = s["x"].float() @ s["w"].float().t()
    y = y * (s["x_scales"].unsqueeze(1) * s["scales"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["silu"]:
        y = y * torch.sigmoid(y)
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(s["out_type"])


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    if s["kind"] in ("attn", "train"):
        found, t = _plain_attention(s, s["kind"] == "train"), s["q"].dtype
        return {n: y if n in ("last", "dinit") else y.to(t) for n, y in found.items()}
    if s["kind"] == "step":
        h = s["decay"].shape[0]
        q, k, v = (_heads(s[n], h) for n in ("q", "k", "v"))
        s["state"].copy_(torch.exp(s["decay"]).view(1, h, 1, 1) * s["state"] + k.unsqueeze(-1) * v.unsqueeze(-2))
        return dict(out=(torch.matmul(q.unsqueeze(-2), s["state"]).squeeze(-2) * s["scale"]).to(s["q"].dtype), state=s["state"])
    return _plain_norm(s) if s["kind"] == "norm" else _plain_product(s)


def _run_own(s):
    from helixml_amd import lm, ssm
    if s["kind"] in ("attn", "train"):
        q, k, v, decay = s["q"], s["k"], s["v"], s["decay"]
        out, last = ssm.decay_attention_fwd(q, k, v, decay, scale=s["scale"], lengths=s["lengths"], init_state=s["init_state"], return_last_state=True)
        if s["kind"] == "attn":
            return dict(out=out, last=last)
        dq, dk, dv, dinit = ssm.decay_attention_bwd(q, k, v, decay, s["dout"], scale=s["scale"], lengths=s["lengths"],
                                                    init_state=s["init_state"], dlast=s["dlast"])
        return dict(out=out, last=last, dq=dq, dk=dk, dv=dv, dinit=dinit)
    if s["kind"] == "step":
        return dict(out=ssm.decay_attention_step(s["state"], s["q"], s["k"], s["v"], s["decay"], scale=s["scale"]), state=s["state"])
    if s["kind"] == "norm":
        # the sum is kept, as the next block's residual stream
        resid = None if s["delta"] is None else torch.empty_like(s["x"])
        found = {} if resid is None else dict(resid=resid)
        y = lm.add_rmsnorm(s["x"], s["weight"], delta=s["delta"], eps=EPS, out_dtype=s["out_type"], resid=resid)
        return dict(found, y=torch.mul(y[0], y[1].unsqueeze(1)) if s["out_type"] == torch.int8 else y)
    # the residual stream is a user's own buffer, added to in place: a copy keeps this state's for the next pass
    out = None if s["add"] is None else s["add"].clone()
    act = (1 if s["silu"] else 0) | (2 if s["add"] is not None else 0)
    return ssm.linear_i8(s["x"], s["x_scales"], s["packed"], s["scales"], bias=s["bias"], act=act, out_dtype=s["out_type"], out=out)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("attn", "train", "step"):
        size, b, h, dk, dv = SIZE[case["dtype"]], case["batch"], case["heads"], case["dk"], case["dv"]
        tokens, state = b * case.get("seqlen", 1), 4 * b * h * dk * dv
        inputs, out = tokens * (case["hq"] * dk + case["hk"] * dk + case["hv"] * dv) * size, tokens * h * dv * size
        if kind == "step":
            return {"bytes": inputs + out + 2 * state, "flops": 5 * b * h * dk * dv}
        if kind == "attn":
            return {"bytes": inputs + out + state * (1 + int(case["chunk"])), "flops": 4 * tokens * h * dk * dv}
        # inputs q, k, v, dout; outputs out, dq, dk, dv; the states and their gradients
        return {"bytes": 2 * inputs + 2 * out + 2 * state * (1 + int(case["chunk"])), "flops": 12 * tokens * h * dk * dv}
    if kind == "norm":
        n, size = case["rows"] * case["dim"], SIZE[case["dtype"]]
        moved = size + (0 if case["delta"] == "none" else SIZE[case["delta"]] + size) + SIZE[case["out"]]
        return {"bytes": n * moved + 4 * case["dim"] * int(case["norm"]) + 4 * case["rows"] * int(case["out"] == "i8"), "flops": n * 8}
    m, n, k = case["rows"], case["out"], case["inner"]
    size = SIZE[case["out_type"]]
    return {"bytes": n * k + m * k + m * n * size * (1 + int(case["add"])) + 4 * m + 4 * n * (1 + int(case["bias"])), "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(s, train):
    h, lengths = s["decay"].shape[0], s["lengths"]
    batch, length = s["q"].shape[:2]
    keep = torch.exp(s["decay"].double()).view(1, h, 1, 1)
    wide = {n: s[n].double()[:, :, torch.arange(h, device=DEV) // (h // s[n].shape[2])].transpose(0, 1).contiguous() for n in ("q", "k", "v")}
    q, k, v = wide["q"], wide["k"], wide["v"]
    dk, dv = q.shape[-1], v.shape[-1]
    n = [length] * batch if lengths is None else lengths.tolist()
    state = torch.zeros(batch, h, dk, dv, device=DEV, dtype=torch.float64) if s["init_state"] is None else s["init_state"].double()
    out = torch.zeros(length, batch, h, dv, device=DEV, dtype=torch.float64)
    dq = torch.zeros_like(q)
    do = s["dout"].double().transpose(0, 1).contiguous() if train else None
    order = sorted(range(batch), key=lambda i: -n[i])  # the sequences that are not over stand before the others
    state, n, place = state[order], [n[i] for i in order], torch.tensor(order, device=DEV)
    back = torch.argsort(place)
    q, k, v = (t[:, place] for t in (q, k, v))
    do = do[:, place] if train else None
    alive = [sum(m > t for m in n) for t in range(length)]
    for t in range(length):  # the definition, token by token
        a = alive[t]
        if not a:
            break
        now = state[:a]
        now.mul_(keep).addcmul_(k[t, :a].unsqueeze(-1), v[t, :a].unsqueeze(-2))
        out[t, :a] = torch.matmul(q[t, :a].unsqueeze(-2), now).squeeze(-2)
        if train:
            dq[t, :a] = torch.matmul(now, do[t, :a].unsqueeze(-1)).squeeze(-1)
    scale = s["scale"]
    found = dict(out=(out[:, back] * scale).transpose(0, 1), last=state[back])
    if not train:
        return found
    grad = torch.zeros_like(state) if s["dlast"] is None else s["dlast"].double()[place]
    dkeys, dvalues = torch.zeros_like(k), torch.zeros_like(v)
    do = do * scale
    for t in reversed(range(length)):
        a = alive[t]
        if not a:
            continue
        now = grad[:a]
        now.addcmul_(q[t, :a].unsqueeze(-1), do[t, :a].unsqueeze(-2))
        dkeys[t, :a] = torch.matmul(now, v[t, :a].unsqueeze(-1)).squeeze(-1)
        dvalues[t, :a] = torch.matmul(k[t, :a].unsqueeze(-2), now).squeeze(-2)
        now.mul_(keep)

    def over(t, name):
        t, each = t[:, back].transpose(0, 1), s[name].shape[2]
        return t.unflatten(2, (each, h // each)).sum(3)

    return dict(found, dq=over(dq * scale, "q"), dk=over(dkeys, "k"), dv=over(dvalues, "v"), dinit=grad[back])


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attn", "train"):
        return _exact_attention(s, kind == "train")
    if kind == "step":
        h = case["heads"]
        q, k, v = (s[n].double()[:, torch.arange(h, device=DEV) // (h // s[n].shape[1])] for n in ("q", "k", "v"))
        state = s["state"].double() * torch.exp(s["decay"].double())[:, None, None]
        state += k[..., :, None] * v[..., None, :]
        return dict(out=(q[..., :, None] * state).sum(-2) * s["scale"], state=state)
    if kind == "norm":
        r = s["x"].double()
        if s["delta"] is not None:
            r = (r + s["delta"].double()).to(torch.float32).to(s["x"].dtype).double()  # the stream is stored, and the norm is of what is stored
        over = torch.ones(r.shape[0], 1, device=DEV, dtype=torch.float64)
        if s["weight"] is not None:
            over, y = torch.sqrt(r.square().sum(1) / r.shape[1] + EPS)[:, None], r * s["weight"].double()
        else:
            y = r
        if s["out_type"] == torch.int8:
            top = y.abs().max(1).values[:, None]
            y = torch.where(top > 0, torch.round(127 * y / top) * top, torch.zeros_like(y)) / 127
        y = y / over
        return dict(y=y) if s["delta"] is None else dict(resid=r, y=y)
    y = torch.matmul(s["x"].double(), s["w"].double().t().contiguous())
    y *= s["x_scales"].double()[:, None] * s["scales"].double()[None]
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["silu"]:
        y = y / (1.0 + torch.exp(-y))
    return y if s["add"] is None else y + s["add"].double()
