"""The operators of a gated recurrent language model, as cases whose time and outputs can be measured.

Five kinds, each through a public entry point of ``helixml_amd`` where ``own`` is true and in plain
32-bit torch operations where it is false:

  scan    a gated linear recurrence over whole sequences or one chunk of a longer one
          (``ssm.gated_scan_fwd``): a = sigmoid(f), h_t = a h_{t-1} + (1 - a) x_t, out = h [silu(z)]
  train   the same with its backward pass (``ssm.gated_scan_fwd`` and ``ssm.gated_scan_bwd``)
  step    one token of that recurrence for every sequence of a batch (``ssm.gated_state_update``)
  w4      activations times 4-bit weights with group scales (``ssm.linear_w4``): OCP MXFP4, elements
          E2M1 in groups of 32 along K, one power of two a group
  logits  penalties for repeated tokens, biases and grammar masks on a decode step's logits
          (``lm.adjust_logits``)
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 32  # elements of one 4-bit weight group
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the codes 0..7; bit 3 is the sign


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one prompt continued by a chunk of odd length, its last state kept for decode
        dict(name="scan_chunk", kind="scan", batch=1, seqlen=1999, dim=768, dtype="bf16", gate=True, chunk=True),
        # one long document through few channels: the time axis holds all of the parallelism
        dict(name="scan_long", kind="scan", batch=1, seqlen=65536, dim=2048, dtype="f32", gate=False, chunk=False),
        # a training batch of ordinary size
        dict(name="train_batch", kind="train", batch=8, seqlen=2048, dim=1536, dtype="bf16", gate=True, chunk=False),
        # a few sequences cut in the middle, the state's gradient handed over, ragged in both axes
        dict(name="train_chunk", kind="train", batch=3, seqlen=1021, dim=1000, dtype="f32", gate=False, chunk=True),
        # a long document in training: the largest call
        dict(name="train_long", kind="train", batch=1, seqlen=65536, dim=2048, dtype="bf16", gate=True, chunk=False),
        # one token of one sequence: the smallest call, latency alone
        dict(name="step_one", kind="step", batch=1, dim=1024, dtype="bf16", gate=True),
        # one token for a full batch
        dict(name="step_batch", kind="step", batch=256, dim=4096, dtype="f32", gate=False),
        # one token through a large block's input projection
        dict(name="w4_token", kind="w4", rows=1, out=8192, inner=2048, out_type="bf16", bias=False, silu=False, add=False),
        # a small batch through its output projection, added to the residual stream
        dict(name="w4_batch", kind="w4", rows=16, out=2048, inner=4096, out_type="f32", bias=True, silu=False, add=True),
        # a few sequences through a wide head: the largest weight read
        dict(name="w4_head", kind="w4", rows=5, out=32768, inner=8192, out_type="f32", bias=False, silu=False, add=False),
        # the byte LM's decode batch with a grammar mask and long histories
        dict(name="logits_bytes", kind="logits", batch=256, vocab=256, history=2048, dtype="f32", prompt=False, bias=False, mask=True),
        # a subword vocabulary of odd size: every feature at once
        dict(name="logits_wide", kind="logits", batch=64, vocab=128257, history=4096, dtype="bf16", prompt=True, bias=True, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "train", "step", "w4", "logits"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    dtype = rng.choice(["f32", "bf16"])
    if kind in ("scan", "train"):
        batch, dim = _log(rng, 1, 16), _log(rng, 64, 2048)
        top = min(65536, 65536 * 2048 // (batch * dim * (1 if kind == "scan" or dtype == "bf16" else 2)))
        return dict(kind=kind, batch=batch, seqlen=_log(rng, 1 if flag() else 64, top), dim=dim, dtype=dtype, gate=flag(), chunk=flag())
    if kind == "step":
        return dict(kind=kind, batch=_log(rng, 1, 512), dim=_log(rng, 256, 8192), dtype=dtype, gate=flag())
    if kind == "w4":
        # inner sizes are whole groups three times in four, any number else
        inner = _log(rng, 256, 8192)
        inner = inner if rng.random() < 0.25 else max(GROUP, inner // GROUP * GROUP)
        return dict(kind=kind, rows=_log(rng, 1, 64), out=_log(rng, 128, 16384), inner=inner, out_type=dtype, bias=flag(), silu=flag(), add=flag())
    vocab = _log(rng, 256, 131072)
    return dict(kind=kind, batch=_log(rng, 1, max(1, min(256, 64 * 131072 // vocab))), vocab=vocab, history=_log(rng, 1, 8192), dtype=dtype,
                prompt=flag(), bias=flag(), mask=flag())


# ------------------------------------------------------------------ inputs
def _pack(w):
    """Row-major 4-bit codes (two a byte, the lower nibble first, rows of whole groups) and group exponents
    (rows padded to 16 bytes) of w [N, K]: the power of two that puts a group's largest element into E2M1's top
    binade, elements rounded to the nearest code, ties to the even code, saturated at 6."""
    n, k = w.shape
    groups = -(-k // GROUP)
    w = torch.nn.functional.pad(w, (0, groups * GROUP - k)).view(n, groups, GROUP)
    exponent = torch.frexp(w.abs().amax(-1)).exponent - 3  # floor(log2(largest)) - 2
    exponent = torch.clamp(exponent, -125, 125)
    v = torch.ldexp(w, -exponent.unsqueeze(-1))
    # midpoints between magnitudes: a tie goes to the even code
    code = sum((v.abs() > t).to(torch.uint8) if even else (v.abs() >= t).to(torch.uint8)
               for t, even in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)))
    code = code | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.view(n, groups * GROUP)
    scales = torch.full((n, -(-groups // 16) * 16), 127, dtype=torch.uint8, device=w.device)
    scales[:, :groups] = (exponent + 127).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)

    kind = case["kind"]
    if kind in ("scan", "train", "step"):
        b, d, t = case["batch"], case["dim"], TYPES[case["dtype"]]
        shape = (b, d) if kind == "step" else (b, case["seqlen"], d)
        # forget gates: a channel's own retention, half-lives from one to some hundred tokens, and the token's part
        f = normal(*shape)
        f += normal(d, std=1.5, mean=2.5)
        s = dict(x=normal(*shape, dtype=t), f=f.to(t), z=normal(*shape, dtype=t) if case["gate"] else None)
        if kind == "step":
            return dict(s, state=normal(b, d))
        chunk = case["chunk"]
        s.update(init_state=normal(b, d) if chunk else None, chunk=chunk)
        if kind == "train":
            s.update(dout=normal(*shape, dtype=t), dlast=normal(b, d) if chunk else None)
        return s
    if kind == "w4":
        n, k, m = case["out"], case["inner"], case["rows"]
        packed, scales = _pack(normal(n, k, std=math.sqrt(2.0 / k)))
        return dict(x=normal(m, k, dtype=torch.bfloat16), packed=packed, scales=scales, bias=normal(n) if case["bias"] else None,
                    silu=case["silu"], add=normal(m, n, dtype=TYPES[case["out_type"]]) if case["add"] else None, out_type=TYPES[case["out_type"]])
    b, v, h = case["batch"], case["vocab"], case["history"]
    # text repeats its frequent tokens: half of a history comes from the vocabulary's first sixteenth
    tokens = torch.where(whole(0, 2, b, h) > 0, whole(0, max(1, v // 16), b, h), whole(0, v, b, h))
    lengths = whole(0, h + 1, b)
    lengths[0] = h
    s = dict(logits=normal(b, v, std=3.0, dtype=TYPES[case["dtype"]]), history=tokens, lengths=lengths,
             prompt_lengths=torch.minimum(whole(0, h + 1, b), lengths) if case["prompt"] else None,
             repetition=1.0 + 0.5 * normal(b).abs(), frequency=0.2 * normal(b), presence=0.4 * normal(b),
             bias=normal(v) if case["bias"] else None, allowed=None)
    if case["mask"]:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (b, -(-v // 32)), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    return s


# ------------------------------------------------------------------ the plain form
def _recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, from h = 0, by doubling the span that each element covers."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat((b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]), 1)
        a = torch.cat((a[:, :span], a[:, span:] * a[:, :-span]), 1)
        span *= 2
    return b


def _plain_scan(s):
    x, f = s["x"].float(), s["f"].float()
    a, i = torch.sigmoid(f), torch.sigmoid(-f)
    b = i * x
    if s["init_state"] is not None:
        b[:, 0] += a[:, 0] * s["init_state"]
    h = _recurrence(a, b)
    z = None if s["z"] is None else s["z"].float()
    out = h if z is None else h * (z * torch.sigmoid(z))
    return x, a, i, z, h, out


def _plain_train(s):
    x, a, i, z, h, out = _plain_scan(s)
    dy = s["dout"].float()
    dz = None
    if z is not None:
        sg = torch.sigmoid(z)
        dz = dy * h * (sg * (1.0 + z * torch.sigmoid(-z)))
        dy = dy * (z * sg)
    if s["dlast"] is not None:
        dy = torch.cat((dy[:, :-1], dy[:, -1:] + s["dlast"].unsqueeze(1)), 1)  # dy can be the state's own tensor
    after = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
    g = _recurrence(after.flip(1), dy.flip(1)).flip(1)
    first = torch.zeros_like(h[:, 0]) if s["init_state"] is None else s["init_state"]
    before = torch.cat((first.unsqueeze(1), h[:, :-1]), 1)
    return out, h[:, -1], g * i, g * (before - x) * a * i, dz, a[:, 0] * g[:, 0]


def _plain_weights(s):
    n, k = s["packed"].shape[0], s["x"].shape[1]
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    code = torch.stack((s["packed"] & 15, s["packed"] >> 4), -1).view(n, -1)
    scale = torch.exp2(s["scales"][:, : code.shape[1] // GROUP].float() - 127.0)
    return (table[code.int()].view(n, -1, GROUP) * scale.unsqueeze(-1)).view(n, -1)[:, :k]


def _plain_logits(s):
    v = s["logits"].float()
    place = torch.arange(s["history"].shape[1], device=DEV)
    held = place < s["lengths"].unsqueeze(1)
    made = held if s["prompt_lengths"] is None else held & (place >= s["prompt_lengths"].unsqueeze(1))
    tokens = s["history"].long()
    seen = torch.zeros_like(v).scatter_add_(1, tokens, held.float()) > 0
    count = torch.zeros_like(v).scatter_add_(1, tokens, made.float())
    r = s["repetition"].unsqueeze(1)
    v = torch.where(seen, torch.where(v > 0, v / r, v * r), v)
    v = v - s["frequency"].unsqueeze(1) * count - s["presence"].unsqueeze(1) * (count > 0)
    if s["bias"] is not None:
        v = v + s["bias"]
    if s["allowed"] is not None:
        bits = (s["allowed"].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        v = torch.where(bits.view(v.shape[0], -1)[:, : v.shape[1]] > 0, v, torch.full_like(v, -math.inf))
    return v


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _run_own(s)
    if "dout" in s:
        t = s["x"].dtype
        out, last, dx, df, dz, dinit = _plain_train(s)
        return dict(out=out.to(t), last=last, dx=dx.to(t), df=df.to(t), dz=None if dz is None else dz.to(t), dinit=dinit)
    if "chunk" in s:
        _, _, _, _, h, out = _plain_scan(s)
        return dict(out=out.to(s["x"].dtype), last=h[:, -1].clone())
    if "state" in s:
        x, f = s["x"].float(), s["f"].float()
        s["state"].copy_(torch.sigmoid(f) * s["state"] + torch.sigmoid(-f) * x)
        z = None if s["z"] is None else s["z"].float()
        out = s["state"] if z is None else s["state"] * (z * torch.sigmoid(z))
        return dict(out=out.to(s["x"].dtype, copy=True), state=s["state"])
    if "packed" in s:
        y = s["x"].float() @ _plain_weights(s).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["silu"]:
            y = y * torch.sigmoid(y)
        if s["add"] is not None:
            y = y + s["add"].float()
        return y.to(s["out_type"])
    return _plain_logits(s).to(s["logits"].dtype)


def _run_own(s):
    from helixml_amd import lm, ssm
    if "dout" in s:
        out, last, states = ssm.gated_scan_fwd(s["x"], s["f"], s["z"], s["init_state"], return_last_state=True, return_states=True)
        dx, df, dz, dinit = ssm.gated_scan_bwd(s["x"], s["f"], s["dout"], states, z=s["z"], dlast=s["dlast"])
        return dict(out=out, last=last, dx=dx, df=df, dz=dz, dinit=dinit)
    if "chunk" in s:
        out, last = ssm.gated_scan_fwd(s["x"], s["f"], s["z"], s["init_state"], return_last_state=True)
        return dict(out=out, last=last)
    if "state" in s:
        return dict(out=ssm.gated_state_update(s["state"], s["x"], s["f"], s["z"]), state=s["state"])
    if "packed" in s:
        # the residual stream is a user's own buffer, added to in place: a copy keeps this state's for the next pass
        out = None if s["add"] is None else s["add"].clone()
        act = (1 if s["silu"] else 0) | (2 if s["add"] is not None else 0)
        return ssm.linear_w4(s["x"], s["packed"], s["scales"], bias=s["bias"], act=act, out_dtype=s["out_type"], out=out)
    return lm.adjust_logits(s["logits"], s["history"], s["lengths"], prompt_lengths=s["prompt_lengths"], repetition=s["repetition"],
                            frequency=s["frequency"], presence=s["presence"], bias=s["bias"], allowed=s["allowed"])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind in ("scan", "train", "step"):
        size, gate = (4 if case["dtype"] == "f32" else 2), int(case["gate"])
        rows = case["batch"] * case["dim"]
        n = rows * case.get("seqlen", 1)
        if kind == "step":
            return {"bytes": n * (size * (3 + gate) + 8), "flops": n * (8 + 5 * gate)}
        states = rows * 4 * (1 + int(case["chunk"]))
        if kind == "scan":
            return {"bytes": n * size * (3 + gate) + states, "flops": n * (8 + 5 * gate)}
        # inputs x, f, dout [z]; outputs out, dx, df [dz]; the states and their gradients
        return {"bytes": n * size * (6 + 2 * gate) + 2 * states, "flops": n * (24 + 12 * gate)}
    if kind == "w4":
        m, n, k = case["rows"], case["out"], case["inner"]
        size = 4 if case["out_type"] == "f32" else 2
        groups = -(-k // GROUP)
        return {"bytes": n * groups * (GROUP // 2 + 1) + m * k * 2 + m * n * size * (1 + int(case["add"])) + 4 * n * int(case["bias"]), "flops": 2 * m * n * k}
    b, v = case["batch"], case["vocab"]
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": b * (2 * size * v + 4 * case["history"] + (v + 7) // 8 * int(case["mask"]) + 20) + 4 * v * int(case["bias"]), "flops": b * v * 6}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _exact_scan(s, train):
    x, f = s["x"].double(), s["f"].double()
    z = None if s["z"] is None else s["z"].double()
    b, length, d = x.shape
    a, i = _exact_sigmoid(f), _exact_sigmoid(-f)
    h = torch.zeros(b, d, device=DEV, dtype=torch.float64) if s["init_state"] is None else s["init_state"].double()
    first = h
    every = torch.empty_like(x)
    for t in range(length):  # the definition, token by token
        h = torch.addcmul(i[:, t] * x[:, t], a[:, t], h)
        every[:, t] = h
    silu = 1.0 if z is None else z * _exact_sigmoid(z)
    found = dict(out=every * silu, last=h)
    if not train:
        return found
    dy = s["dout"].double()
    p = _exact_sigmoid(z) if z is not None else None
    found["dz"] = None if z is None else dy * every * (p + z * p * (1.0 - p))
    g = torch.zeros_like(h) if s["dlast"] is None else s["dlast"].double()
    dh = dy * silu
    dx, df = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(range(length)):
        g = g + dh[:, t]
        gi = g * i[:, t]
        dx[:, t] = gi
        df[:, t] = gi * a[:, t] * ((every[:, t - 1] if t else first) - x[:, t])
        g = g * a[:, t]
    return dict(found, dx=dx, df=df, dinit=g)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("scan", "train"):
        return _exact_scan(s, kind == "train")
    if kind == "step":
        a = _exact_sigmoid(s["f"].double())
        state = a * s["state"].double() + (1.0 - a) * s["x"].double()
        z = None if s["z"] is None else s["z"].double()
        return dict(out=state.clone() if z is None else state * z * _exact_sigmoid(z), state=state)
    if kind == "w4":
        n, k = s["packed"].shape[0], s["x"].shape[1]
        code = torch.empty(n, 2 * s["packed"].shape[1], dtype=torch.int32, device=DEV)
        code[:, 0::2], code[:, 1::2] = s["packed"] % 16, s["packed"] // 16
        e, fraction = code // 2 % 4, (code % 2).double() / 2
        w = torch.where(e == 0, fraction, (1 + fraction) * 2.0 ** (e - 1).double()) * (1 - 2 * (code // 8)).double()
        del code, e, fraction
        power = s["scales"].double() - 127
        w = w[:, :k] * (2.0 ** power).repeat_interleave(GROUP, 1)[:, :k]
        y = torch.matmul(s["x"].double(), w.t().contiguous())
        if s["bias"] is not None:
            y += s["bias"].double()
        if s["silu"]:
            y = y * _exact_sigmoid(y)
        return y if s["add"] is None else y + s["add"].double()
    b, v = case["batch"], case["vocab"]
    out = s["logits"].double()
    lengths, prompts = s["lengths"].tolist(), None if s["prompt_lengths"] is None else s["prompt_lengths"].tolist()
    for row in range(b):  # the definition, sequence by sequence
        tokens = s["history"][row, : lengths[row]].long()
        once = torch.unique(tokens)
        r = float(s["repetition"][row])
        picked = out[row, once]
        out[row, once] = torch.where(picked > 0, picked / r, picked * r)
        made, times = torch.unique(tokens if prompts is None else tokens[prompts[row]:], return_counts=True)
        out[row, made] -= float(s["frequency"][row]) * times.double() + float(s["presence"][row])
        if s["bias"] is not None:
            out[row] += s["bias"].double()
        if s["allowed"] is not None:
            at = torch.arange(v, device=DEV)
            out[row, (s["allowed"][row].long()[at // 32] >> (at % 32)) % 2 == 0] = -math.inf
    return out
