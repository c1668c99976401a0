"""The work that users of this framework have it do, as cases whose time and outputs can be measured.

Six kinds, each through a public entry point of ``helixml_amd``:

  scan     one fused selective scan (``ssm.selective_scan_fwd``), whole sequences or one chunk of a
           longer one (an entry state given, the last state returned), fp32 or bf16 storage
  block    one Mamba block forward, bf16 (``ssm.MambaBlock``)
  prefill  the byte LM over whole prompts, logits and decode state (``lm.ByteLM.prefill``)
  decode   one token for every sequence of a batch, a captured HIP graph (``ByteLM.decode_graph``)
  s4       the S4 recurrence of the reference, one state for all channels (``ssm.s4_ref_fwd``):
           bit-exact to the reference, or time-parallel for long sequences
  s4d      the diagonal complex S4D recurrence (``ssm.s4d_complex_fwd``)

Value distributions are those of the repository's benchmark and tests. Every case is a forward; the
gated recurrence's backward pass is among the operators of ``perf/operators.py``.
"""
import math

import torch

from helixml_amd import lm, ssm

DEV = "cuda"
N = 16  # state size, the only one that the block and the LM take
LM = dict(layers=12, d_model=512, d_inner=1024, rank=32, vocab=256, conv=4)


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the benchmark's headline: a training or scoring batch through one layer's scan
        dict(name="scan_batch", kind="scan", batch=8, seqlen=2048, dim=1536, dtype="f32", chunk=False),
        # one prompt alone, its last state kept for decode: few channels, a serial sequence
        dict(name="scan_prompt", kind="scan", batch=1, seqlen=2048, dim=1536, dtype="f32", chunk=True),
        # one long document: the largest scan
        dict(name="scan_long", kind="scan", batch=1, seqlen=65536, dim=2048, dtype="f32", chunk=False),
        # a few sequences continued by a chunk of odd length, 16-bit storage, ragged channel tiles
        dict(name="scan_chunk", kind="scan", batch=3, seqlen=1021, dim=1000, dtype="bf16", chunk=True),
        # a large model's block over a batch: matrix products and scan at full size
        dict(name="block_batch", kind="block", batch=4, seqlen=4096, d_model=2048),
        # an ordinary model's block over one prompt whose length is no multiple of a tile
        dict(name="block_prompt", kind="block", batch=1, seqlen=1999, d_model=768),
        # the README example's sizes: the smallest call, launches and latency
        dict(name="block_small", kind="block", batch=1, seqlen=100, d_model=64),
        # the byte LM's whole prefill over a full batch of long prompts: the largest call
        dict(name="prefill_batch", kind="prefill", batch=16, seqlen=8192),
        # its recurrent decode for a full batch of sequences
        dict(name="decode_batch", kind="decode", batch=256),
        # the reference's own S4 benchmark size, bit-exact: a small serial recurrence
        dict(name="s4_small", kind="s4", d_model=512, seqlen=256, parallel=False),
        # the S4 recurrence over one long document, time-parallel
        dict(name="s4_long", kind="s4", d_model=2048, seqlen=65536, parallel=True),
        # S4D over the same document
        dict(name="s4d_long", kind="s4d", batch=1, seqlen=65536, dim=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "block", "block", "prefill", "decode", "s4", "s4", "s4d"])
    if kind == "scan":
        batch, dim = _log(rng, 1, 16), 2 * _log(rng, 64, 1024)
        top = min(65536, 65536 * 2048 // (batch * dim))
        return dict(kind=kind, batch=batch, seqlen=_log(rng, 64, top), dim=dim, dtype=rng.choice(["f32", "bf16"]),
                    chunk=rng.random() < 0.5)
    if kind == "block":
        batch, d_model = _log(rng, 1, 4), 2 * _log(rng, 32, 1024)
        return dict(kind=kind, batch=batch, seqlen=_log(rng, 32, 4096), d_model=d_model)
    if kind == "prefill":
        return dict(kind=kind, batch=_log(rng, 1, 16), seqlen=_log(rng, 64, 8192))
    if kind == "decode":
        return dict(kind=kind, batch=_log(rng, 1, 256))
    if kind == "s4":
        seqlen = _log(rng, 64, 65536)
        return dict(kind=kind, d_model=_log(rng, 64, 2048), seqlen=seqlen, parallel=seqlen >= 2048)
    batch = _log(rng, 1, 4)
    dim = _log(rng, 64, 2048)
    return dict(kind=kind, batch=batch, seqlen=_log(rng, 256, min(65536, 65536 * 2048 // (batch * dim))), dim=dim)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)

    kind = case["kind"]
    if kind == "scan":
        b, l, d = case["batch"], case["seqlen"], case["dim"]
        t = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        x = dict(u=normal(b, l, d, dtype=t), delta=normal(b, l, d, std=0.5, mean=-4.0, dtype=t),
                 A=-torch.arange(1, N + 1, device=DEV, dtype=torch.float32).repeat(d, 1),
                 B=normal(b, l, N, dtype=t), C=normal(b, l, N, dtype=t), D=normal(d), z=normal(b, l, d, dtype=t))
        if case["chunk"]:
            x.update(dt_bias=normal(d, std=0.1), init_state=normal(b, d, N, std=0.1), return_last_state=True)
        return x
    if kind == "block":
        block = ssm.MambaBlock(case["d_model"], device=DEV, generator=torch.Generator().manual_seed(seed))
        return dict(block=block, x=normal(case["batch"], case["seqlen"], case["d_model"], dtype=torch.bfloat16))
    if kind == "prefill":
        tokens = torch.randint(0, LM["vocab"], (case["batch"], case["seqlen"]), generator=g, device=DEV, dtype=torch.int32)
        return dict(model=lm.ByteLM(device=DEV, seed=seed), tokens=tokens)
    if kind == "decode":
        model, b = lm.ByteLM(device=DEV, seed=seed), case["batch"]
        state = model.new_state(b)
        for s, c in state:
            s.copy_(normal(*s.shape, std=0.2))
            c.copy_(normal(*c.shape))
        tokens = torch.randint(0, LM["vocab"], (b,), generator=g, device=DEV, dtype=torch.int32)
        return dict(model=model, tokens=tokens, state=state, step=model.decode_graph(state))
    if kind == "s4":
        m, l = case["d_model"], case["seqlen"]
        if case["parallel"]:
            x = normal(m, l)
            a_real = torch.full((N,), -0.5, device=DEV)
            a_imag = math.pi * torch.arange(N, device=DEV, dtype=torch.float32)
            D = normal(m)
        else:  # the reference's own initialisation
            x = torch.rand((m, l), generator=g, device=DEV) * 2 - 1
            a_real, a_imag, D = torch.zeros(N, device=DEV), normal(N), torch.zeros(m, device=DEV)
        return dict(x=x, a_real=a_real, a_imag=a_imag, B=normal(N, m, std=0.1), C=normal(m, N, std=0.1), D=D,
                    a=ssm.s4_discretize(a_real, a_imag, 0.1, device=DEV), parallel=case["parallel"])
    b, l, d = case["batch"], case["seqlen"], case["dim"]
    parts = {k: normal(d, N, std=0.1) for k in ("B_re", "B_im", "C_re", "C_im")}
    return dict(x=normal(b, l, d), dt=torch.full((d,), 0.1, device=DEV), a_re=torch.full((d, N), -0.5, device=DEV),
                a_im=(math.pi * torch.arange(N, device=DEV, dtype=torch.float32)).repeat(d, 1), D=normal(d), **parts)


# ------------------------------------------------------------------ one pass
def run(state):
    if "step" in state:
        return state["step"](state["tokens"]), state["state"]
    if "model" in state:
        return state["model"].prefill(state["tokens"])
    if "block" in state:
        return state["block"](state["x"])
    if "u" in state:
        return ssm.selective_scan_fwd(**state)
    if "parallel" in state:
        return ssm.s4_ref_fwd(**state)
    return ssm.s4d_complex_fwd(**state)


# ------------------------------------------------------------------ what a pass cannot do without
def _scan_flops(tokens, dim):
    # per state and step: dt*A, exp, B*(dt*u), the recurrence's and the readout's multiply-add
    return tokens * dim * (7 * N + 10)


def _block_flops(tokens, dm, di, rank):
    return 2 * tokens * (2 * di * dm + (rank + 2 * N) * di + rank * di + di * dm) + _scan_flops(tokens, di)


def _block_bytes(dm, di, rank):
    return 2 * (2 * di * dm + (rank + 2 * N) * di + rank * di + di * dm) + 4 * di * (N + 7)


def work(case):
    kind = case["kind"]
    if kind == "scan":
        b, l, d = case["batch"], case["seqlen"], case["dim"]
        es = 4 if case["dtype"] == "f32" else 2
        return dict(bytes=es * b * l * (4 * d + 2 * N) + 4 * d * (N + 1) + (8 * b * d * N + 4 * d if case["chunk"] else 0),
                    flops=_scan_flops(b * l, d))
    if kind == "block":
        t, dm = case["batch"] * case["seqlen"], case["d_model"]
        di, rank = 2 * dm, -(-dm // 16)
        return dict(bytes=4 * t * dm + _block_bytes(dm, di, rank), flops=_block_flops(t, dm, di, rank))
    if kind in ("prefill", "decode"):
        b = case["batch"]
        t = b * case.get("seqlen", 1)
        dm, di, rank, vocab = LM["d_model"], LM["d_inner"], LM["rank"], LM["vocab"]
        state = 4 * b * di * (N + LM["conv"] - 1) * (1 if kind == "prefill" else 2)
        return dict(bytes=4 * t * (1 + vocab) + 6 * vocab * dm + LM["layers"] * (_block_bytes(dm, di, rank) + 4 * dm + state),
                    flops=LM["layers"] * _block_flops(t, dm, di, rank) + 2 * t * vocab * dm)
    if kind == "s4":
        m, l = case["d_model"], case["seqlen"]
        return dict(bytes=8 * m * l + 4 * m * (2 * N + 1), flops=m * l * (4 * N + 2) + 2 * l * N)
    b, l, d = case["batch"], case["seqlen"], case["dim"]
    # per complex state and step: the rotation and input (4 multiply-adds), the real readout (2)
    return dict(bytes=8 * b * l * d + 4 * d * (6 * N + 2), flops=b * l * d * (12 * N + 2))


def tolerance(case):
    """About four times what the path's own forms differ by (its other kernels, tilings and segment counts, which sum in
    other orders): 3e-8 to 3e-7 in fp32; 2e-5 where fp32 results are rounded to 16-bit outputs, one unit of which is
    6e-3 of a value; 1e-3 through one block's 16-bit intermediates, 3e-3 to 1.5e-2 through twelve layers."""
    kind = case["kind"]
    if kind == "s4" and not case["parallel"]:
        return "exact"  # this mode keeps the reference's order of operations bit for bit
    if kind in ("s4", "s4d") or kind == "scan" and case["dtype"] == "f32":
        return dict(rel=1.5e-6, max=3e-5)
    if kind == "scan":
        return dict(rel=1e-4, max=0.025)
    if kind == "block":
        return dict(rel=4e-3, max=0.05)
    return dict(rel=1.4e-2, max=0.16) if kind == "decode" else dict(rel=0.03, max=0.99)


# ------------------------------------------------------------------ the same in 64 bits
def _silu(x):
    return x * torch.sigmoid(x)


def _scan64(u, dt, A, B, C, D, z, h):
    """The recurrence in 64 bits, 128 steps' decays at a time; the output and the last state."""
    out = torch.empty_like(u)
    for t0 in range(0, u.shape[1], 128):
        s = slice(t0, min(t0 + 128, u.shape[1]))
        decay = torch.exp(dt[:, s, :, None] * A)
        hs = (dt[:, s] * u[:, s])[..., None] * B[:, s, None, :]
        for k in range(hs.shape[1]):
            h = torch.addcmul(hs[:, k], decay[:, k], h)
            hs[:, k] = h
        out[:, s] = ((hs * C[:, s, None, :]).sum(-1) + D * u[:, s]) * _silu(z[:, s])
    return out, h


def _conv64(x, weight, bias):
    """Causal depthwise convolution and SiLU over [batch, seqlen, channels] that starts with width - 1 earlier rows."""
    w = weight.shape[1]
    l = x.shape[1] - w + 1
    return _silu(bias + sum(x[:, j:j + l] * weight[:, j] for j in range(w)))


def _block64(x, p, window=None, h=None):
    """One Mamba block: output, last state, and the last width - 1 rows that the convolution saw."""
    p = {k: v.double() for k, v in p.items()}
    di, rank = p["w_dt"].shape
    b = x.shape[0]
    xz = x @ p["w_in"].T
    w = p["conv_w"].shape[1]
    seen = torch.cat([x.new_zeros(b, w - 1, di) if window is None else window, xz[..., :di]], 1)
    u = _conv64(seen, p["conv_w"], p["conv_b"])
    low, B, C = (u @ p["w_x"].T).split([rank, N, N], -1)
    dt = torch.nn.functional.softplus(low @ p["w_dt"].T + p["dt_bias"], threshold=60)
    y, h = _scan64(u, dt, p["A"], B, C, p["D"], xz[..., di:], x.new_zeros(b, di, N) if h is None else h)
    return y @ p["w_out"].T, h, seen[:, -(w - 1):]


def _norm64(x, weight, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "scan":
        f = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
        dt = f["delta"] + f["dt_bias"] if "dt_bias" in f else f["delta"]
        dt = torch.nn.functional.softplus(dt, threshold=60)
        h = f.get("init_state")
        if h is None:
            h = f["u"].new_zeros(case["batch"], case["dim"], N)
        out = _scan64(f["u"], dt, f["A"], f["B"], f["C"], f["D"], f["z"], h)
        return out if case["chunk"] else out[0]
    if kind == "block":
        return _block64(s["x"].double(), s["block"].parameters())[0]
    if kind in ("prefill", "decode"):
        m, state = s["model"], []
        x = m.embed.double()[s["tokens"].long()]
        x = x if kind == "prefill" else x[:, None]
        for i, layer in enumerate(m.layers):
            h, window = (v.double() for v in s["state"][i]) if kind == "decode" else (None, None)
            p = {k: v for k, v in layer.items() if k != "norm_w"}
            y, h, window = _block64(_norm64(x, layer["norm_w"], m.eps), p, window, h)
            x = x + y
            state.append((h, window))
        logits = _norm64(x, m.norm_f, m.eps) @ m.w_head.double().T
        return logits if kind == "prefill" else logits[:, 0], state
    f = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    if kind == "s4":
        a = torch.exp(f["a_real"] * 0.1) * torch.cos(f["a_imag"] * 0.1)
        hs = (f["x"].T @ (0.1 * f["B"]).T).contiguous()
        h = torch.zeros(N, device=DEV, dtype=torch.float64)
        for t in range(hs.shape[0]):
            h = torch.addcmul(hs[t], a, h)
            hs[t] = h
        return hs @ f["C"].T + f["D"] * f["x"].T
    dt, x = f["dt"][:, None], f["x"]
    a = torch.exp(dt * torch.complex(f["a_re"], f["a_im"]))
    gain = torch.complex(f["C_re"], f["C_im"]) * torch.complex(f["B_re"], f["B_im"]) * dt
    h = torch.zeros(case["batch"], *a.shape, device=DEV, dtype=torch.complex128)
    y = torch.empty_like(x)
    for t0 in range(0, x.shape[1], 64):
        hs = x[:, t0:t0 + 64, :, None].to(torch.complex128).repeat(1, 1, 1, N)
        for k in range(hs.shape[1]):
            h = torch.addcmul(hs[:, k], a, h)
            hs[:, k] = h
        y[:, t0:t0 + 64] = 2 * (hs * gain).sum(-1).real + f["D"] * x[:, t0:t0 + 64]
    return y
