"""Timed cases of the sequence operators: layer norm, the short causal convolution and the selective state space scan.

A sequence tensor is [sequences, tokens, channels] with the channels contiguous, or [rows, channels] where sequences of
several lengths lie one behind the other.  A case is one of

* ``norm``:       y = layer norm of x (+ a residual stream, which is written too); the forward pass alone.
* ``norm_train``: that and its backward pass: gradients of x, gamma and beta.
* ``conv``:       y = silu(short causal convolution of every channel with its own filter), state in and state out.
* ``conv_train``: that without states and its backward pass: gradients of x, filters and bias.
* ``conv_step``:  one token of every sequence; the state (the last tokens) is moved on in place.
* ``scan``:       the selective scan of prompts, gated by z: state in and state out.
* ``scan_train``: that without a state in, and its backward pass: the gradients of all eight inputs.
* ``scan_step``:  one token of every sequence; the state is moved on in place.

``own`` False computes them in elementary torch operations in 32 bits; True calls ``theano_b200.sequence``.
x and z are halves of one projection's result, and B and C parts of another's, as a model's projections leave them.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NAMES = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}
EPS = 1e-5


def listed():
    return [
        # a generation step of eight sequences: the norm in front of a block, on the residual stream
        dict(name="norm_decode", kind="norm", dtype="bf16", seqs=8, tokens=1, C=1024, residual=True),
        # prompts of odd length, odd channel count
        dict(name="norm_prompt_odd", kind="norm", dtype="f16", seqs=3, tokens=2001, C=1000, residual=True),
        # training, forward and backward
        dict(name="norm_train", kind="norm_train", dtype="bf16", seqs=8, tokens=2048, C=2048, residual=False),
        # a generation step of 64 sequences
        dict(name="conv_decode", kind="conv_step", dtype="bf16", seqs=64, C=2048, width=4),
        # prompts of many lengths, packed
        dict(name="conv_prompt_ragged", kind="conv", dtype="bf16", seqs=37, tokens=8192, C=2048, width=4, ragged=True),
        # training in float32, odd length
        dict(name="conv_train_f32", kind="conv_train", dtype="f32", seqs=4, tokens=2047, C=1024, width=4),
        # a generation step of one sequence, the shortest call
        dict(name="scan_decode_one", kind="scan_step", dtype="bf16", seqs=1, C=1024, N=16, groups=1),
        # a generation step of many sequences: the states are what is read and written
        dict(name="scan_decode_batch", kind="scan_step", dtype="bf16", seqs=256, C=2048, N=16, groups=1),
        # one long prompt: few rows, the work has to be split along the tokens
        dict(name="scan_prompt_long", kind="scan", dtype="bf16", seqs=1, tokens=8192, C=2048, N=16, groups=1, ragged=False),
        # prompts of many lengths, packed
        dict(name="scan_prompt_ragged", kind="scan", dtype="f16", seqs=23, tokens=5000, C=1024, N=16, groups=1, ragged=True),
        # training
        dict(name="scan_train", kind="scan_train", dtype="bf16", seqs=4, tokens=2048, C=2048, N=16, groups=1),
        # training in float32, odd sizes, two groups of B and C
        dict(name="scan_train_f32_odd", kind="scan_train", dtype="f32", seqs=3, tokens=501, C=202, N=13, groups=2),
    ]


# ---- drawn cases -------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, lo, hi):
    c = _log(rng, lo, hi)
    return max(16, c // 16 * 16) if rng.random() < 0.7 else c


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "conv", "conv_train", "conv_step", "scan", "scan_train", "scan_step"])
    case = dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16"]))
    if kind in ("norm", "norm_train"):
        case.update(seqs=_log(rng, 1, 64), tokens=_log(rng, 1, 4096), C=_channels(rng, 32, 8192), residual=rng.random() < 0.5)
        most, axis = 32 << 20, "tokens"
        size = lambda c: c["seqs"] * c["tokens"] * c["C"]  # noqa: E731
    elif kind == "conv_step":
        case.update(seqs=_log(rng, 1, 512), C=_channels(rng, 64, 8192), width=rng.choice([2, 3, 4, 4, 4, 7]))
        most, axis = 4 << 20, "seqs"
        size = lambda c: c["seqs"] * c["C"]  # noqa: E731
    elif kind in ("conv", "conv_train"):
        case.update(seqs=_log(rng, 1, 64), tokens=_log(rng, 1, 8192), C=_channels(rng, 64, 4096), width=rng.choice([2, 3, 4, 4, 4, 7]))
        most, axis = 16 << 20, "tokens"
        if kind == "conv":
            case["ragged"] = rng.random() < 0.5
        size = lambda c: (1 if c.get("ragged") else c["seqs"]) * c["tokens"] * c["C"]  # noqa: E731
    else:
        groups = rng.choice([1, 1, 1, 2, 4])
        N = rng.choice([16, 16, 16, 8, 32, 5, 64])
        C = _channels(rng, 64, 4096)
        case.update(seqs=_log(rng, 1, 512 if kind == "scan_step" else 32), C=-(-C // groups) * groups, N=N, groups=groups)
        most, axis = 1 << 27, "tokens"
        if kind == "scan_step":
            most, axis = 1 << 23, "seqs"
            size = lambda c: c["seqs"] * c["C"] * c["N"]  # noqa: E731
        else:
            case["tokens"] = _log(rng, 1, 4096)
            if kind == "scan":
                case["ragged"] = rng.random() < 0.5
            size = lambda c: (1 if c.get("ragged") else c["seqs"]) * c["tokens"] * c["C"] * c["N"]  # noqa: E731
    while size(case) > most:                       # fewer tokens (of a step: sequences) until the pass is affordable
        case[axis] = (case[axis] + 1) // 2
    return case


def _lengths(case):
    """Lengths of a ragged case, which add up to its tokens: an empty sequence, one of a single token, the rest spread."""
    rng = random.Random(case["seqs"] * 1000003 + case["tokens"])
    n, left = case["seqs"], case["tokens"]
    cuts = sorted(rng.randint(0, left) for _ in range(n - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [left])]
    if n > 3:
        for i, want in ((1, 0), (2, 1)):
            lengths[3] += lengths[i] - want
            lengths[i] = want
        if lengths[3] < 0:                         # fewer tokens than that
            lengths = [left] + [0] * (n - 1)
    return lengths


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    C, S = case["C"], case["seqs"]
    rows = case.get("tokens", 1) * (1 if case.get("ragged") else S)
    n = rows * C
    kind = case["kind"]
    if kind == "norm":
        return {"bytes": es * (n * (4 if case["residual"] else 2) + 2 * C) + 8 * rows, "flops": 8 * n}
    if kind == "norm_train":                       # x, dy and y, dx
        return {"bytes": es * (n * (6 if case["residual"] else 4) + 4 * C) + 8 * rows, "flops": 20 * n}
    if kind == "conv_step":
        w = case["width"]
        return {"bytes": es * (2 * n + 2 * n * (w - 1) + C * (w + 1)), "flops": n * (2 * w + 5)}
    if kind == "conv":
        w = case["width"]
        return {"bytes": es * (2 * n + 2 * S * (w - 1) * C + C * (w + 1)), "flops": n * (2 * w + 5)}
    if kind == "conv_train":
        w = case["width"]
        return {"bytes": es * (4 * n + 2 * C * (w + 1)), "flops": n * (8 * w + 20)}
    N, bc = case["N"], 2 * rows * case["groups"] * case["N"]
    if kind == "scan_step":
        return {"bytes": es * (4 * n + bc) + 8 * n * N + 4 * C * (N + 2), "flops": n * (7 * N + 20)}
    if kind == "scan":
        return {"bytes": es * (4 * n + bc) + 8 * S * C * N + 4 * C * (N + 2), "flops": n * (7 * N + 20)}
    # x, dt, z, dy and y, dx, ddt, dz; B, C and their gradients; the parameters and theirs
    return {"bytes": es * (8 * n + 2 * bc) + 8 * C * (N + 2) + 4 * S * C * N, "flops": n * (28 * N + 60)}


# ---- inputs ------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    C, S, kind = case["C"], case["seqs"], case["kind"]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32) * (hi - lo) + lo

    st = dict(case=case)
    lead = (case["tokens"],) if case.get("ragged") else (S, case["tokens"]) if "tokens" in case else (S,)
    if case.get("ragged"):
        st["lengths"] = _lengths(case)
        starts = [0]
        for n in st["lengths"]:
            starts.append(starts[-1] + n)
        st["starts"] = torch.tensor(starts, dtype=torch.int64, device="cuda")
        st["seq_of"] = torch.repeat_interleave(torch.arange(S, device="cuda"), st["starts"].diff())
    empty = lambda *s, dtype=dtype: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
    if kind in ("norm", "norm_train"):
        st.update(x=normal(*lead, C) + normal(*lead, 1, scale=0.3), gamma=1 + normal(C, scale=0.2), beta=normal(C, scale=0.2), y=empty(*lead, C),
                  stats=empty(*lead, 2, dtype=torch.float32))
        if case["residual"]:
            st.update(residual=normal(*lead, C, scale=2.0), total=empty(*lead, C))
        if kind == "norm_train":
            st.update(dy=normal(*lead, C), dx=empty(*lead, C), dgamma=empty(C), dbeta=empty(C))
        return st
    projected = normal(*lead, 2 * C)               # what the convolution or scan reads and its gate, side by side
    st["x"] = projected[..., :C]
    if kind.startswith("conv"):
        w = case["width"]
        st.update(w=normal(C, w, scale=w ** -0.5), bias=normal(C, scale=0.2), y=empty(*lead, C))
        if kind == "conv_train":
            st.update(dy=normal(*lead, C), dx=empty(*lead, C), dw=empty(C, w), dbias=empty(C))
        elif kind == "conv":
            st.update(initial=normal(S, w - 1, C), final=empty(S, w - 1, C))
        else:
            st.update(state=normal(S, w - 1, C))
        return st
    N, G = case["N"], case["groups"]
    bc = normal(*lead, 2 * G * N)
    # step sizes between 1/1000 and 1/10 and decays of 1 to N, as such layers start their training with
    step = torch.exp(uniform(C, lo=math.log(1e-3), hi=math.log(1e-1)))
    st.update(z=projected[..., C:], dt=normal(*lead, C, scale=0.5), B=bc[..., :G * N].unflatten(-1, (G, N)), C=bc[..., G * N:].unflatten(-1, (G, N)),
              A=-torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * torch.exp(normal(C, N, scale=0.1, dtype=torch.float32)),
              D=1 + normal(C, scale=0.1, dtype=torch.float32), dt_bias=step + torch.log(-torch.expm1(-step)), y=empty(*lead, C))
    if kind == "scan_step":
        st.update(state=normal(S, C, N, dtype=torch.float32))
    elif kind == "scan":
        st.update(initial=normal(S, C, N, dtype=torch.float32), final=empty(S, C, N, dtype=torch.float32))
    else:
        st.update(final=empty(S, C, N, dtype=torch.float32), dy=normal(*lead, C), grads=dict(
            x=empty(*lead, C), dt=empty(*lead, C), z=empty(*lead, C), B=empty(*lead, G, N), C=empty(*lead, G, N),
            A=empty(C, N, dtype=torch.float32), D=empty(C, dtype=torch.float32), dt_bias=empty(C, dtype=torch.float32)))
    return st


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _plain_norm(st):
    dtype, x = st["x"].dtype, st["x"].float()
    out = {}
    if "residual" in st:
        out["total"] = (x + st["residual"].float()).to(dtype)
        x = out["total"].float()
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
    hat = (x - mean) * rstd
    out["y"] = (hat * st["gamma"].float() + st["beta"].float()).to(dtype)
    out["stats"] = torch.cat([mean, rstd], -1)
    if "dy" in st:
        dy = st["dy"].float()
        rows = tuple(range(dy.dim() - 1))
        g = dy * st["gamma"].float()
        out["dx"] = (rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))).to(dtype)
        out["dgamma"] = (dy * hat).sum(rows).to(dtype)
        out["dbeta"] = dy.sum(rows).to(dtype)
    return out


def _windows(st):
    """[..., channels, width]: the tokens that each result reads, the newest last, in 32 bits; zeros or the state before a sequence."""
    x, width = st["x"].float(), st["case"]["width"]
    if "starts" not in st:
        before = st["initial"].float() if "initial" in st else x.new_zeros(x.shape[0], width - 1, x.shape[2])
        return torch.cat([before, x], 1).unfold(1, width, 1)
    start = st["starts"][:-1][st["seq_of"]]
    row = torch.arange(x.shape[0], device=x.device)
    at = row[:, None] - torch.arange(width - 1, -1, -1, device=x.device)
    inside = at >= start[:, None]
    old = st["initial"].float()[st["seq_of"][:, None], (at - start[:, None] + width - 1).clamp(0, max(0, width - 2))]
    return torch.where(inside[..., None], x[at.clamp(min=0)], old).transpose(1, 2)


def _last_tokens(st):
    """The state behind each sequence: its last width - 1 tokens, those of the state before it where it is shorter."""
    x, width, initial = st["x"], st["case"]["width"], st["initial"]
    if "starts" not in st:
        return torch.cat([initial, x], 1)[:, x.shape[1]:]
    back = torch.arange(width - 1, device=x.device) - (width - 1)
    length = st["starts"].diff()
    at = length[:, None] + back                    # token of the sequence; negative: of the state before it
    new = x[(st["starts"][:-1, None] + at).clamp(0, x.shape[0] - 1)]
    old = torch.gather(initial, 1, (at + width - 1).clamp(0, width - 2)[..., None].expand(-1, -1, x.shape[1]))
    return torch.where((at >= 0)[..., None], new, old)


def _plain_conv(st):
    dtype = st["x"].dtype
    w = st["w"].float().flip(1)                    # a true convolution: the first weight meets the newest token
    win = _windows(st)
    pre = (win * w).sum(-1) + st["bias"].float()
    sig = torch.sigmoid(pre)
    out = dict(y=(pre * sig).to(dtype))
    if "initial" in st:
        out["final"] = _last_tokens(st)
    if "dy" in st:
        width, T = w.shape[1], pre.shape[1]
        g = st["dy"].float() * sig * (1 + pre * (1 - sig))
        ahead = torch.cat([g, g.new_zeros(g.shape[0], width - 1, g.shape[2])], 1).unfold(1, width, 1)
        out["dx"] = (ahead * w.flip(1)).sum(-1)[:, :T].to(dtype)
        out["dw"] = (g[..., None] * win).sum((0, 1)).flip(1).to(dtype)
        out["dbias"] = g.sum((0, 1)).to(dtype)
    return out


def _plain_conv_step(st):
    x, state = st["x"], st["state"]
    win = torch.cat([state, x[:, None]], 1)
    pre = (win.float() * st["w"].float().flip(1).t()).sum(1) + st["bias"].float()
    state.copy_(win[:, 1:])
    return dict(y=(pre * torch.sigmoid(pre)).to(x.dtype), state=state)


def _running(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along the second axis, in a logarithmic number of steps: after each, an entry stands for
    twice as many tokens."""
    a, b = a.clone(), b.clone()
    n = 1
    while n < a.shape[1]:
        b[:, n:] += a[:, n:] * b[:, :-n].clone()
        a[:, n:] *= a[:, :-n].clone()
        n *= 2
    return b


def _per_channel(v, channels):
    """B or C of a group for each of the channels that share it."""
    return v.float().repeat_interleave(channels // v.shape[-2], -2)


def _plain_scan(st):
    dtype = st["x"].dtype
    packed = "starts" in st
    batch = (lambda v: v[None]) if packed else (lambda v: v)
    x, dt, z = (batch(st[k]).float() for k in ("x", "dt", "z"))
    channels = x.shape[-1]
    raw = dt + st["dt_bias"]
    delta = torch.nn.functional.softplus(raw)
    decay = torch.exp(delta[..., None] * st["A"])
    B, C = (_per_channel(batch(st[k]), channels) for k in ("B", "C"))
    drive = (delta * x)[..., None] * B
    if "initial" in st:
        first = st["starts"][:-1][st["starts"].diff() > 0] if packed else torch.zeros(1, dtype=torch.int64, device=x.device)
        init = st["initial"][st["starts"].diff() > 0][None] if packed else st["initial"][:, None]
        drive[:, first] += decay[:, first] * init
        if packed:                                 # nothing of the sequence before it reaches a sequence's first token
            decay[:, first] = 0
    h = _running(decay, drive)
    y0 = (h * C).sum(-1) + st["D"] * x
    sig = torch.sigmoid(z)
    out = dict(y=(y0 * z * sig).to(dtype))
    if packed:
        out["y"] = out["y"][0]
        some = (st["starts"].diff() > 0)[:, None, None]
        out["final"] = torch.where(some, h[0][(st["starts"][1:] - 1).clamp(min=0)], st["initial"])
    else:
        out["final"] = h[:, -1]
    if "dy" not in st:
        return out
    dy = st["dy"].float()
    dy0 = dy * z * sig
    out["z"] = (dy * y0 * sig * (1 + z * (1 - sig))).to(dtype)
    del y0
    groups = lambda v: v.unflatten(-2, (st["B"].shape[-2], -1)).sum(-2)  # noqa: E731
    out["D"] = (dy0 * x).sum((0, 1))
    out["C"] = groups(dy0[..., None] * h).to(dtype)
    # adjoint of the states, from the last token to the first
    lam = _running(torch.cat([decay[:, :1], decay[:, 1:].flip(1)], 1), (dy0[..., None] * C).flip(1)).flip(1)
    del C
    lb = (lam * B).sum(-1)
    out["B"] = groups(lam * (delta * x)[..., None]).to(dtype)
    out["x"] = (delta * lb + dy0 * st["D"]).to(dtype)
    # what the decay passes on: lam[t] decay[t] h[t - 1]
    lam[:, 1:] *= decay[:, 1:] * h[:, :-1]
    lam[:, 0] = 0
    ddt = ((lam * st["A"]).sum(-1) + x * lb) * torch.sigmoid(raw)
    out["A"] = (lam * delta[..., None]).sum((0, 1))
    out["dt"] = ddt.to(dtype)
    out["dt_bias"] = ddt.sum((0, 1))
    return out


def _plain_scan_step(st):
    x, dt, z, state = st["x"].float(), st["dt"].float(), st["z"].float(), st["state"]
    delta = torch.nn.functional.softplus(dt + st["dt_bias"])
    B, C = (_per_channel(st[k], x.shape[-1]) for k in ("B", "C"))
    state.copy_(torch.exp(delta[..., None] * st["A"]) * state + (delta * x)[..., None] * B)
    y = ((state * C).sum(-1) + st["D"] * x) * z * torch.sigmoid(z)
    return dict(y=y.to(st["x"].dtype), state=state)


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _tensors(st):
    """The framework's tensors over the state's memory, made once, as a program that keeps its buffers does.  Who reads the results with
    torch waits for the device first."""
    if "tensors" not in st:
        from theano_b200 import sequence, shim
        ctx = shim.get_context(0)
        torch.cuda.synchronize()               # the inputs come from torch's stream, the calls run on the context's

        def wrap(t):
            return sequence.DeviceArray(ctx, t.shape, NAMES[t.dtype], strides=t.stride(), _ptr=t.data_ptr())
        st["tensors"] = {k: wrap(v) for k, v in st.items() if isinstance(v, torch.Tensor) and v.dtype in NAMES}
        if "grads" in st:
            st["tensors"]["grads"] = {k: wrap(v) for k, v in st["grads"].items()}
        st["tensors"]["sequences"] = sequence.Sequences(ctx, st["lengths"]) if "lengths" in st else None
        st["sequence"] = sequence
    return st["sequence"], st["tensors"]


def _own(st):
    q, t = _tensors(st)
    kind = st["case"]["kind"]
    if kind in ("norm", "norm_train"):
        q.device_layer_norm(t["x"], t["gamma"], t["beta"], EPS, residual=t.get("residual"), total=t.get("total"), stats=t["stats"], out=t["y"])
        if kind == "norm_train":
            q.device_layer_norm_grad(t["dy"], t.get("total") or t["x"], t["gamma"], t["stats"], out=t["dx"], dgamma=t["dgamma"], dbeta=t["dbeta"])
    elif kind == "conv":
        q.device_causal_conv1d(t["x"], t["w"], t["bias"], silu=True, initial=t["initial"], final=t["final"], sequences=t["sequences"], out=t["y"])
    elif kind == "conv_train":
        q.device_causal_conv1d(t["x"], t["w"], t["bias"], silu=True, out=t["y"])
        q.device_causal_conv1d_grad(t["dy"], t["x"], t["w"], t["bias"], silu=True, out=t["dx"], dw=t["dw"], dbias=t["dbias"])
    elif kind == "conv_step":
        q.device_causal_conv1d_step(t["x"], t["state"], t["w"], t["bias"], silu=True, out=t["y"])
    elif kind == "scan_step":
        q.device_selective_scan_step(t["x"], t["dt"], t["A"], t["B"], t["C"], t["state"], D=t["D"], z=t["z"], dt_bias=t["dt_bias"],
                                     softplus=True, out=t["y"])
    else:
        more = dict(D=t["D"], z=t["z"], dt_bias=t["dt_bias"], softplus=True, initial=t.get("initial"), sequences=t["sequences"])
        q.device_selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], final=t["final"], out=t["y"], **more)
        if kind == "scan_train":
            q.device_selective_scan_grad(t["dy"], t["x"], t["dt"], t["A"], t["B"], t["C"], grads=t["grads"], **more)
    written = ("y", "total", "stats", "dx", "dgamma", "dbeta", "final", "dw", "dbias", "state")
    return {**{k: st[k] for k in written if k in st}, **st.get("grads", {})}


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("norm", "norm_train"):
        return _plain_norm(state)
    if kind in ("conv", "conv_train"):
        return _plain_conv(state)
    if kind == "conv_step":
        return _plain_conv_step(state)
    return _plain_scan_step(state) if kind == "scan_step" else _plain_scan(state)


# ---- the definitions in 64 bits, token by token ----------------------------------------------------------------------
def _exact_norm(st):
    x = st["x"].double()
    out = {}
    if "residual" in st:
        out["total"] = (x + st["residual"].double()).to(st["x"].dtype)
        x = out["total"].double()
    mean = x.sum(-1) / x.shape[-1]
    var = ((x - mean[..., None]) ** 2).sum(-1) / x.shape[-1]
    rstd = 1 / torch.sqrt(var + EPS)
    hat = (x - mean[..., None]) * rstd[..., None]
    gamma = st["gamma"].double()
    out["y"] = hat * gamma + st["beta"].double()
    out["stats"] = torch.stack([mean, rstd], -1)
    if "total" in out:
        out["total"] = out["total"].double()
    if "dy" in st:
        dy = st["dy"].double()
        g = dy * gamma
        c1, c2 = (v.sum(-1, keepdim=True) / x.shape[-1] for v in (g, g * hat))
        out["dx"] = rstd[..., None] * (g - c1 - hat * c2)
        rows = tuple(range(x.dim() - 1))
        out["dgamma"], out["dbeta"] = (dy * hat).sum(rows), dy.sum(rows)
    return out


def _exact_conv(st):
    """Tap by tap; sequences of a ragged case one after the other."""
    width, w, bias = st["case"]["width"], st["w"].double(), st["bias"].double()
    step = "state" in st
    if "starts" in st:
        s = st["starts"].tolist()
        xs = [st["x"][a:b].double() for a, b in zip(s, s[1:])]
    else:
        xs = list(st["x"].double()[:, None] if step else st["x"].double())
    olds = st["state"] if step else st.get("initial")
    ys, finals, dxs, dw, db = [], [], [], torch.zeros_like(w), torch.zeros_like(bias)
    for i, x in enumerate(xs):
        old = olds[i].double() if olds is not None else x.new_zeros(width - 1, x.shape[1])
        ext = torch.cat([old, x])
        n = x.shape[0]
        pre = bias.expand(n, -1).clone()
        for k in range(width):                     # weight k meets the token k steps back
            pre += ext[width - 1 - k:width - 1 - k + n] * w[:, k]
        sig = 1 / (1 + torch.exp(-pre))
        ys.append(pre * sig)
        finals.append(ext[n:])
        if "dy" in st:
            g = st["dy"][i].double() * (sig + pre * sig * (1 - sig))
            dext = torch.zeros_like(ext)
            for k in range(width):
                dext[width - 1 - k:width - 1 - k + n] += g * w[:, k]
                dw[:, k] += (g * ext[width - 1 - k:width - 1 - k + n]).sum(0)
            db += g.sum(0)
            dxs.append(dext[width - 1:])
    out = dict(y=torch.cat(ys) if "starts" in st or step else torch.stack(ys))
    if olds is not None:
        out["state" if step else "final"] = torch.stack(finals)
    if dxs:
        out.update(dx=torch.stack(dxs), dw=dw, dbias=db)
    return out


def _exact_scan(st):
    packed, step = "starts" in st, "state" in st
    flat = (lambda v: v.double()[None]) if packed else (lambda v: v.double()[:, None]) if step else (lambda v: v.double())
    x, dt, z, B, C = (flat(st[k]) for k in ("x", "dt", "z", "B", "C"))
    A, D, bias = (st[k].double() for k in ("A", "D", "dt_bias"))
    rows, T, channels = x.shape
    G, N = B.shape[-2:]
    share = torch.arange(channels, device=x.device) // (channels // G)
    raw = dt + bias
    delta = raw.clamp(min=0) + torch.log1p(torch.exp(-raw.abs()))
    starts = st["starts"].tolist() if packed else None
    begin = {a: i for i, (a, b) in enumerate(zip(starts, starts[1:])) if b > a} if packed else {}
    end = {b - 1: i for i, (a, b) in enumerate(zip(starts, starts[1:])) if b > a} if packed else {}
    old = st["state"] if step else st.get("initial")
    final = old.double().clone() if old is not None else x.new_zeros(rows, channels, N)
    h = x.new_zeros(rows, channels, N) if packed else final.clone()
    grads = "dy" in st
    hs = x.new_empty(rows, T, channels, N) if grads else None
    y0 = torch.empty_like(x)
    for t in range(T):
        if t in begin:
            h = final[begin[t]][None].clone()
        d = delta[:, t, :, None]
        h = torch.exp(d * A) * h + d * x[:, t, :, None] * B[:, t, share]
        y0[:, t] = (h * C[:, t, share]).sum(-1)
        if grads:
            hs[:, t] = h
        if t in end:
            final[end[t]] = h[0]
    y0 += D * x
    gate = z / (1 + torch.exp(-z))
    y = y0 * gate
    out = dict(y=y[0] if packed else y[:, 0] if step else y)
    out["state" if step else "final"] = final if packed else h
    if not grads:
        return out
    dy = st["dy"].double()
    sig = 1 / (1 + torch.exp(-z))
    out["z"] = dy * y0 * (sig + z * sig * (1 - sig))
    dy0 = dy * gate
    dx, ddt = D * dy0, torch.empty_like(x)
    dB, dC, dA = torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    lam = torch.zeros_like(h)
    for t in range(T - 1, -1, -1):
        lam = lam + dy0[:, t, :, None] * C[:, t, share]
        d = delta[:, t, :, None]
        dC[:, t] = (dy0[:, t, :, None] * hs[:, t]).unflatten(1, (G, -1)).sum(2)
        dB[:, t] = (lam * d * x[:, t, :, None]).unflatten(1, (G, -1)).sum(2)
        lb = (lam * B[:, t, share]).sum(-1)
        lam = lam * torch.exp(d * A)
        through = lam * hs[:, t - 1] if t else torch.zeros_like(lam)
        dA += (through * d).sum(0)
        ddt[:, t] = (through * A).sum(-1) + x[:, t] * lb
        dx[:, t] += delta[:, t] * lb
    ddt = ddt / (1 + torch.exp(-raw))
    out.update(x=dx, dt=ddt, B=dB, C=dC, A=dA, D=(dy0 * x).sum((0, 1)), dt_bias=ddt.sum((0, 1)))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] in ("norm", "norm_train"):
        return _exact_norm(st)
    if case["kind"].startswith("conv"):
        return _exact_conv(st)
    return _exact_scan(st)
