"""What is timed of the state-space operators: the short causal convolution, the selective scan and the gated group norm.

``listed()`` names twelve cases, ``draw(rng)`` gives one more of the same ranges.  Each case is a dict of plain values with
a ``kind``:

  conv    causal depthwise convolution over the last few tokens with SiLU: ``task`` "step" (one token, the kept inputs
          updated in place), "prompt" (a run of tokens from nothing, kept inputs returned) or "train" (every gradient)
  scan    selective scan s_t = exp(delta_t a) s_(t-1) + delta_t b_t x_t, y_t = c_t . s_t + d x_t: the same three tasks
  norm    normalisation of groups of channels of each token, gated by silu(gate): "prompt" (no gradients) or "train"

Activations are time-major ``[tokens, batch, channels]`` as everywhere in this package.  What a layer's projections put side
by side in one array (the convolution's input and the gate; the step size's low-rank part, b and c) is handed over as views
of that array.  Step sizes softplus(dt + dt_bias) are spread over about 0.001 to 0.1 by their biases, a = -(1 ... N) with
some noise; padded sequences have lengths uniform in [T/2, T].
"""
import math

import torch
import torch.nn.functional as F

DEV = "cuda"
own = False
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # interactive generation: the convolution of one token of eight sequences; launches and latency
        dict(name="conv_step", kind="conv", task="step", batch=8, tokens=1, channels=1024, width=4, dtype="float16", padded=False),
        # prompt of a generation at the headline batch
        dict(name="conv_prompt", kind="conv", task="prompt", batch=8, tokens=2048, channels=2048, width=4, dtype="bfloat16", padded=False),
        # training step on a padded batch of sentences
        dict(name="conv_train", kind="conv", task="train", batch=24, tokens=150, channels=1024, width=4, dtype="float16", padded=True),
        # interactive generation: the scan's step of one layer
        dict(name="scan_step", kind="scan", task="step", batch=8, tokens=1, channels=2048, states=16, groups=1, dtype="bfloat16", padded=False),
        # batch generation: the states of 256 sequences stream from memory for every token
        dict(name="scan_step_batch", kind="scan", task="step", batch=256, tokens=1, channels=2048, states=16, groups=1, dtype="bfloat16", padded=False),
        # prompt of a generation at the headline batch: outputs and the state that decoding goes on from
        dict(name="scan_prompt", kind="scan", task="prompt", batch=8, tokens=2048, channels=2048, states=16, groups=1, dtype="bfloat16", padded=False),
        # one long document: few rows, so the time axis itself has to be split
        dict(name="scan_long", kind="scan", task="prompt", batch=1, tokens=16384, channels=1024, states=16, groups=1, dtype="float16", padded=False),
        # training step at the headline batch
        dict(name="scan_train", kind="scan", task="train", batch=8, tokens=2048, channels=2048, states=16, groups=1, dtype="bfloat16", padded=False),
        # a small single-precision model on a ragged batch, sizes that are multiples of little, two groups of b and c
        dict(name="scan_ragged", kind="scan", task="train", batch=3, tokens=531, channels=520, states=12, groups=2, dtype="float32", padded=True),
        # the norm of one token of eight sequences: launches and latency
        dict(name="norm_step", kind="norm", task="prompt", batch=8, tokens=1, channels=1024, groups=16, dtype="float16"),
        # prompt of a generation at the headline batch, groups of a head's width
        dict(name="norm_prompt", kind="norm", task="prompt", batch=8, tokens=2048, channels=2048, groups=32, dtype="bfloat16"),
        # training step on few sequences of a length that is a multiple of nothing
        dict(name="norm_train", kind="norm", task="train", batch=3, tokens=1531, channels=2048, groups=32, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["conv", "scan", "scan", "norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    task = rng.choice(["prompt", "train"] if kind == "norm" else ["step", "prompt", "train"])
    # widths of real layers are multiples of 64; other ones are allowed, and every fourth case has one
    channels = 64 * _log(rng, 1, 32) if rng.random() < 0.75 else _log(rng, 5, 2000)
    tokens = 1 if task == "step" else _log(rng, 2, 8192)
    case = dict(kind=kind, task=task, tokens=tokens, channels=channels, dtype=dtype)
    case["batch"] = _log(rng, 1, max(1, min(256, 32 * 2 ** 20 // (tokens * channels))))
    if kind == "conv":
        return dict(case, width=rng.choice([2, 3, 4, 4, 4]), padded=task != "step" and rng.random() < 0.5)
    if kind == "norm":
        return dict(case, groups=rng.choice([g for g in range(1, channels + 1) if channels % g == 0 and channels // g <= 2048]))
    states = rng.choice([4, 8, 12, 16, 16, 16, 32, 64])
    case["batch"] = max(1, case["batch"] * 16 // max(16, states))
    return dict(case, states=states, groups=rng.choice([g for g in (1, 1, 2, 4) if channels % g == 0]), padded=task != "step" and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _padding(gen, batch, tokens):
    """[batch, tokens] with True at the padded positions, lengths uniform in [tokens / 2, tokens]."""
    lengths = torch.randint((tokens + 1) // 2, tokens + 1, (batch, 1), generator=gen, device=DEV)
    return torch.arange(tokens, device=DEV)[None] >= lengths


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    T, B, D, half = case["tokens"], case["batch"], case["channels"], TYPES[case["dtype"]]
    train = case["task"] == "train"

    def randn(*shape, scale=1.0, dtype=half):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    st = dict(kind=case["kind"], task=case["task"], pad=_padding(gen, B, T) if case.get("padded") else None)
    if train:
        st["g"] = randn(T, B, D)
    if case["kind"] == "conv":
        W = case["width"]
        st["x"] = randn(T, B, 2 * D)[..., :D]                   # the first half of the input projection
        st["weight"], st["bias"] = randn(D, W, scale=W ** -0.5), randn(D, scale=0.1)
        if case["task"] == "step":
            st["state"] = randn(B, W - 1, D)
        names = ("x", "weight", "bias")
    elif case["kind"] == "scan":
        N, G, R = case["states"], case["groups"], max(1, D // 16)
        proj = randn(T, B, R + 2 * G * N)                       # [low-rank dt | b | c] of one projection
        st["x"] = F.silu(randn(T, B, D, dtype=torch.float32)).to(half)
        st["dt"] = randn(T, B, D, scale=0.5)
        st["a"] = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32).repeat(D, 1) * torch.exp(0.1 * randn(D, N, dtype=torch.float32))
        st["b"], st["c"] = proj[..., R:R + G * N].unflatten(-1, (G, N)), proj[..., R + G * N:].unflatten(-1, (G, N))
        st["d"] = 1 + 0.1 * randn(D, dtype=torch.float32)
        step = torch.exp(rand(D) * math.log(100.0) + math.log(1e-3))
        st["dt_bias"] = step + torch.log(-torch.expm1(-step))   # softplus of it is the step
        if case["task"] == "step":
            st["s"] = randn(B, D, N, dtype=torch.float32, scale=0.3)
        names = ("x", "dt", "a", "b", "c", "d", "dt_bias")
    else:
        st["groups"] = case["groups"]
        st["x"], st["gate"] = randn(T, B, D, scale=2.0), randn(T, B, 2 * D)[..., D:]      # the second half of the input projection
        st["weight"], st["bias"] = (1 + randn(D, scale=0.1).float()).to(half), randn(D, scale=0.1)
        names = ("x", "weight", "bias", "gate")
    if train:
        for n in names:
            st[n] = st[n].detach().requires_grad_()
        st["leaves"] = [st[n] for n in names]
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _columns(t):
    """A mask [batch, tokens] beside activations [tokens, batch, channels]."""
    return t.t().unsqueeze(-1)


def _conv_plain(st):
    """As though padded tokens were not there; these are padded at the end, so that they only have to be left out."""
    x, w, bias = st["x"].detach().float(), st["weight"].detach().float(), st["bias"].detach().float()
    T, W = x.size(0), w.size(1)
    real = None if st["pad"] is None else _columns(~st["pad"])
    if real is not None:
        x = torch.where(real, x, 0.0)
    before = st["state"].float().transpose(0, 1) if st["task"] == "step" else x.new_zeros(W - 1, *x.shape[1:])
    ext = torch.cat([before, x])                                # [W - 1 + T, B, D]
    win = ext.unfold(0, W, 1)                                   # [T, B, D, W]
    pre = (win * w).sum(-1) + bias
    sig = torch.sigmoid(pre)
    y = pre * sig
    if real is not None:
        y = torch.where(real, y, 0.0)
    if st["task"] == "step":
        st["state"].copy_(ext[1:].transpose(0, 1))
        return y.to(st["x"].dtype), st["state"]
    if st["task"] == "prompt":
        last = torch.full((x.size(1),), T, device=x.device) if real is None else (~st["pad"]).sum(1)
        rows = last[:, None] + torch.arange(W - 1, device=x.device)             # of ext: the last W - 1 inputs of each sequence
        kept = ext[rows, torch.arange(x.size(1), device=x.device)[:, None]]     # [B, W - 1, D]
        return y.to(st["x"].dtype), kept.to(st["x"].dtype)
    g = st["g"].float()
    if real is not None:
        g = torch.where(real, g, 0.0)
    g = g * sig * (1 + pre * (1 - sig))
    gw, gb = (g.unsqueeze(-1) * win).sum((0, 1)), g.sum((0, 1))
    after = torch.cat([g, g.new_zeros(W - 1, *g.shape[1:])])
    gx = (after.unfold(0, W, 1) * w.flip(1)).sum(-1)
    if real is not None:
        gx = torch.where(real, gx, 0.0)
    return y.to(st["x"].dtype), gx.to(st["x"].dtype), gw.to(st["weight"].dtype), gb.to(st["bias"].dtype)


def _recurrence(delta, a, u, first):
    """Every s_t = exp(delta_t a) s_(t-1) + u_t: delta [T, B, D], a [D, N], u [T, B, D, N], first [B, D, N] -> [T, B, D, N].
    Runs of about sqrt(T) tokens are taken side by side, each from zero; then what each of them starts from is carried along."""
    T = u.size(0)
    L = max(1, math.isqrt(T))
    C = -(-T // L)
    fill = C * L - T
    if fill:
        delta, u = F.pad(delta, (0, 0, 0, 0, 0, fill)), F.pad(u, (0, 0, 0, 0, 0, 0, 0, fill))
    delta, u = delta.unflatten(0, (C, L)), u.unflatten(0, (C, L))
    s = torch.empty_like(u)
    s[:, 0] = u[:, 0]
    for l in range(1, L):
        s[:, l] = torch.exp(delta[:, l, ..., None] * a) * s[:, l - 1] + u[:, l]
    since = delta.cumsum(1)
    carry = torch.empty_like(s[:, 0])
    carry[0] = first
    for k in range(1, C):
        carry[k] = torch.exp(since[k - 1, -1, ..., None] * a) * carry[k - 1] + s[k - 1, -1]
    return (s + torch.exp(since[..., None] * a) * carry[:, None]).flatten(0, 1)[:T]


def _scan_plain(st):
    x, dt, b, c = (st[n].detach().float() for n in ("x", "dt", "b", "c"))
    a, d, bias = st["a"].detach(), st["d"].detach(), st["dt_bias"].detach()
    T, B, D = x.shape
    real = None if st["pad"] is None else _columns(~st["pad"])
    raw = dt + bias
    delta = F.softplus(raw, threshold=80.0)
    if real is not None:
        delta, x, b, c = torch.where(real, delta, 0.0), torch.where(real, x, 0.0), torch.where(real[..., None], b, 0.0), torch.where(real[..., None], c, 0.0)
    heads = D // b.size(2)
    bb, cc = b.repeat_interleave(heads, 2), c.repeat_interleave(heads, 2)       # [T, B, D, N]
    if st["task"] == "step":
        st["s"].copy_(torch.exp(delta[0, ..., None] * a) * st["s"] + (delta * x)[0, ..., None] * bb[0])
        return ((st["s"] * cc[0]).sum(-1) + d * x[0]).unsqueeze(0).to(st["x"].dtype), st["s"]
    zero = x.new_zeros(B, D, a.size(1))
    s = _recurrence(delta, a, (delta * x).unsqueeze(-1) * bb, zero)
    y = ((s * cc).sum(-1) + d * x).to(st["x"].dtype)
    if st["task"] == "prompt":
        return y, s[-1].clone()
    g = st["g"].float()
    if real is not None:
        g = torch.where(real, g, 0.0)
    gc = (s * g.unsqueeze(-1)).unflatten(2, (-1, heads)).sum(3)
    # the gradient of the state runs backwards: G_t = c_t g_t + exp(delta_(t+1) a) G_(t+1)
    after = torch.cat([delta[1:], delta.new_zeros(1, B, D)])
    G = _recurrence(after.flip(0), a, (cc * g.unsqueeze(-1)).flip(0), zero).flip(0)
    gu = (G * bb).sum(-1)                                                       # of delta x
    gb = (G * (delta * x).unsqueeze(-1)).unflatten(2, (-1, heads)).sum(3)
    del bb, cc
    before = torch.cat([zero[None], s[:-1]])
    del s
    G = G * torch.exp(delta[..., None] * a) * before                            # of delta a
    del before
    ga = (G * delta.unsqueeze(-1)).sum((0, 1))
    graw = ((G * a).sum(-1) + x * gu) * torch.sigmoid(raw)
    if real is not None:
        graw = torch.where(real, graw, 0.0)
    gx = delta * gu + d * g
    half = st["x"].dtype
    return y, gx.to(half), graw.to(half), ga, gb.to(half), gc.to(half), (x * g).sum((0, 1)), graw.sum((0, 1))


def _norm_plain(st):
    x, gate, w, bias = (st[n].detach().float() for n in ("x", "gate", "weight", "bias"))
    half, groups = st["x"].dtype, st["groups"]
    xg = x.unflatten(-1, (groups, -1))
    xc = xg - xg.mean(-1, keepdim=True)
    rstd = torch.rsqrt(xc.square().mean(-1, keepdim=True) + 1e-5)
    xn = xc * rstd
    n = xn.flatten(-2) * w + bias
    sig = torch.sigmoid(gate)
    y = n * gate * sig
    if st["task"] == "prompt":
        return y.to(half)
    g = st["g"].float()
    ggate = g * n * sig * (1 + gate * (1 - sig))
    gn = g * gate * sig
    gw, gb = (gn * xn.flatten(-2)).sum((0, 1)), gn.sum((0, 1))
    gxn = (gn * w).unflatten(-1, (groups, -1))
    gx = rstd * (gxn - gxn.mean(-1, keepdim=True) - xn * (gxn * xn).mean(-1, keepdim=True))
    return y.to(half), gx.flatten(-2).to(half), gw.to(half), gb.to(half), ggate.to(half)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _conv_own(st):
    from rfa_b200 import state_space as ss
    if st["task"] == "train":
        y = ss.causal_conv(x=st["x"], weight=st["weight"], bias=st["bias"], key_padding_mask=st["pad"])
        return (y, *torch.autograd.grad(y, st["leaves"], st["g"]))
    return ss.incremental_causal_conv(x=st["x"], weight=st["weight"], bias=st["bias"], key_padding_mask=st["pad"], state=st.get("state"))


def _scan_own(st):
    from rfa_b200 import state_space as ss
    args = dict(x=st["x"], dt=st["dt"], a=st["a"], b=st["b"], c=st["c"], d=st["d"], dt_bias=st["dt_bias"], key_padding_mask=st["pad"])
    if st["task"] == "train":
        y = ss.selective_scan(**args)
        return (y, *torch.autograd.grad(y, st["leaves"], st["g"]))
    return ss.incremental_selective_scan(**args, s=st.get("s"))


def _norm_own(st):
    from rfa_b200 import state_space as ss
    y = ss.group_norm(x=st["x"], num_groups=st["groups"], weight=st["weight"], bias=st["bias"], gate=st["gate"])
    return (y, *torch.autograd.grad(y, st["leaves"], st["g"])) if st["task"] == "train" else y


def run(state):
    kind = state["kind"]
    if own:
        return _conv_own(state) if kind == "conv" else _scan_own(state) if kind == "scan" else _norm_own(state)
    return _conv_plain(state) if kind == "conv" else _scan_plain(state) if kind == "scan" else _norm_plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    T, B, D, size = case["tokens"], case["batch"], case["channels"], 4 if case["dtype"] == "float32" else 2
    rows, train = T * B * D, case["task"] == "train"
    if case["kind"] == "conv":
        W = case["width"]
        kept = B * (W - 1) * D * size
        moved = {"step": 2 * rows * size + 2 * kept, "prompt": 2 * rows * size + kept, "train": 4 * rows * size}[case["task"]]
        return {"bytes": moved + (2 if train else 1) * D * (W + 1) * size, "flops": rows * (2 * W + 5) * (3 if train else 1)}
    if case["kind"] == "norm":
        moved = (6 if train else 3) * rows * size                # x, gate, y; and g, and the gradients of x and gate
        return {"bytes": moved + (4 if train else 2) * D * size, "flops": rows * (30 if train else 12)}
    N, G = case["states"], case["groups"]
    bc, state, weights = 2 * T * B * G * N * size, B * D * N * 4, D * (N + 2) * 4
    moved = {"step": 3 * rows * size + bc + 2 * state, "prompt": 3 * rows * size + bc + state,
             "train": 6 * rows * size + 2 * bc + weights}[case["task"]]          # x, dt, y; and g, and the gradients
    return {"bytes": moved + weights, "flops": rows * N * (24 if train else 7)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        return _norm_exact(st)
    if case["tokens"] * case["batch"] * case["channels"] * case.get("states", 1) > 2 ** 30:
        return None
    return _conv_exact(st) if case["kind"] == "conv" else _scan_exact(st)


def _double(st, *names):
    return [st[n].detach().double() for n in names]


def _conv_exact(st):
    """Token by token, with the last inputs of each sequence at hand."""
    x, w, bias = _double(st, "x", "weight", "bias")
    T, B, D = x.shape
    W = w.size(1)
    last = [torch.zeros(B, D, device=x.device, dtype=torch.float64) for _ in range(W)]
    if st["task"] == "step":
        last[1:] = list(st["state"].double().unbind(1))
    ys, wins, pres = [], [], []
    for t in range(T):
        new = last[1:] + [x[t]]
        pre = sum(w[:, j] * new[j] for j in range(W)) + bias
        y = pre / (1 + torch.exp(-pre))
        if st["pad"] is not None:
            gone = st["pad"][:, t, None]
            y = torch.where(gone, 0.0, y)
            new = [torch.where(gone, o, n) for o, n in zip(last, new)]
        last = new
        ys.append(y)
        wins.append(new)
        pres.append(pre)
    y = torch.stack(ys)
    if st["task"] != "train":
        return y, torch.stack(last[1:], 1)
    g = st["g"].double()
    gw, gb, gx = torch.zeros_like(w), torch.zeros_like(bias), torch.zeros_like(x)
    for t in range(T):
        e = 1 / (1 + torch.exp(-pres[t]))
        p = g[t] * (e + pres[t] * e * (1 - e))
        if st["pad"] is not None:
            p = torch.where(st["pad"][:, t, None], 0.0, p)
        gb += p.sum(0)
        for j in range(W):
            gw[:, j] += (p * wins[t][j]).sum(0)
            if t - (W - 1 - j) >= 0:
                gx[t - (W - 1 - j)] += p * w[:, j]
    return y, gx, gw, gb


def _scan_exact(st):
    """The recurrence token by token, and its gradient token by token from the end."""
    x, dt, a, b, c, d, bias = _double(st, "x", "dt", "a", "b", "c", "d", "dt_bias")
    T, B, D = x.shape
    G, N = b.shape[2:]
    s = st["s"].double() if st["task"] == "step" else torch.zeros(B, D, N, device=x.device, dtype=torch.float64)
    keep = st["task"] == "train"
    states, y = [s], torch.zeros_like(x)

    def wide(t):                                                 # [B, G, N] -> [B, D, N]
        return t[:, :, None].expand(B, G, D // G, N).reshape(B, D, N)

    def step_of(t):
        raw = dt[t] + bias
        return torch.logaddexp(raw, torch.zeros_like(raw))[..., None]

    for t in range(T):
        delta = step_of(t)
        new = torch.exp(delta * a) * s + delta * x[t][..., None] * wide(b[t])
        out = (new * wide(c[t])).sum(-1) + d * x[t]
        if st["pad"] is not None:
            gone = st["pad"][:, t, None]
            new, out = torch.where(gone[..., None], s, new), torch.where(gone, 0.0, out)
        s = new
        y[t] = out
        if keep:
            states.append(s)
    if not keep:
        return y, s
    g = st["g"].double()
    gx, gdt, ga, gb, gc, gd = (torch.zeros_like(t) for t in (x, dt, a, b, c, d))
    gs = torch.zeros_like(s)
    for t in reversed(range(T)):
        real = torch.ones(B, 1, device=x.device, dtype=torch.float64) if st["pad"] is None else (~st["pad"][:, t, None]).double()
        gt, delta = g[t] * real, step_of(t)
        here = gs + wide(c[t]) * gt[..., None]
        gc[t] = (states[t + 1] * gt[..., None]).unflatten(1, (G, -1)).sum(2)
        gu = here * real[..., None]
        gb[t] = (gu * delta * x[t][..., None]).unflatten(1, (G, -1)).sum(2)
        into = (gu * wide(b[t])).sum(-1)
        decay = torch.exp(delta * a)
        power = gu * decay * states[t]
        ga += (power * delta).sum(0)
        gdt[t] = ((power * a).sum(-1) + into * x[t]) * torch.sigmoid(dt[t] + bias)
        gx[t] = into * delta[..., 0] + d * gt
        gd += (gt * x[t]).sum(0)
        gs = torch.where(real[..., None] > 0, here * decay, gs)
    return y, gx, gdt, ga, gb, gc, gd, gdt.sum((0, 1))


def _norm_exact(st):
    """Gradients by the chain rule over each group's own mean and deviation."""
    x, gate, w, bias = _double(st, "x", "gate", "weight", "bias")
    shape, groups = x.shape, st["groups"]
    x = x.reshape(-1, groups, shape[-1] // groups)
    mean = x.mean(-1, keepdim=True)
    dev = torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    xn = (x - mean) / dev
    act = (gate / (1 + torch.exp(-gate))).reshape(x.shape)
    w, bias = w.reshape(groups, -1), bias.reshape(groups, -1)
    y = ((xn * w + bias) * act).reshape(shape)
    if st["task"] == "prompt":
        return y
    g = st["g"].double().reshape(x.shape)
    e = torch.sigmoid(gate).reshape(x.shape)
    ggate = g * (xn * w + bias) * (e + act * (1 - e))
    h = g * act
    gw, gb = (h * xn).sum(0).flatten(), h.sum(0).flatten()
    h = h * w
    m = x.size(-1)
    gdev = -(h * (x - mean)).sum(-1, keepdim=True) / dev ** 2
    gx = h / dev + gdev * (x - mean) / (m * dev)
    gx = gx - gx.mean(-1, keepdim=True)
    return y, gx.reshape(shape), gw, gb, ggate.reshape(shape)
