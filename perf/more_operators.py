"""What is timed of the two attentions of bounded memory that stand beside causal RFA: linear attention whose state decays, and
softmax attention over a sliding window with a few first tokens that stay visible.

``listed()`` names twelve cases, ``draw(rng)`` gives one more of the same ranges.  Each case is a dict of plain values with
a ``kind``:

  decay   S_t = exp(log_decay_t) S_(t-1) + k_t (x) v_t, out_t = scale q_t S_t per head, the decay one number for each head
          ("head") or one for each token and head ("token")
  window  softmax attention of token i over the tokens j <= i with i - j < window or j < sinks; the query heads share the
          key heads in equal groups

``task`` is "step" (one token, the kept state or cache updated in place), "prompt" (a run of tokens from nothing, without
gradients; the decay's last state returned) or "train" (the output and every gradient).

Activations are time-major ``[tokens, batch, heads, head width]`` as everywhere in this package, and q, k and v are views of
one projection's output.  Padded sequences have lengths uniform in [T/2, T].
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
        # interactive generation: one token of eight sequences; launches and latency
        dict(name="decay_step", kind="decay", task="step", batch=8, tokens=1, heads=16, key_dim=64, head_dim=64, decay="token", dtype="float16", padded=False),
        # batch generation: the states of 256 sequences stream from memory for every token
        dict(name="decay_step_batch", kind="decay", task="step", batch=256, tokens=1, heads=16, key_dim=128, head_dim=128, decay="token", dtype="bfloat16", padded=False),
        # prompt of a generation at the headline batch, a fixed decay for each head
        dict(name="decay_prompt", kind="decay", task="prompt", batch=8, tokens=2048, heads=16, key_dim=64, head_dim=64, decay="head", dtype="bfloat16", padded=False),
        # one long document: few rows, so the time axis itself has to be split
        dict(name="decay_long", kind="decay", task="prompt", batch=1, tokens=32768, heads=16, key_dim=128, head_dim=128, decay="token", dtype="bfloat16", padded=False),
        # training step at the headline batch, decays that are learned
        dict(name="decay_train", kind="decay", task="train", batch=8, tokens=2048, heads=16, key_dim=128, head_dim=128, decay="token", dtype="bfloat16", padded=False),
        # a small single-precision model on a ragged batch, sizes that are multiples of little
        dict(name="decay_ragged", kind="decay", task="train", batch=3, tokens=531, heads=4, key_dim=40, head_dim=52, decay="token", dtype="float32", padded=True),
        # interactive generation: one token of eight sequences; launches and latency
        dict(name="window_step", kind="window", task="step", batch=8, tokens=1, heads=16, kv_heads=16, head_dim=64, window=512, sinks=4, dtype="float16", padded=False),
        # batch generation: the caches of 256 sequences stream from memory for every token
        dict(name="window_step_batch", kind="window", task="step", batch=256, tokens=1, heads=32, kv_heads=8, head_dim=128, window=1024, sinks=4, dtype="bfloat16", padded=False),
        # prompt of a generation at the headline batch
        dict(name="window_prompt", kind="window", task="prompt", batch=8, tokens=2048, heads=16, kv_heads=4, head_dim=64, window=256, sinks=4, dtype="bfloat16", padded=False),
        # one long document
        dict(name="window_long", kind="window", task="prompt", batch=1, tokens=32768, heads=16, kv_heads=4, head_dim=128, window=1024, sinks=4, dtype="bfloat16", padded=False),
        # training step at the headline batch
        dict(name="window_train", kind="window", task="train", batch=8, tokens=2048, heads=16, kv_heads=16, head_dim=64, window=512, sinks=4, dtype="bfloat16", padded=False),
        # training step on a padded batch of sentences, sizes that are multiples of little
        dict(name="window_ragged", kind="window", task="train", batch=24, tokens=150, heads=6, kv_heads=2, head_dim=40, window=37, sinks=3, dtype="float16", padded=True),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    """Width of a head: the usual ones, other multiples of 8, and every sixth case any number."""
    return rng.choice([32, 64, 64, 96, 128, 128, 8 * rng.randint(1, 16), 8 * rng.randint(1, 16), rng.randint(3, 200)])


def draw(rng):
    kind, task = rng.choice(["decay", "window"]), rng.choice(["step", "prompt", "train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    tokens = 1 if task == "step" else _log(rng, 2, 8192)
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    case = dict(kind=kind, task=task, tokens=tokens, heads=heads, dtype=dtype, padded=task != "step" and rng.random() < 0.5)
    most = 256 if task == "step" else max(1, (2 ** 18 if dtype != "float32" else 2 ** 16) // (tokens * heads))
    case["batch"] = _log(rng, 1, min(256, most))
    if kind == "decay":
        return dict(case, key_dim=_width(rng), head_dim=_width(rng), decay=rng.choice(["head", "token"]))
    return dict(case, kv_heads=rng.choice([n for n in range(1, heads + 1) if heads % n == 0]), head_dim=_width(rng),
                window=_log(rng, 1, 1024), sinks=rng.choice([0, 1, 4, 4, rng.randint(0, 130)]))


# ------------------------------------------------------------------------------------------------ inputs
def _padding(gen, batch, tokens):
    """[batch, tokens] with True at the padded positions, lengths uniform in [tokens / 2, tokens]."""
    lengths = torch.randint((tokens + 1) // 2, tokens + 1, (batch, 1), generator=gen, device=DEV)
    return torch.arange(tokens, device=DEV)[None] >= lengths


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    T, B, H, half, task = case["tokens"], case["batch"], case["heads"], TYPES[case["dtype"]], case["task"]
    D = case["head_dim"]

    def randn(*shape, scale=1.0, dtype=half):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    st = dict(kind=case["kind"], task=task, pad=_padding(gen, B, T) if case["padded"] else None)
    if case["kind"] == "decay":
        K = case["key_dim"]
        proj = randn(T, B, H * (2 * K + D))                     # [q | k | v] of one projection
        q, k, v = proj.split([H * K, H * K, H * D], dim=-1)
        st["q"], st["k"], st["v"] = q.unflatten(-1, (H, K)), k.unflatten(-1, (H, K)), v.unflatten(-1, (H, D))
        if case["decay"] == "head":                             # horizons of 32 tokens and more, each head's longer than the one before
            st["log_decay"] = torch.log1p(-torch.exp2(-5.0 - 8.0 * torch.arange(H, device=DEV) / H))
        else:                                                   # a sixteenth of log sigmoid, as gates are initialised
            st["log_decay"] = (F.logsigmoid(randn(T, B, H, dtype=torch.float32)) / 16).to(half)
        if task == "step":
            st["s"] = randn(B, H, K, D, dtype=torch.float32, scale=3.0)
        names = ("q", "k", "v", "log_decay") if case["decay"] == "token" else ("q", "k", "v")
    else:
        G, W, sinks = case["kv_heads"], case["window"], case["sinks"]
        proj = randn(T, B, (H + 2 * G) * D)
        q, k, v = proj.split([H * D, G * D, G * D], dim=-1)
        st["q"], st["k"], st["v"] = q.unflatten(-1, (H, D)), k.unflatten(-1, (G, D)), v.unflatten(-1, (G, D))
        st["window"], st["sinks"] = W, sinks
        if task == "step":                                      # sequences of every age, some with a cache that is not full yet
            st["prev_k"], st["prev_v"] = randn(B, G, sinks + W, D), randn(B, G, sinks + W, D)
            st["prev_len"] = torch.randint(0, 4 * (sinks + W), (B,), generator=gen, device=DEV)
        names = ("q", "k", "v")
    if task == "train":
        st["g"] = randn(T, B, H, D)
        for n in names:
            st[n] = st[n].detach().requires_grad_()
        st["leaves"] = [st[n] for n in names]
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _decay_tokens(st):
    """The log decays [T, B, H] in 64 bits: sums of many are subtracted from each other."""
    g = st["log_decay"].double()
    return g if g.dim() == 3 else g.expand(*st["q"].shape[:2], -1)


def _decay_plain(st):
    """In chunks: the products of a chunk's tokens with each other, and with the state in front of it, which is a sum over the chunks
    before.  Padded tokens, which are at the end, add nothing and decay nothing."""
    q, k, v, g = st["q"].float(), st["k"].float(), st["v"].float(), _decay_tokens(st)
    T, B, H, K = q.shape
    scale = K ** -0.5
    if st["task"] == "step":
        st["s"].mul_(torch.exp(g[0]).float()[..., None, None]).add_(k[0, ..., None] * v[0, ..., None, :])
        return (scale * (q[0, ..., None] * st["s"]).sum(-2))[None].to(st["q"].dtype), st["s"]
    if st["pad"] is not None:
        real = ~st["pad"].t()[..., None]
        g, k, v = torch.where(real, g, 0.0), torch.where(real[..., None], k, 0.0), torch.where(real[..., None], v, 0.0)
    C = min(128, T)
    fill = -T % C

    def chunks(x):                                              # [T, B, H, ...] -> [B, H, chunks, C, ...]
        x = torch.cat([x, x.new_zeros(fill, *x.shape[1:])]) if fill else x
        return x.unflatten(0, (-1, C)).movedim((2, 3), (0, 1))

    q, k, v, g = chunks(q), chunks(k), chunks(v), chunks(g).cumsum(-1)
    total = g[..., -1]
    lower = torch.ones(C, C, dtype=torch.bool, device=DEV).tril()
    w = torch.exp((g[..., :, None] - g[..., None, :]).masked_fill(~lower, -math.inf).float())
    out = (w * (q @ k.transpose(-1, -2))) @ v
    u = (k * torch.exp((total[..., None] - g).float())[..., None]).transpose(-1, -2) @ v            # [B, H, chunks, K, D]: what each chunk adds
    ends = total.cumsum(-1)
    n = ends.size(-1)
    across = torch.exp((ends[..., :, None] - ends[..., None, :]).masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), -math.inf).float())
    s = (across @ u.flatten(-2)).unflatten(-1, u.shape[-2:])    # the state behind each chunk
    front = torch.cat([torch.zeros_like(s[:, :, :1]), s[:, :, :-1]], 2)
    out = scale * (out + torch.exp(g.float())[..., None] * (q @ front))
    out = out.movedim((0, 1), (2, 3)).flatten(0, 1)[:T]
    if st["pad"] is not None:
        out = torch.where(real[..., None], out, 0.0)
    return out.to(st["q"].dtype), s[:, :, -1].contiguous()


def _window_step_plain(st):
    q, k, v, pk, pv, n = (st[x] for x in ("q", "k", "v", "prev_k", "prev_v", "prev_len"))
    sinks, W, D = st["sinks"], st["window"], q.size(-1)
    rows, slot = torch.arange(n.size(0), device=DEV), torch.where(n < sinks, n, sinks + (n - sinks) % W)
    pk[rows, :, slot], pv[rows, :, slot] = k[0], v[0]
    n += 1
    scores = D ** -0.5 * (q[0].float().unflatten(1, (k.size(2), -1)) @ pk.float().transpose(-1, -2))            # [B, kv heads, group, slots]
    scores = scores.masked_fill((torch.arange(sinks + W, device=DEV) >= n[:, None])[:, None, None], -math.inf)
    out = torch.softmax(scores, -1) @ pv.float()
    return out.flatten(1, 2)[None].to(q.dtype), pk, pv, n


def _window_plain(st):
    """In blocks of queries of a window's length, each beside its own and the last block's keys, and the first tokens in front."""
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    T, B, H, D = q.shape
    G, W, sinks, pad = k.size(2), st["window"], min(st["sinks"], T), st["pad"]
    if pad is not None:
        real = ~pad.t()[..., None, None]
        k, v = torch.where(real, k, 0.0), torch.where(real, v, 0.0)
    C = min(T, max(W, 64))
    fill = -T % C

    def blocks(x, before):                                      # [T, B, heads, D] -> [B, heads, blocks, C (2 C with the block before), D]
        x = torch.cat([x.new_zeros(before, *x.shape[1:]), x, x.new_zeros(fill, *x.shape[1:])])
        return x.unfold(0, C + before, C).permute(1, 2, 0, 4, 3)

    def beside(x):
        x2 = blocks(x, C)
        first = x[:sinks].permute(1, 2, 0, 3)[:, :, None].expand(-1, -1, x2.size(2), -1, -1)
        return torch.cat([first, x2], 3)

    qb, kb, vb = blocks(q, 0).unflatten(1, (G, -1)), beside(k)[:, :, None], beside(v)[:, :, None]
    at = torch.arange(qb.size(3), device=DEV)[:, None, None] * C
    i, j = at + torch.arange(C, device=DEV)[:, None], at - C + torch.arange(2 * C, device=DEV)
    near = (j >= 0) & (j <= i) & (i - j < W) & (j >= sinks)     # the first tokens are seen among the ones in front
    seen = torch.cat([torch.arange(sinks, device=DEV) <= i, near], -1)          # [blocks, C, sinks + 2 C]
    if pad is not None:
        number = torch.cat([torch.arange(sinks, device=DEV).expand(len(at), 1, -1), j], -1)
        lengths = (~pad).sum(1)
        seen = seen & (number < lengths[:, None, None, None])
        seen = seen[:, None, None]
    scores = (D ** -0.5 * (qb @ kb.transpose(-1, -2))).masked_fill(~seen, -math.inf)
    top = scores.detach().amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    out = (e @ vb) / e.sum(-1, keepdim=True).clamp_min(1e-30)   # [B, kv heads, group, blocks, C, D]
    out = out.flatten(1, 2).flatten(2, 3)[:, :, :T].permute(2, 0, 1, 3)
    if pad is not None:
        out = torch.where(real, out, 0.0)
    return out.to(st["q"].dtype)


def _plain(st):
    if st["kind"] == "decay":
        with torch.set_grad_enabled(st["task"] == "train"):
            out, s = _decay_plain(st)
        if st["task"] != "train":
            return out, s
    elif st["task"] == "step":
        return _window_step_plain(st)
    else:
        with torch.set_grad_enabled(st["task"] == "train"):
            out = _window_plain(st)
        if st["task"] != "train":
            return out
    return (out.detach(), *torch.autograd.grad(out, st["leaves"], st["g"]))


# ------------------------------------------------------------------------------------------------ the framework's calls
def _decay_own(st):
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    args = dict(q=st["q"], k=st["k"], v=st["v"], log_decay=st["log_decay"], key_padding_mask=st["pad"])
    if st["task"] == "train":
        out = decay_attention(**args)
        return (out, *torch.autograd.grad(out, st["leaves"], st["g"]))
    return incremental_decay_attention(**args, s=st.get("s"))


def _window_own(st):
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    args = dict(q=st["q"], k=st["k"], v=st["v"], window=st["window"], sinks=st["sinks"])
    if st["task"] == "step":
        return incremental_window_attention(**args, prev_k=st["prev_k"], prev_v=st["prev_v"], prev_len=st["prev_len"])
    out = window_attention(**args, key_padding_mask=st["pad"])
    return (out, *torch.autograd.grad(out, st["leaves"], st["g"])) if st["task"] == "train" else out


def run(state):
    if own:
        return _decay_own(state) if state["kind"] == "decay" else _window_own(state)
    return _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    T, B, H, D, size = case["tokens"], case["batch"], case["heads"], case["head_dim"], 4 if case["dtype"] == "float32" else 2
    rows, train = T * B * H, case["task"] == "train"
    if case["kind"] == "decay":
        K, state = case["key_dim"], B * H * case["key_dim"] * D * 4
        gates = rows * size if case["decay"] == "token" else H * 4
        once = rows * 2 * (K + D) * size + gates                                  # q, k, v, the decays and the output
        moved = {"step": once + 2 * state, "prompt": once + state, "train": once + rows * (2 * K + 2 * D) * size + (gates if case["decay"] == "token" else 0)}[case["task"]]
        return {"bytes": moved, "flops": rows * K * D * (16 if train else 4)}      # the update and the product; five more of each kind behind them
    G, W, sinks = case["kv_heads"], case["window"], case["sinks"]
    if case["task"] == "step":
        cache = 2 * B * G * (sinks + W) * D * size
        return {"bytes": cache + 2 * rows * D * size + 4 * B * G * D * size, "flops": 4 * rows * (sinks + W) * D}
    length = 0.75 * T if case["padded"] else T
    full = min(length, W)
    pairs = full * (full + 1) / 2 + max(0, length - W) * W + sum(min(sinks, i - W + 1) for i in range(W, int(length)))
    kv = 2 * T * B * G * D * size
    return {"bytes": rows * 2 * D * size * (2 if train else 1) + kv * (2 if train else 1), "flops": int(pairs) * B * H * D * (14 if train else 4)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["task"] == "step":
        return _decay_step_exact(st) if case["kind"] == "decay" else _window_step_exact(st)
    if case["tokens"] ** 2 * case["batch"] * case["heads"] > 2 ** 35:
        return None
    return _decay_exact(st) if case["kind"] == "decay" else _window_exact(st)


def _decay_step_exact(st):
    q, k, v = (st[n][0].double() for n in ("q", "k", "v"))
    g = st["log_decay"].double()
    g = g[0] if g.dim() == 3 else g.expand(q.shape[:2])
    s = torch.exp(g)[..., None, None] * st["s"].double() + torch.einsum("bhk,bhd->bhkd", k, v)
    return torch.einsum("bhk,bhkd->bhd", q, s)[None] / math.sqrt(q.size(-1)), s


def _decay_exact(st):
    """Sequence by sequence and head by head, every pair of tokens by itself, rows of queries at a time."""
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    T, B, H, K = q.shape
    train = st["task"] == "train"
    log = st["log_decay"].detach().double()
    log = log.expand(T, B, H) if log.dim() == 1 else log
    out, s = torch.zeros(T, B, H, v.size(-1), device=DEV, dtype=torch.float64), torch.zeros(B, H, K, v.size(-1), device=DEV, dtype=torch.float64)
    gq, gk, gv, gg = (torch.zeros_like(x) for x in (q, k, v, log))
    counts = [T] * B if st["pad"] is None else (~st["pad"]).sum(1).tolist()
    for b, n in enumerate(counts):
        for h in range(H):
            Q, K_, V, L = q[:n, b, h], k[:n, b, h], v[:n, b, h], log[:n, b, h].cumsum(0)
            s[b, h] = (K_ * torch.exp(L[-1] - L)[:, None]).t() @ V
            reach = torch.zeros(n, device=DEV, dtype=torch.float64)             # of a row less what columns give
            for r in range(0, n, 2048):
                i = slice(r, min(n, r + 2048))
                upto = i.stop
                ahead = torch.arange(upto, device=DEV) > torch.arange(r, upto, device=DEV)[:, None]
                w = torch.exp((L[i, None] - L[:upto]).masked_fill(ahead, -math.inf)) / math.sqrt(K)
                p = w * (Q[i] @ K_[:upto].t())
                out[i, b, h] = p @ V[:upto]
                if train:
                    g = st["g"][i, b, h].double()
                    gp = g @ V[:upto].t()
                    gq[i, b, h] = (gp * w) @ K_[:upto]
                    gk[:upto, b, h] += (gp * w).t() @ Q[i]
                    gv[:upto, b, h] += p.t() @ g
                    m = p * gp
                    reach[i] += m.sum(1)
                    reach[:upto] -= m.sum(0)
            if train:
                gg[:n, b, h] = reach.flip(0).cumsum(0).flip(0)
    if not train:
        return out, s
    return (out, gq, gk, gv, gg) if len(st["leaves"]) == 4 else (out, gq, gk, gv)


def _window_step_exact(st):
    q, k, v = (st[n][0] for n in ("q", "k", "v"))
    pk, pv, n = st["prev_k"].clone(), st["prev_v"].clone(), st["prev_len"]
    B, H, D = q.shape
    group = H // k.size(1)
    out = torch.zeros(1, B, H, D, device=DEV, dtype=torch.float64)
    for b, age in enumerate(n.tolist()):
        slot = age if age < st["sinks"] else st["sinks"] + (age - st["sinks"]) % st["window"]
        pk[b, :, slot], pv[b, :, slot] = k[b], v[b]
        have = min(age + 1, pk.size(2))
        K_, V = pk[b, :, :have].double(), pv[b, :, :have].double()
        logits = torch.einsum("gud,gsd->gus", q[b].double().reshape(-1, group, D), K_) / math.sqrt(D)
        p = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
        out[0, b] = torch.einsum("gus,gsd->gud", p, V).reshape(H, D)
    return out, pk, pv, n + 1


def _window_exact(st):
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    T, B, H, D = q.shape
    group, train = H // k.size(2), st["task"] == "train"
    out, gq, gk, gv = (torch.zeros_like(x) for x in (q, q, k, v))
    counts = [T] * B if st["pad"] is None else (~st["pad"]).sum(1).tolist()
    for b, n in enumerate(counts):
        for r in range(0, n, 2048):
            i = slice(r, min(n, r + 2048))
            far = torch.arange(r, i.stop, device=DEV)[:, None] - torch.arange(i.stop, device=DEV)
            hidden = (far < 0) | ((far >= st["window"]) & (torch.arange(i.stop, device=DEV) >= st["sinks"]))
            for h in range(H):
                Q, K_, V = q[i, b, h], k[:i.stop, b, h // group], v[:i.stop, b, h // group]
                logits = (Q @ K_.t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
                p = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
                out[i, b, h] = p @ V
                if train:
                    g = st["g"][i, b, h].double()
                    gp = g @ V.t()
                    gl = p * (gp - (p * gp).sum(1, keepdim=True)) / math.sqrt(D)
                    gq[i, b, h] = gl @ K_
                    gk[:i.stop, b, h // group] += gl.t() @ Q
                    gv[:i.stop, b, h // group] += p.t() @ g
    return (out, gq, gk, gv) if train else out
