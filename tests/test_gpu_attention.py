"""Decaying linear attention and sliding-window attention against dense forms in 64 bits.

Tolerances, before the first run.  A half type's u = eps / 2 bounds one rounding.  A result passes through three of them that do not depend
on each other (the weights or the state as operands, the softmax's or decay's factor, the result), each u / sqrt(3) of its norm in the
mean: u together, 3 u allowed.  Gradients through a softmax take the difference of g . v and delta, each with one rounding more: 4 u.
In fp32 a sum of n terms is off by about sqrt(n) u of its norm, n up to 1000 here: 32 u; the decay's gradient is a difference of sums over all
tokens: 128 u, and of the terms' norm as well as the result's, because g_t = sum over i >= t of (q_i . gq_i - k_i . gk_i), each product with its own
roundings, may cancel to nothing (with one token, or for the first one, it does).  The same holds for a softmax's gradients: gq_i = scale sum_j p_ij (g_i . v_j - delta_i) k_j, both
terms rounded, and nothing is left of them where one key is seen; the k are of size 1, so the terms are of size scale delta_i.  A single element may be 8 times as far as the norm's mean allows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, dtype, roundings=3.0, name="", terms=None):
    assert got.shape == want.shape, name
    if not want.numel():
        return
    got, tol = got.double(), unit(dtype) * (roundings if dtype != torch.float32 else 32 / 3 * roundings)
    assert torch.isfinite(got).all(), name
    err, norm = got - want, want.norm() if terms is None else torch.hypot(want.norm(), terms.norm() * math.sqrt(want.numel() / terms.numel()))
    rms = norm / math.sqrt(want.numel())
    assert err.norm() <= tol * norm + 1e-30, (name, (err.norm() / norm).item(), tol)
    assert (err.abs() <= 8 * tol * torch.maximum(want.abs(), rms) + 1e-30).all(), (name, (err.abs() / rms).max().item(), 8 * tol)


def places(mask, T, B):
    """[B, T] numbers of the real tokens, and which are real."""
    real = torch.ones(B, T, dtype=torch.bool, device="cuda") if mask is None else ~mask.bool()
    return real.cumsum(1) - 1, real


# ------------------------------------------------------------------------------------------------ references
def decay_dense(q, k, v, g, s=None, mask=None, scale=None):
    """-> out, last state, differentiable in 64 bits."""
    T, B, H, K = q.shape
    scale = K ** -0.5 if scale is None else scale
    _, real = places(mask, T, B)
    on = real.t()[..., None]
    g = g.expand(T, B, H) if g.dim() == 1 else g
    g = torch.where(on, g, 0.0)
    q, k, v = (torch.where(on[..., None], x, 0.0) for x in (q, k, v))
    L = g.cumsum(0)
    ahead = torch.arange(T, device="cuda")[:, None] < torch.arange(T, device="cuda")
    w = torch.exp((L[:, None] - L[None]).masked_fill(ahead[..., None, None], -math.inf))            # [T, T, B, H]
    out = torch.einsum("tsbh,tbhk,sbhk,sbhd->tbhd", w, q, k, v) if T * T * B * H * K < 2 ** 24 else \
        torch.einsum("tsbh,sbhd->tbhd", w * torch.einsum("tbhk,sbhk->tsbh", q, k), v)
    last = torch.einsum("sbh,sbhk,sbhd->bhkd", torch.exp(L[-1] - L), k, v) if T else torch.zeros(B, H, K, v.size(-1), device="cuda", dtype=torch.float64)
    if s is not None:
        out = out + torch.exp(L)[..., None] * torch.einsum("tbhk,bhkd->tbhd", q, s)
        last = last + torch.exp(L[-1])[..., None, None] * s
    return scale * out, last


def window_dense(q, k, v, window, sinks, mask=None, scale=None):
    T, B, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    n, real = places(mask, T, B)
    far = n[:, :, None] - n[:, None, :]
    at = torch.arange(T, device="cuda")
    seen = real[:, :, None] & real[:, None, :] & (at[:, None] >= at) & ((far < window) | (n[:, None, :] < sinks))
    k, v = (torch.where(real.t()[..., None, None], x, 0.0).repeat_interleave(H // k.size(2), 2) for x in (k, v))
    q = torch.where(real.t()[..., None, None], q, 0.0)
    s = (scale * torch.einsum("tbhd,sbhd->bhts", q, k)).masked_fill(~seen[:, None], -math.inf)
    p = torch.where(seen[:, None], torch.exp(s - s.detach().amax(-1, keepdim=True).clamp_min(-1e300)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return torch.einsum("bhts,sbhd->tbhd", p, v)


def grads(f, leaves, g):
    leaves = [x.detach().double().requires_grad_() for x in leaves]
    out = f(*leaves)
    out = out if isinstance(out, tuple) else (out,)
    return [o.detach() for o in out], torch.autograd.grad(out[:len(g)], leaves, [x.double() for x in g])


def some_mask(kind, B, T):
    if kind is None:
        return None
    m = torch.rand(B, T, device="cuda") < 0.3 if kind == "any" else torch.arange(T, device="cuda")[None] >= torch.randint((T + 1) // 2, T + 1, (B, 1), device="cuda")
    if kind == "left":
        m = m.flip(1)
    if kind == "gap":           # stretches without a token, longer than a tile
        m = torch.zeros(B, T, dtype=torch.bool, device="cuda")
        m[:, T // 5:T // 5 + T // 2] = True
        m[-1, :T // 8] = m[-1, -3:] = True
    if kind == "any" and B > 1:
        m[0] = True             # a row with nothing in it
    return m


def make(T, B, heads, widths, dtype, view=True):
    """Activations as views of one projection's output, or by themselves."""
    n = [h * w for h, w in zip(heads, widths)]
    if view:
        return [x.unflatten(-1, (h, w)) for x, h, w in zip(torch.randn(T, B, sum(n), device="cuda").to(dtype).split(n, -1), heads, widths)]
    return [torch.randn(T, B, h, w, device="cuda").to(dtype) for h, w in zip(heads, widths)]


# ------------------------------------------------------------------------------------------------ decay
DECAY = [
    # T, B, H, K, D, decay, mask, dtype
    (1, 1, 1, 1, 1, "token", None, "fp32"),
    (2, 3, 2, 3, 5, "token", "any", "fp32"),
    (31, 2, 3, 16, 40, "head", "right", "fp32"),
    (33, 2, 2, 40, 16, "token", "left", "fp32"),
    (200, 1, 2, 200, 72, "token", "any", "fp32"),
    (1000, 1, 2, 24, 33, "token", None, "fp32"),
    (65, 2, 2, 64, 64, "token", None, "fp16"),
    (127, 2, 2, 64, 64, "head", "any", "bf16"),
    (128, 2, 3, 128, 128, "token", None, "fp16"),
    (129, 2, 2, 128, 64, "token", "right", "fp16"),
    (257, 3, 2, 64, 128, "head", "left", "fp16"),
    (300, 2, 2, 128, 128, "token", "any", "bf16"),
    (700, 1, 2, 72, 104, "token", "any", "fp16"),
    (385, 2, 2, 8, 8, "token", None, "fp16"),
    (1500, 1, 3, 128, 128, "token", None, "fp16"),
    (1000, 1, 2, 64, 64, "head", None, "bf16"),
    (140, 1, 2, 37, 90, "token", "any", "fp16"),
    (130, 1, 2, 256, 256, "token", None, "bf16"),
    (640, 40, 4, 64, 64, "token", "right", "bf16"),
    (1, 3, 2, 64, 64, "token", "any", "fp16"),
    (3, 200, 2, 128, 64, "head", "any", "fp16"),
    (2100, 2, 1, 128, 128, "token", "any", "fp16"),
    (5000, 1, 1, 64, 128, "token", None, "bf16"),
    (64, 2, 2, 33, 127, "token", "any", "fp16"),
    (63, 2, 2, 33, 127, "token", "any", "fp16"),
    (500, 1, 2, 100, 5, "head", None, "bf16"),
    (300, 2, 3, 1, 64, "token", "right", "fp16"),
]


def decay_terms(q, gq, g):
    terms = (q.double().nan_to_num() * gq).sum(-1)
    return terms if g.dim() == 3 else terms.square().sum((0, 1)).sqrt()


def decay_inputs(T, B, H, K, D, decay, mask, dtype, view=True):
    torch.manual_seed(T * 7 + K)
    dt = TYPES[dtype]
    q, k, v = make(T, B, (H, H, H), (K, K, D), dt, view)
    g = -torch.rand(H, device="cuda") * 0.2 if decay == "head" else (torch.nn.functional.logsigmoid(torch.randn(T, B, H, device="cuda")) / 4).to(dt)
    return q, k, v, g, some_mask(mask, B, T), dt


@pytest.mark.parametrize("case", DECAY, ids=str)
def test_decay_forward_and_gradients(case):
    from rfa_b200.decay_attention import decay_attention
    q, k, v, g, mask, dt = decay_inputs(*case)
    go = torch.randn_like(v)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, g)]
    out = decay_attention(q=leaves[0], k=leaves[1], v=leaves[2], log_decay=leaves[3], key_padding_mask=mask)
    got = torch.autograd.grad(out, leaves, go)
    (want, _), gw = grads(lambda *a: decay_dense(*a, mask=mask), (q, k, v, g), [go])
    near(out, want, dt, name="out")
    for n, a, b in zip("qkv", got, gw):
        near(a, b, dt, name=n)
    near(got[3], gw[3], dt, 12.0, name="decay", terms=decay_terms(q, gw[0], g))
    if mask is not None:
        gone = mask.t().bool()
        for x in (out, *got[:3]):
            assert (x[gone] == 0).all()
    with torch.no_grad():
        assert torch.equal(out, decay_attention(q=q, k=k, v=v, log_decay=g, key_padding_mask=mask))


@pytest.mark.parametrize("case", DECAY[1:], ids=str)
def test_decay_state_in_and_out(case):
    from rfa_b200.decay_attention import incremental_decay_attention
    q, k, v, g, mask, dt = decay_inputs(*case, view=False)
    s = torch.randn(q.size(1), q.size(2), q.size(3), v.size(3), device="cuda")
    want, last = decay_dense(*(x.double() for x in (q, k, v, g, s)), mask=mask)
    mine = s.clone()
    out, s1 = incremental_decay_attention(q=q, k=k, v=v, log_decay=g, s=mine, key_padding_mask=mask)
    assert s1 is mine
    near(out, want, dt, name="out")
    near(s1, last, torch.float32, 8.0, name="state")      # bf16's operands in two parts of 8 bits are off by 2^-17 each, 2^-18 / sqrt(3) in the mean: 37 u
    leaves = [x.detach().requires_grad_() for x in (q, k, v, g, s)]
    out2, s2 = incremental_decay_attention(q=leaves[0], k=leaves[1], v=leaves[2], log_decay=leaves[3], s=leaves[4], key_padding_mask=mask)
    assert s2 is not leaves[4] and torch.equal(leaves[4], s)
    go, gs = torch.randn_like(v), torch.randn_like(s)
    got = torch.autograd.grad((out2, s2), leaves, (go, gs))
    _, gw = grads(lambda *a: decay_dense(*a, mask=mask), (q, k, v, g, s), [go, gs])
    for n, a, b in zip(("q", "k", "v"), got, gw):
        near(a, b, dt, name=n)
    near(got[3], gw[3], dt, 12.0, name="decay", terms=decay_terms(q, gw[0], g))
    near(got[4], gw[4], torch.float32, 8.0, name="s")


@pytest.mark.parametrize("dtype,K,D", [("fp32", 40, 52), ("fp16", 64, 64), ("bf16", 128, 128), ("fp16", 33, 7), ("bf16", 256, 200)])
def test_decay_token_by_token(dtype, K, D):
    """A prompt, then tokens one by one, is the whole run."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    q, k, v, g, mask, dt = decay_inputs(40, 3, 2, K, D, "token", "any", dtype)
    want, last = decay_dense(*(x.double() for x in (q, k, v, g)), mask=mask)
    s, outs = None, []
    for a, b in [(0, 20)] + [(i, i + 1) for i in range(20, 40)]:
        o, s = incremental_decay_attention(q=q[a:b], k=k[a:b], v=v[a:b], log_decay=g[a:b], s=s, key_padding_mask=mask[:, a:b])
        outs.append(o)
    near(torch.cat(outs), want, dt)
    near(s, last, torch.float32, 8.0)
    o, s = incremental_decay_attention(q=q[:1], k=k[:1], v=v[:1], log_decay=g[:1], key_padding_mask=mask[:, :1])
    near(o, want[:1], dt)


def test_decay_resets_growth_and_masked_rubbish():
    """-inf forgets; long decays stay exact beside it; padded places may hold anything."""
    from rfa_b200.decay_attention import decay_attention
    for dt, K in ((torch.float32, 24), (torch.float16, 64), (torch.bfloat16, 128)):
        torch.manual_seed(3)
        q, k, v = make(300, 2, (2, 2, 2), (K, K, K), dt, False)
        g = -0.02 * torch.rand(300, 2, 2, device="cuda")
        for t in (0, 40, 41, 42, 127, 128, 200, 256):
            g[t] = -math.inf
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = decay_attention(q=leaves[0], k=leaves[1], v=leaves[2], log_decay=g)
        go = torch.randn_like(out)
        (want, _), gw = grads(lambda a, b, c: decay_dense(a, b, c, g.double().clamp_min(-1e4)), (q, k, v), [go])
        near(out, want, dt)
        for a, b in zip(torch.autograd.grad(out, leaves, go), gw):
            near(a, b, dt)
        mask = torch.zeros(2, 300, dtype=torch.bool, device="cuda")
        mask[0, 10:30] = mask[1, 100:260] = mask[1, 299] = True
        clean = decay_attention(q=q, k=k, v=v, log_decay=g, key_padding_mask=mask)
        for x in (q, k, v):
            x[mask.t()] = math.nan
        g[mask.t()] = math.nan
        q2, k2, v2 = (x.detach().requires_grad_() for x in (q, k, v))
        dirty = decay_attention(q=q2, k=k2, v=v2, log_decay=g, key_padding_mask=mask)
        assert torch.equal(clean, dirty)
        go[mask.t()] = math.inf
        for x in torch.autograd.grad(dirty, (q2, k2, v2), go):
            assert torch.isfinite(x).all() and (x[mask.t()] == 0).all()


def test_decay_strides_streams_and_sizes_of_zero():
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    torch.manual_seed(5)
    base = torch.randn(2, 3, 140, 200, device="cuda").half()           # [B, H, T, width]: another order, and rows off 16 bytes
    for off in (0, 1, 3, 8):
        q, k, v = (base[..., off + i * 64:off + i * 64 + 64].permute(2, 0, 1, 3) for i in range(3))
        g = -0.1 * torch.rand(3, 2, 140, device="cuda").permute(2, 1, 0)
        want, _ = decay_dense(*(x.double() for x in (q, k, v, g)))
        near(decay_attention(q=q, k=k, v=v, log_decay=g), want, torch.float16)
    near(decay_attention(q=q, k=k, v=v, log_decay=g[:1].expand(140, 2, 3), scale=0.5), decay_dense(*(x.double() for x in (q, k, v, g[:1].expand(140, 2, 3))), scale=0.5)[0],
         torch.float16)
    shared = k[:, :, :1].expand(-1, -1, 3, -1)                         # one head's keys for all: a stride of zero
    near(decay_attention(q=q, k=shared, v=v, log_decay=g), decay_dense(*(x.double() for x in (q, shared, v, g)))[0], torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = decay_attention(q=q, k=k, v=v, log_decay=g)
    torch.cuda.current_stream().wait_stream(side)
    near(y, want, torch.float16)
    for T, B, H in ((0, 2, 3), (5, 0, 3), (5, 2, 0)):
        q = torch.zeros(T, B, H, 16, device="cuda", dtype=torch.half, requires_grad=True)
        g = torch.zeros(T, B, H, device="cuda", requires_grad=True)
        out, s = incremental_decay_attention(q=q, k=q, v=q, log_decay=g)
        assert out.shape == q.shape and s.shape == (B, H, 16, 16)
        out.sum().backward()
        assert q.grad.shape == q.shape and g.grad.shape == g.shape


# ------------------------------------------------------------------------------------------------ window
WINDOW = [
    # T, B, H, G, D, window, sinks, mask, dtype
    (1, 1, 1, 1, 1, 1, 0, None, "fp32"),
    (5, 2, 2, 1, 3, 2, 1, "any", "fp32"),
    (33, 2, 4, 2, 17, 7, 0, "right", "fp32"),
    (100, 1, 3, 3, 40, 33, 4, "left", "fp32"),
    (200, 2, 2, 1, 130, 64, 70, "any", "fp32"),
    (70, 1, 1, 1, 256, 20, 2, None, "fp32"),
    (64, 2, 2, 2, 64, 1, 0, None, "fp16"),
    (127, 2, 4, 1, 64, 500, 0, "any", "bf16"),
    (128, 2, 4, 2, 128, 128, 4, None, "fp16"),
    (129, 2, 2, 2, 64, 64, 0, "left", "fp16"),
    (300, 2, 6, 2, 40, 37, 3, "any", "fp16"),
    (513, 1, 4, 4, 128, 200, 130, None, "fp16"),
    (700, 1, 2, 1, 72, 256, 1, "right", "fp16"),
    (1000, 1, 2, 2, 64, 129, 5, None, "bf16"),
    (640, 2, 2, 2, 64, 512, 4, "any", "fp16"),
    (260, 1, 2, 1, 33, 50, 9, "any", "bf16"),
    (140, 1, 2, 1, 200, 60, 2, "any", "fp16"),
    (300, 12, 16, 4, 64, 100, 4, "right", "bf16"),
    (1, 3, 2, 2, 64, 5, 1, "any", "fp16"),
    (700, 2, 2, 1, 64, 30, 70, "gap", "fp16"),
    (1100, 1, 3, 3, 128, 1, 0, "gap", "fp16"),
    (1500, 1, 2, 2, 64, 2000, 3, None, "fp16"),
    (64, 2, 2, 1, 35, 20, 2, "any", "fp16"),
    (63, 2, 2, 1, 35, 20, 2, "any", "fp16"),
    (400, 1, 4, 2, 127, 90, 0, None, "bf16"),
    # first tokens whose many queries are split
    (1500, 1, 2, 1, 64, 30, 4, None, "bf16"),
    (1501, 1, 2, 1, 64, 30, 4, "left", "fp16"),
    (1100, 2, 2, 1, 33, 16, 70, "any", "fp32"),
    (2100, 1, 3, 3, 128, 100, 130, "right", "bf16"),
    (1300, 2, 2, 2, 24, 40, 3, "gap", "fp32"),
    (1300, 1, 2, 1, 128, 1, 200, "gap", "fp16"),
    (1000, 1, 4, 1, 64, 3, 1, "any", "fp16"),
    (1030, 2, 2, 1, 100, 8, 5, "right", "bf16"),
]


def window_inputs(T, B, H, G, D, window, sinks, mask, dtype, view=True):
    torch.manual_seed(T * 5 + D)
    dt = TYPES[dtype]
    return (*make(T, B, (H, G, G), (D, D, D), dt, view), some_mask(mask, B, T), dt)


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window_forward_and_gradients(case):
    from rfa_b200.window_attention import window_attention
    q, k, v, mask, dt = window_inputs(*case)
    kw = dict(window=case[5], sinks=case[6], key_padding_mask=mask)
    go = torch.randn_like(q)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = window_attention(q=leaves[0], k=leaves[1], v=leaves[2], **kw)
    got = torch.autograd.grad(out, leaves, go)
    (want,), gw = grads(lambda *a: window_dense(*a, case[5], case[6], mask), (q, k, v), [go])
    near(out, want, dt, name="out")
    delta = case[4] ** -0.5 * (go.double() * want).sum(-1)
    for n, a, b in zip("qkv", got, gw):
        near(a, b, dt, 4.0, name=n, terms=delta if n != "v" else None)
    if mask is not None:
        for x in (out, *got):
            assert (x[mask.t().bool()] == 0).all()
    with torch.no_grad():
        assert torch.equal(out, window_attention(q=q, k=k, v=v, **kw))


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window_prompt_then_tokens(case):
    """Runs of tokens and single ones through the cache give the whole run's outputs, and the cache holds what it says."""
    from rfa_b200.window_attention import incremental_window_attention
    q, k, v, mask, dt = window_inputs(*case)
    T, B, window, sinks = q.size(0), q.size(1), case[5], case[6]
    want = window_dense(q.double(), k.double(), v.double(), window, sinks, mask)
    cuts = sorted({0, T // 2, T // 2 + (T - T // 2) // 3, *range(max(T - 12, T // 2), T + 1), T})
    state, outs = dict(prev_k=None, prev_v=None, prev_len=None), []
    for a, b in zip(cuts, cuts[1:]):
        if a == b:
            continue
        o, *new = incremental_window_attention(q=q[a:b], k=k[a:b], v=v[a:b], window=window, sinks=sinks, **state,
                                               key_padding_mask=None if mask is None else mask[:, a:b])
        if state["prev_k"] is not None:
            assert new[0] is state["prev_k"] and new[2] is state["prev_len"]
        state = dict(zip(state, new))
        outs.append(o)
    near(torch.cat(outs), want, dt)
    n, real = places(mask, T, B)
    assert torch.equal(state["prev_len"], real.sum(1))
    for b in range(B):
        total = int(real[b].sum())
        for kept, x in ((state["prev_k"], k), (state["prev_v"], v)):
            expect = torch.zeros_like(kept[b])
            for t in range(T):
                p = int(n[b, t])
                if bool(real[b, t]) and (p < sinks or p >= total - window):
                    expect[:, p if p < sinks else sinks + (p - sinks) % window] = x[t, b]
            assert torch.equal(kept[b], expect)


@pytest.mark.parametrize("dtype,H,G,D,window,sinks,B", [("fp32", 4, 4, 40, 300, 4, 2), ("fp16", 16, 16, 64, 512, 4, 2), ("bf16", 8, 1, 128, 1000, 0, 3), ("fp16", 24, 2, 64, 90, 3, 2),
                                                        ("fp16", 3, 1, 50, 70, 1, 2), ("bf16", 10, 2, 256, 200, 5, 2), ("fp32", 8, 2, 200, 64, 64, 1), ("bf16", 4, 2, 24, 5000, 4, 1)])
def test_window_step_on_caches_of_every_age(dtype, H, G, D, window, sinks, B):
    from rfa_b200.window_attention import incremental_window_attention
    torch.manual_seed(D)
    dt, cap = TYPES[dtype], window + sinks
    for age in (0, 1, sinks, cap - 1, cap, cap + 1, 5 * cap + 3, 2 ** 33 + 7):
        q, k, v = make(1, B, (H, G, G), (D, D, D), dt)
        pk, pv = torch.randn(B, G, cap, D, device="cuda").to(dt), torch.randn(B, G, cap, D, device="cuda").to(dt)
        length = torch.full((B,), age, device="cuda")
        length[-1] += 3
        mask = torch.zeros(B, 1, dtype=torch.bool, device="cuda")
        mask[0] = B > 2
        ek, ev, outs = pk.clone(), pv.clone(), []
        for b, n in enumerate(length.tolist()):
            if mask[b]:
                outs.append(torch.zeros(H, D, device="cuda", dtype=torch.float64))
                continue
            slot = n if n < sinks else sinks + (n - sinks) % window
            ek[b, :, slot], ev[b, :, slot] = k[0, b], v[0, b]
            have = min(n + 1, cap)
            s = torch.einsum("gud,gsd->gus", q[0, b].double().view(G, -1, D), ek[b, :, :have].double()) * D ** -0.5
            outs.append(torch.einsum("gus,gsd->gud", s.softmax(-1), ev[b, :, :have].double()).reshape(H, D))
        after = length + (~mask[:, 0]).long()
        for b in range(B):          # what no token has reached may hold anything
            ek[b, :, min(int(after[b]), cap):] = pk[b, :, min(int(after[b]), cap):] = math.nan
            ev[b, :, min(int(after[b]), cap):] = pv[b, :, min(int(after[b]), cap):] = math.nan
        out, nk, nv, nl = incremental_window_attention(q=q, k=k, v=v, window=window, sinks=sinks, prev_k=pk, prev_v=pv, prev_len=length, key_padding_mask=mask)
        near(out[0], torch.stack(outs), dt)
        assert nk is pk and torch.equal(nk.nan_to_num(7.0), ek.nan_to_num(7.0)) and torch.equal(nv.nan_to_num(7.0), ev.nan_to_num(7.0)) and torch.equal(nl, after)


def test_window_masked_rubbish_strides_and_streams():
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    for dt, D in ((torch.float32, 24), (torch.float16, 64), (torch.bfloat16, 128)):
        torch.manual_seed(9)
        q, k, v = make(300, 2, (4, 2, 2), (D, D, D), dt, False)
        mask = torch.zeros(2, 300, dtype=torch.bool, device="cuda")
        mask[0, 10:30] = mask[1, 100:260] = mask[1, 299] = True
        kw = dict(window=50, sinks=3, key_padding_mask=mask)
        clean = window_attention(q=q, k=k, v=v, **kw)
        for x in (q, k, v):
            x[mask.t()] = math.nan
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        dirty = window_attention(q=leaves[0], k=leaves[1], v=leaves[2], **kw)
        assert torch.equal(clean, dirty)
        go = torch.randn_like(clean)
        go[mask.t()] = math.inf
        for x in torch.autograd.grad(dirty, leaves, go):
            assert torch.isfinite(x).all() and (x[mask.t()] == 0).all()
        out, *_ = incremental_window_attention(q=q, k=k, v=v, **kw)
        assert torch.equal(out, clean)
    base = torch.randn(2, 3, 140, 200, device="cuda").half()
    for off in (0, 1, 3, 8):
        q, k, v = (base[..., off + i * 64:off + i * 64 + 64].permute(2, 0, 1, 3) for i in range(3))
        want = window_dense(q.double(), k.double(), v.double(), 40, 2)
        near(window_attention(q=q, k=k, v=v, window=40, sinks=2), want, torch.float16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = window_attention(q=q, k=k, v=v, window=40, sinks=2)
    torch.cuda.current_stream().wait_stream(side)
    near(y, want, torch.float16)
    for T, B, H in ((0, 2, 3), (5, 0, 3), (5, 2, 0)):
        q = torch.zeros(T, B, H, 16, device="cuda", dtype=torch.half, requires_grad=True)
        out = window_attention(q=q, k=q, v=q, window=3)
        out.sum().backward()
        assert out.shape == q.shape and q.grad.shape == q.shape
        with torch.no_grad():
            assert incremental_window_attention(q=q, k=q, v=q, window=3)[0].shape == q.shape


# ------------------------------------------------------------------------------------------------ gradients that are zero
@pytest.mark.parametrize("dtype,D", [("fp32", 16), ("fp16", 64), ("bf16", 128), ("fp16", 33), ("bf16", 200)])
def test_gradients_that_are_zero(dtype, D):
    """A query that sees one key weighs it by 1, and a sequence's first token decays nothing, whatever the inputs are: zeros, and not the roundings of sums that cancel."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    from rfa_b200.window_attention import window_attention
    torch.manual_seed(D)
    T, B, H = 150, 3, 2
    one = torch.ones(B, T, dtype=torch.bool, device="cuda")              # a single token in each sequence, at another place
    one[0, 0] = one[1, 140] = one[2, 149] = False
    left = torch.arange(T, device="cuda")[None] < torch.tensor([[0], [7], [100]], device="cuda")

    def leaves(heads, t=T):
        return [torch.randn(t, B, h, D, device="cuda").to(TYPES[dtype]).requires_grad_() for h in heads]

    for t, window, sinks, mask in ((T, 1, 0, None), (T, 1, 0, left), (1, 5, 0, None), (1, 5, 2, None), (T, 5, 0, one), (T, 5, 2, one)):
        q, k, v = leaves((H, 1, 1), t)
        out = window_attention(q=q, k=k, v=v, window=window, sinks=sinks, key_padding_mask=mask)
        gq, gk, gv = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
        assert not gq.any() and not gk.any() and gv.any(), (t, window, sinks)
    q, k, v = leaves((H, 1, 1))
    out = window_attention(q=q, k=k, v=v, window=5, sinks=2, key_padding_mask=left)
    gq, gk, _ = torch.autograd.grad(out, (q, k, v), torch.randn_like(out))
    for b, n in enumerate((0, 7, 100)):
        assert not gq[:n + 1, b].any() and gq[n + 1:, b].any(-1).all() and not gk[:n, b].any() and gk[n:, b].any(-1).all()

    for t, mask, first in ((T, None, (0, 0, 0)), (T, left, (0, 7, 100)), (1, None, (0, 0, 0)), (2, torch.tensor([[0, 1]] * 3, device="cuda").bool(), (0, 0, 0))):
        q, k, v = leaves((H, H, H), t)
        g = (-0.1 * torch.rand(t, B, H, device="cuda")).to(TYPES[dtype]).requires_grad_()
        out = decay_attention(q=q, k=k, v=v, log_decay=g, key_padding_mask=mask)
        gg, = torch.autograd.grad(out, g, torch.randn_like(out))
        real = torch.ones(t, B, dtype=torch.bool, device="cuda") if mask is None else ~mask.t()
        for b, n in enumerate(first):
            assert not gg[:n + 1, b].any() and gg[n + 1:, b][real[n + 1:, b]].any(-1).all(), (t, b)
        per_head = torch.full((H,), -0.1, device="cuda", requires_grad=True)
        out = decay_attention(q=q, k=k, v=v, log_decay=per_head, key_padding_mask=mask)
        assert bool(torch.autograd.grad(out, per_head, torch.randn_like(out))[0].any()) == (t == T)
    q, k, v = leaves((H, H, H), 1)                                       # a state in front of the first token is decayed by it
    g, s = torch.full((1, B, H), -0.1, device="cuda", requires_grad=True), torch.randn(B, H, D, D, device="cuda")
    out, _ = incremental_decay_attention(q=q, k=k, v=v, log_decay=g, s=s)
    assert torch.autograd.grad(out, g, torch.randn_like(out))[0].all()


# ------------------------------------------------------------------------------------------------ gradients against differences
def test_gradients_against_differences():
    from rfa_b200.decay_attention import decay_attention
    from rfa_b200.window_attention import window_attention
    torch.manual_seed(11)
    q, k, v = (torch.randn(50, 1, 2, 12, device="cuda") for _ in range(3))
    g = -0.2 * torch.rand(50, 1, 2, device="cuda")
    w = torch.randn_like(v)
    for f, leaves in ((lambda q, k, v, g: decay_attention(q=q, k=k, v=v, log_decay=g), (q, k, v, g)),
                      (lambda q, k, v: window_attention(q=q, k=k, v=v, window=9, sinks=2), (q, k, v))):
        leaves = [x.clone().requires_grad_() for x in leaves]
        got = torch.autograd.grad((f(*leaves) * w).sum(), leaves)
        for i, x in enumerate(leaves):
            d, e = torch.randn_like(x), 3e-3
            if i == 3:
                d = -d.abs()
            with torch.no_grad():
                up, down = ([y + s * e * d if j == i else y for j, y in enumerate(leaves)] for s in (1, -1))
                slope = ((f(*up) - f(*down)).double() * w.double()).sum() / (2 * e)
            # the difference's own error: e^2 / 6 of a third derivative of the same size as the slope's terms, and roundings of 2^-24 |f w| / e
            assert abs(slope - (got[i].double() * d.double()).sum()) <= 1e-3 * (got[i].norm() * d.norm()), i


# ------------------------------------------------------------------------------------------------ as they are used
def test_layers_whole_runs_prompts_and_tokens():
    """A block of both layers: a whole run, a prompt and then single tokens, beams that change places, all gradients."""
    from rfa_b200 import DecayAttention, WindowAttention
    torch.manual_seed(13)
    layers = [DecayAttention(embed_dim=128, num_heads=2).cuda().half(), WindowAttention(embed_dim=128, num_heads=4, num_kv_heads=2, window=20, sinks=2).cuda().half(),
              DecayAttention(embed_dim=128, num_heads=2, decay="head").cuda().half()]
    x = torch.randn(150, 3, 128, device="cuda").half()
    pad = torch.arange(150, device="cuda")[None] >= torch.tensor([150, 90, 149], device="cuda")[:, None]

    def block(x, pad=None, states=None):
        for i, layer in enumerate(layers):
            x = x + layer(x, key_padding_mask=pad, saved_state=None if states is None else states[i])
        return x

    y = block(x, pad)
    y.float().square().sum().backward()
    for layer in layers:
        for n, p in layer.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, n
    with torch.no_grad():
        whole, states = block(x), [{} for _ in layers]
        outs = [block(x[:100], None, states)]
        for t in range(100, 125):
            outs.append(block(x[t:t + 1], None, states))
        order = torch.tensor([2, 0, 1], device="cuda")
        states = [layer.reorder_incremental_state(s, order) for layer, s in zip(layers, states)]
        for t in range(125, 150):
            outs.append(block(x[t:t + 1, order], None, states)[:, order.argsort()])
        # six fp16 sums of a residual stream, each rounded once, and a token's own small differences through three layers
        assert (torch.cat(outs) - whole).double().norm() <= 16 * unit(torch.float16) * whole.double().norm()


def test_decoding_inside_a_graph():
    from rfa_b200.decay_attention import incremental_decay_attention
    from rfa_b200.window_attention import incremental_window_attention
    torch.manual_seed(17)
    T, B, H, D, W = 12, 2, 4, 64, 5
    q, k, v = make(T, B, (H, H, H), (D, D, D), torch.float16, False)
    g = -0.1 * torch.rand(T, B, H, device="cuda")
    sq, sk, sv, sg = (x[:1].clone() for x in (q, k, v, g))
    s = torch.zeros(B, H, D, D, device="cuda")
    cache = dict(prev_k=torch.zeros(B, H, W + 1, D, device="cuda").half(), prev_v=torch.zeros(B, H, W + 1, D, device="cuda").half(), prev_len=torch.zeros(B, device="cuda", dtype=torch.long))

    def step():
        a, _ = incremental_decay_attention(q=sq, k=sk, v=sv, log_decay=sg, s=s)
        b, *_ = incremental_window_attention(q=sq, k=sk, v=sv, window=W, sinks=1, **cache)
        return a, b

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = step()
    s.zero_()
    cache["prev_len"].zero_()
    outs = []
    for t in range(T):
        for dst, src in ((sq, q), (sk, k), (sv, v), (sg, g)):
            dst.copy_(src[t:t + 1])
        graph.replay()
        outs.append((a.clone(), b.clone()))
    near(torch.cat([o[0] for o in outs]), decay_dense(*(x.double() for x in (q, k, v, g)))[0], torch.float16)
    near(torch.cat([o[1] for o in outs]), window_dense(q.double(), k.double(), v.double(), W, 1), torch.float16)


def test_training_step_inside_a_graph():
    from rfa_b200.decay_attention import decay_attention
    from rfa_b200.window_attention import window_attention
    torch.manual_seed(19)
    q, k, v = (x.requires_grad_() for x in make(200, 2, (2, 2, 2), (64, 64, 64), torch.float16, False))
    g = (-0.1 * torch.rand(200, 2, 2, device="cuda")).requires_grad_()
    go = torch.randn_like(v)

    def step():
        a = torch.autograd.grad(decay_attention(q=q, k=k, v=v, log_decay=g), (q, k, v, g), go)
        return (*a, *torch.autograd.grad(window_attention(q=q, k=k, v=v, window=30, sinks=1), (q, k, v), go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    z = lambda *s, dt=torch.half: torch.zeros(*s, device="cuda", dtype=dt)
    q, g = z(4, 2, 2, 16), z(4, 2, 2, dt=torch.float32)
    with pytest.raises(TypeError):
        decay_attention(q=q, k=q.float(), v=q, log_decay=g)
    with pytest.raises(TypeError):
        decay_attention(q=q, k=q, v=q, log_decay=g.bfloat16())
    with pytest.raises(TypeError):
        decay_attention(q=q.double(), k=q.double(), v=q.double(), log_decay=g)
    with pytest.raises(AssertionError):
        decay_attention(q=q, k=q, v=q, log_decay=g[:3])
    with pytest.raises(AssertionError):
        decay_attention(q=q, k=q, v=q, log_decay=g, key_padding_mask=z(4, 2))
    with pytest.raises(ValueError):
        decay_attention(q=z(4, 2, 2, 257), k=z(4, 2, 2, 257), v=q, log_decay=g)
    with pytest.raises(ValueError):
        incremental_decay_attention(q=q, k=q, v=q, log_decay=g, s=z(2, 2, 16, 16, dt=torch.float32).transpose(-1, -2))
    with pytest.raises(TypeError):
        incremental_decay_attention(q=q, k=q, v=q, log_decay=g, s=z(2, 2, 16, 16))
    with pytest.raises(ValueError):
        window_attention(q=q, k=q, v=q, window=0)
    with pytest.raises(ValueError):
        window_attention(q=q, k=q, v=q, window=3, sinks=-1)
    with pytest.raises(ValueError):
        window_attention(q=z(4, 2, 3, 16), k=q, v=q, window=3)
    with pytest.raises(AssertionError):
        window_attention(q=q, k=q, v=z(4, 2, 2, 8), window=3)
    cache = dict(prev_k=z(2, 2, 3, 16), prev_v=z(2, 2, 3, 16), prev_len=z(2, dt=torch.long))
    with pytest.raises(AssertionError):
        incremental_window_attention(q=q, k=q, v=q, window=4, **cache)
    with pytest.raises(ValueError):
        incremental_window_attention(q=q, k=q, v=q, window=3, prev_k=cache["prev_k"])
    with pytest.raises(ValueError):
        incremental_window_attention(q=q, k=q, v=q, window=3, **{**cache, "prev_v": cache["prev_k"]})
    with pytest.raises(TypeError):
        incremental_window_attention(q=q, k=q, v=q, window=3, **{**cache, "prev_len": z(2, dt=torch.int32)})
    with pytest.raises(RuntimeError):
        incremental_window_attention(q=q.clone().requires_grad_(), k=q, v=q, window=3, **cache)
    x = z(4, 2, 2, 16).requires_grad_()
    for y in (decay_attention(q=x, k=q, v=q, log_decay=g), window_attention(q=x, k=q, v=q, window=3)):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_decay_backward_without_what_the_forward_kept():
    """The tensor-level backward computes the states again where it is not handed them, with the same bits."""
    from rfa_b200 import ops
    torch.manual_seed(23)
    for K, D in ((64, 64), (128, 128)):
        q, k, v = make(400, 2, (2, 2, 2), (K, K, D), torch.float16, False)
        g, s = (-0.1 * torch.rand(400, 2, 2, device="cuda")).half(), torch.randn(2, 2, K, D, device="cuda")
        go = torch.randn_like(v)
        out, last, kept = ops.decay_attention_fwd(q, k, v, g, s, save=True, return_state=True)
        assert kept is not None and ops.decay_attention_fwd(q, k, v, g, s)[2] is None
        with_it = ops.decay_attention_bwd(q, k, v, g, s, None, None, go, kept=kept, need_state=True)
        without = ops.decay_attention_bwd(q, k, v, g, s, None, None, go, need_state=True)
        _, want = grads(lambda *a: decay_dense(*a), (q, k, v, g, s), [go])
        for a, b, w in zip(with_it, without, want):
            near(a, w, torch.float16, 12.0, terms=q.double().square().sum(-1) * 0 + 1 if w.dim() == 3 else None)
            near(b, w, torch.float16, 12.0, terms=q.double().square().sum(-1) * 0 + 1 if w.dim() == 3 else None)
        with pytest.raises(ValueError):
            ops.decay_attention_bwd(q, k, v, g, s, None, None, go, kept=kept[:100])


def test_calls_on_two_streams_at_once_and_the_same_bits_again():
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    from rfa_b200.window_attention import window_attention
    torch.manual_seed(29)
    jobs = []
    for i in range(2):
        q, k, v = make(900, 2, (4, 4, 4), (64, 64, 64), torch.float16)
        jobs.append((q, k, v, -0.1 * torch.rand(900, 2, 4, device="cuda")))

    def work(q, k, v, g):
        a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
        o = decay_attention(q=a, k=b, v=c, log_decay=g) + window_attention(q=a, k=b, v=c, window=200, sinks=3)
        return (o, *torch.autograd.grad(o, (a, b, c), q), *incremental_decay_attention(q=q, k=k, v=v, log_decay=g))

    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(*j))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)


def test_offsets_beyond_32_bits():
    """A cache of 2^31 numbers a row and key head, and a batch whose activations pass 2^31 numbers: the last rows are what they are by themselves."""
    from rfa_b200.decay_attention import decay_attention
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    torch.manual_seed(31)
    D, window = 128, 2 ** 24
    pk, pv = (torch.zeros(2, 1, window, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    at = window - 3                                       # only the last few slots of the second row weigh anything
    pk[1, 0, at:], pv[1, 0, at:] = torch.randn(3, D, device="cuda").bfloat16(), torch.randn(3, D, device="cuda").bfloat16()
    q = torch.randn(1, 2, 4, D, device="cuda").bfloat16() * 40
    k, v = (torch.randn(1, 2, 1, D, device="cuda").bfloat16() for _ in range(2))
    length = torch.tensor([5, 3 * window + at + 2], device="cuda")
    out, nk, nv, nl = incremental_window_attention(q=q, k=k, v=v, window=window, prev_k=pk, prev_v=pv, prev_len=length)
    assert nl.tolist() == [6, 3 * window + at + 3] and torch.equal(nk[1, 0, -1], k[0, 1, 0]) and torch.equal(nv[1, 0, -1], v[0, 1, 0])
    s = torch.einsum("hd,sd->hs", q[0, 1].double(), pk[1, 0, at:].double()) * D ** -0.5
    rest = (window - 3) * torch.exp(-s.amax(1, keepdim=True))
    p = torch.exp(s - s.amax(1, keepdim=True))
    near(out[0, 1], (p / (p.sum(1, keepdim=True) + rest)) @ pv[1, 0, at:].double(), torch.bfloat16)
    del pk, pv, nk, nv
    T, B, H = 4200, 64, 64                                # 2.2e9 numbers an array
    q, k, v = (torch.empty(T, B, H, D, device="cuda", dtype=torch.bfloat16).normal_() for _ in range(3))
    g = torch.full((H,), -0.5, device="cuda")             # e^-64 after 128 tokens
    w = [x[-300:, -1:, -2:].clone() for x in (q, k, v)]
    with torch.no_grad():
        near(decay_attention(q=q, k=k, v=v, log_decay=g)[-100:, -1:, -2:], decay_dense(*(x.double() for x in w), g[-2:].double())[0][-100:], torch.bfloat16)
        near(window_attention(q=q, k=k, v=v, window=100)[-100:, -1:, -2:], window_dense(*(x.double() for x in w), 100, 0)[-100:], torch.bfloat16)
