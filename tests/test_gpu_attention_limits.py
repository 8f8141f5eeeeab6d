"""Decaying and windowed attention at the limits of numbers: tokens that are not finite, scores and decays beyond usual ranges, zeros behind long padding, and what is refused.

Tolerances are those of test_gpu_attention.py."""
import math

import pytest
import torch
from test_gpu_attention import TYPES, decay_dense, grads, make, near, places, some_mask, window_dense

pytestmark = pytest.mark.gpu


def sees(mask, T, B, window, sinks):
    """[B, query, key]"""
    n, real = places(mask, T, B)
    at = torch.arange(T, device="cuda")
    return real[:, :, None] & real[:, None, :] & (at[:, None] >= at) & ((n[:, :, None] - n[:, None, :] < window) | (n[:, None, :] < sinks))


def window_by_rows(q, k, v, seen, scale):
    """Each query with the keys that it sees alone, in 64 bits: what is not seen cannot reach it, whatever it is."""
    T, B, H, D = q.shape
    q, k, v = (x.double() for x in (q, k, v))
    out = torch.zeros(T, B, H, D, device="cuda", dtype=torch.float64)
    for b in range(B):
        for t in range(T):
            js = seen[b, t].nonzero()[:, 0]
            if len(js):
                K, V = (x[js, b].repeat_interleave(H // k.size(2), 1) for x in (k, v))
                out[t, b] = torch.einsum("hj,jhd->hd", torch.softmax(scale * torch.einsum("hd,jhd->hj", q[t, b], K), -1), V)
    return out


# ------------------------------------------------------------------------------------------------ window
# fp32; 16 bits beyond 128; 16 bits with a scale that the tensor cores leave alone; the tensor cores at both widths, without and with padding
NOT_FINITE = [("fp32", 24, None, None), ("fp32", 40, None, "any"), ("bf16", 200, None, None), ("fp16", 64, -0.125, None), ("fp16", 64, None, None), ("bf16", 128, None, None),
              ("fp16", 40, None, "any"), ("bf16", 128, None, "left")]


@pytest.mark.parametrize("what,value", [("q", math.nan), ("k", math.nan), ("k", math.inf), ("v", math.nan), ("v", -math.inf)])
@pytest.mark.parametrize("dtype,D,scale,pad", NOT_FINITE)
def test_window_passes_on_what_is_not_finite(dtype, D, scale, pad, what, value):
    """A query that sees a NaN or an infinite score has what softmax gives, in a prompt as in single tokens: never zeros."""
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    torch.manual_seed(D)
    T, B, H, G, window, sinks, at = 200, 2, 4, 2, 60, 2, 90
    q, k, v = make(T, B, (H, G, G), (D, D, D), TYPES[dtype], False)
    mask = some_mask(pad, B, T)
    if mask is not None:
        mask[1] = False
        mask[1, 20:31] = True
    dict(q=q, k=k, v=v)[what][at, 1, 1, 3] = value
    seen, s = sees(mask, T, B, window, sinks), D ** -0.5 if scale is None else scale
    want = window_by_rows(q, k, v, seen, s)
    kw = dict(window=window, sinks=sinks, scale=scale)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = window_attention(q=leaves[0], k=leaves[1], v=leaves[2], key_padding_mask=mask, **kw)
    with torch.no_grad():
        got = [out, incremental_window_attention(q=q, k=k, v=v, key_padding_mask=mask, **kw)[0]]
        state, outs = {}, []
        for a, b in [(0, 80)] + [(t, t + 1) for t in range(80, 100)] + [(100, T)]:
            o, *new = incremental_window_attention(q=q[a:b], k=k[a:b], v=v[a:b], key_padding_mask=None if mask is None else mask[:, a:b], **state, **kw)
            state = dict(zip(("prev_k", "prev_v", "prev_len"), new))
            outs.append(o)
        got.append(torch.cat(outs))
    reached = seen[1, :, at] if what != "q" else torch.arange(T, device="cuda") == at
    assert not torch.isfinite(want[reached, 1]).all() and torch.isfinite(want[~reached]).all()
    for x in got:
        assert torch.equal(torch.isfinite(x[reached]), torch.isfinite(want[reached]))
        near(x[:, 0], want[:, 0], TYPES[dtype])
        if what != "v":                                     # a weight of nothing times a NaN is one: how far values reach is tested by itself
            near(x[:, 1][~reached], want[:, 1][~reached], TYPES[dtype])
    gq, = torch.autograd.grad(out, leaves[0], torch.randn_like(out))
    bad = ~torch.isfinite(want).all(-1)
    assert not torch.isfinite(gq[bad]).all(-1).any() and torch.isfinite(gq[:, 0]).all()


@pytest.mark.parametrize("dtype,D,pad", [("fp32", 24, None), ("bf16", 64, None), ("bf16", 128, "any"), ("bf16", 200, None)])
def test_window_scores_far_below_zero(dtype, D, pad):
    """Scores of -1e32 and less have a largest one too."""
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    torch.manual_seed(D)
    T, B, H, window, dt = 150, 2, 2, 7, TYPES[dtype]
    v = torch.randn(T, B, H, D, device="cuda").to(dt)
    q = torch.full_like(v, 1e16)
    k = (torch.full_like(v, -1e16).float() * (1 + torch.arange(T, device="cuda") % 10 / 16)[:, None, None, None]).to(dt)      # steps of 6 %, so that one key has all the weight
    mask = some_mask(pad, B, T)
    want = window_by_rows(q, k, v, sees(mask, T, B, window, 1), D ** -0.5)
    near(window_attention(q=q, k=k, v=v, window=window, sinks=1, key_padding_mask=mask), want, dt)
    state, outs = {}, []
    for a, b in [(0, 30)] + [(t, t + 1) for t in range(30, T)]:
        o, *new = incremental_window_attention(q=q[a:b], k=k[a:b], v=v[a:b], window=window, sinks=1, key_padding_mask=None if mask is None else mask[:, a:b], **state)
        state = dict(zip(("prev_k", "prev_v", "prev_len"), new))
        outs.append(o)
    near(torch.cat(outs), want, dt)


@pytest.mark.parametrize("dtype,D,pad,window,sinks,at", [("fp32", 24, None, 64, 4, 40), ("fp16", 64, None, 64, 4, 40), ("bf16", 128, None, 64, 4, 40), ("fp16", 64, "left", 64, 4, 90),
                                                         ("bf16", 128, "gap", 50, 70, 100), ("bf16", 200, None, 64, 4, 20), ("fp16", 64, None, 2, 0, 832), ("fp16", 64, None, 300, 130, 140),
                                                         ("fp32", 24, "right", 2, 1, 9), ("bf16", 100, None, 30, 1, 2)])
def test_window_reach_of_what_is_not_finite(dtype, D, pad, window, sinks, at):
    """Outputs and queries' gradients 320 tokens and more from the last that sees a token, and the same in front of it, are what they are without it -- behind first tokens
    that lie beside it, too."""
    from rfa_b200.window_attention import incremental_window_attention, window_attention
    torch.manual_seed(D)
    T, B, H, G, dt = 1500, 2, 4, 2, TYPES[dtype]
    q, k, v = make(T, B, (H, G, G), (D, D, D), dt, False)
    mask = some_mask(pad, B, T)
    n, real = places(mask, T, B)
    place = ((n[1] == at) & real[1]).nonzero()[0, 0]
    assert at >= sinks
    k[place, 1] = v[place, 1] = 0.0
    go = torch.randn_like(q)
    (want,), gw = grads(lambda *a: window_dense(*a, window, sinks, mask), (q, k, v), [go])
    beyond = real[1] & ((n[1] >= at + window - 1 + 320) | (n[1] <= at - 320))
    spared = ~sees(mask, T, B, window, sinks)[1, :, place] & beyond
    assert spared.any()
    k[place, 1], v[place, 1] = math.nan, math.inf
    kw = dict(window=window, sinks=sinks, key_padding_mask=mask)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = window_attention(q=leaves[0], k=leaves[1], v=leaves[2], **kw)
    gq, = torch.autograd.grad(out, leaves[0], go)
    with torch.no_grad():
        later = incremental_window_attention(q=q, k=k, v=v, **kw)[0]
        first = incremental_window_attention(q=q[:600], k=k[:600], v=v[:600], **{**kw, "key_padding_mask": None if mask is None else mask[:, :600]})
        then = incremental_window_attention(q=q[600:], k=k[600:], v=v[600:], prev_k=first[1], prev_v=first[2], prev_len=first[3],
                                            **{**kw, "key_padding_mask": None if mask is None else mask[:, 600:]})[0]
    delta = D ** -0.5 * (go.double() * want).sum(-1)
    for x in (out, later, torch.cat([first[0], then])):
        near(x[spared, 1], want[spared, 1], dt)
        near(x[:, 0], want[:, 0], dt)
    near(gq[spared, 1], gw[0][spared, 1], dt, 4.0, terms=delta[spared, 1])
    near(gq[:, 0], gw[0][:, 0], dt, 4.0, terms=delta[:, 0])


@pytest.mark.parametrize("dtype,D,G,pad,window,sinks", [("fp32", 24, 2, None, 64, 4), ("fp16", 64, 2, None, 64, 4), ("bf16", 128, 2, "right", 50, 4), ("bf16", 64, 1, None, 30, 70), ("fp16", 64, 2, None, 40, 0)])
def test_window_reach_of_gradients_that_are_not_finite(dtype, D, G, pad, window, sinks):
    from rfa_b200.window_attention import window_attention
    torch.manual_seed(D)
    T, B, H, dt = 1500, 2, 4, TYPES[dtype]
    q, k, v = make(T, B, (H, G, G), (D, D, D), dt, False)
    mask, at = some_mask(pad, B, T), 700
    n, real = places(mask, T, B)
    go = torch.randn_like(q)
    go[at, 1] = 0.0
    (want,), gw = grads(lambda *a: window_dense(*a, window, sinks, mask), (q, k, v), [go])
    go[at, 1] = math.nan
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    gq, gk, gv = torch.autograd.grad(window_attention(q=leaves[0], k=leaves[1], v=leaves[2], window=window, sinks=sinks, key_padding_mask=mask), leaves, go)
    delta = D ** -0.5 * (go.nan_to_num().double() * want).sum(-1)
    others = torch.arange(T, device="cuda") != at
    near(gq[others, 1], gw[0][others, 1], dt, 4.0, terms=delta[others, 1])
    assert not torch.isfinite(gq[at, 1]).any()
    seen = sees(mask, T, B, window, sinks)[1, at]
    assert not torch.isfinite(gk[seen, 1]).any() and not torch.isfinite(gv[seen, 1]).any()
    spared = real[1] & ((n[1] >= at + 320) | (n[1] <= at - (window - 1) - 320)) & (n[1] >= (sinks + 128 if sinks else 0))
    assert spared.sum() > 300
    near(gk[spared, 1], gw[1][spared, 1], dt, 4.0, terms=delta[spared, 1])
    near(gv[spared, 1], gw[2][spared, 1], dt, 4.0)
    for x, w in ((gk, gw[1]), (gv, gw[2])):
        near(x[:, 0], w[:, 0], dt, 4.0, terms=delta[:, 0] if w is gw[1] else None)


def test_window_caches_that_overlap_are_refused():
    from rfa_b200.window_attention import incremental_window_attention
    room = torch.zeros(2 * 2 * 4 * 16 + 64, device="cuda").half()
    q, n = torch.zeros(1, 2, 2, 16, device="cuda").half(), 2 * 2 * 4 * 16
    length = torch.zeros(2, device="cuda", dtype=torch.long)
    pk = room[:n].view(2, 2, 4, 16)
    for off in (64, 16, 8):
        for a, b in ((pk, room[off:off + n].view_as(pk)), (room[off:off + n].view_as(pk), pk)):
            with pytest.raises(ValueError):
                incremental_window_attention(q=q, k=q, v=q, window=4, prev_k=a, prev_v=b, prev_len=length)
    both = torch.zeros(2 * n, device="cuda").half()      # side by side is fine
    incremental_window_attention(q=q, k=q, v=q, window=4, prev_k=both[:n].view_as(pk), prev_v=both[n:].view_as(pk), prev_len=length)
    assert length.tolist() == [1, 1]


# ------------------------------------------------------------------------------------------------ decay
@pytest.mark.parametrize("value", [math.nan, math.inf, 1e30])
@pytest.mark.parametrize("at", [0, 150])
@pytest.mark.parametrize("dtype,K,D,decay", [("fp32", 24, 40, "token"), ("fp16", 64, 64, "token"), ("bf16", 128, 128, "token"), ("bf16", 64, 128, "fp32"), ("bf16", 200, 64, "token"),
                                             ("fp16", 33, 90, "token")])
def test_decay_that_is_not_finite(dtype, K, D, decay, at, value):
    """A decay that is no number, or growth beyond all numbers, shows in every result that it is part of, in prompts, states, gradients and single tokens alike."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    torch.manual_seed(K)
    T, dt = 400, TYPES[dtype]
    if value == 1e30 and dt == torch.float16:
        value = 60000.0
    q, k, v = make(T, 2, (2, 2, 2), (K, K, D), dt, False)
    g = (-0.1 * torch.rand(T, 2, 2, device="cuda")).to(torch.float32 if decay == "fp32" else dt)
    s = torch.randn(2, 2, K, D, device="cuda")
    go = torch.randn_like(v)
    bad = g.clone()
    bad[at, 1, 1] = value

    def results(g):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, g)]
        out = decay_attention(q=leaves[0], k=leaves[1], v=leaves[2], log_decay=leaves[3])
        with_state, last = incremental_decay_attention(q=q, k=k, v=v, log_decay=g, s=s.clone())
        tokens, one = [], s.clone()
        for t in range(max(at - 2, 0), at + 3):
            tokens.append(incremental_decay_attention(q=q[t:t + 1], k=k[t:t + 1], v=v[t:t + 1], log_decay=g[t:t + 1], s=one)[0])
        return [out, with_state, *torch.autograd.grad(out, leaves, go)], [last, one], torch.cat(tokens)

    clean, dirty = results(g), results(bad)
    for x, y in zip(clean[0], dirty[0]):                    # other rows and heads, and what came before, as they were
        assert torch.isfinite(x).all()
        assert torch.equal(x[:, 0], y[:, 0]) and torch.equal(x[:, 1, 0], y[:, 1, 0])
    out, with_state, gq, gk, gv, gg = (x[:, 1, 1] for x in dirty[0])
    assert not torch.isfinite(with_state[at:]).all(-1).any()
    if at:
        assert not torch.isfinite(out[at:]).all(-1).any() and not torch.isfinite(gq[at:]).all(-1).any()
        assert torch.equal(out[:at], clean[0][0][:at, 1, 1]) and torch.equal(with_state[:at], clean[0][1][:at, 1, 1])
        assert not torch.isfinite(gk[:at]).all(-1).any() and not torch.isfinite(gv[:at]).all(-1).any() and not torch.isfinite(gg[1:at]).any()
    for x, y in zip(clean[1], dirty[1]):
        assert torch.isfinite(x).all() and not torch.isfinite(y[1, 1]).any() and torch.equal(x[0], y[0]) and torch.equal(x[1, 0], y[1, 0])
    first = min(at, 2)
    assert not torch.isfinite(dirty[2][first:, 1, 1]).all(-1).any() and torch.equal(dirty[2][:first], clean[2][:first])


def test_decay_of_a_head_that_is_not_finite():
    from rfa_b200.decay_attention import decay_attention
    torch.manual_seed(2)
    for dt, K in ((torch.float32, 24), (torch.float16, 64), (torch.bfloat16, 128)):
        q, k, v = make(300, 2, (3, 3, 3), (K, K, K), dt, False)
        g = torch.tensor([-0.1, math.nan, -0.2], device="cuda", requires_grad=True)
        out = decay_attention(q=q, k=k, v=v, log_decay=g)
        gg, = torch.autograd.grad(out, g, torch.randn_like(out))
        assert torch.isfinite(out[:, :, ::2]).all() and torch.isnan(out[:, :, 1]).all()
        assert torch.isfinite(gg).tolist() == [True, False, True]


@pytest.mark.parametrize("T", [20, 300])
def test_decay_scores_beyond_half(T):
    """fp16, raw scores of 131072: what counts is the scaled score."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    torch.manual_seed(3)
    q, k = (torch.full((T, 2, 2, 128), 32.0, device="cuda").half() for _ in range(2))
    v = (0.1 * torch.randn(T, 2, 2, 128, device="cuda")).half()
    g = torch.full((T, 2, 2), -0.1, device="cuda")
    want, last = decay_dense(*(x.double() for x in (q, k, v, g)))
    near(decay_attention(q=q, k=k, v=v, log_decay=g), want, torch.float16)
    out, s = incremental_decay_attention(q=q, k=k, v=v, log_decay=g)
    near(out, want, torch.float16)
    near(s, last, torch.float32, 8.0)


def test_decay_scores_that_fit_without_their_scale():
    """fp16, scores of 100 and a scale of 1e4: what counts is the product with the values."""
    from rfa_b200.decay_attention import decay_attention
    torch.manual_seed(4)
    q, k = (torch.randn(150, 2, 2, 64, device="cuda").half() for _ in range(2))
    v = (1e-3 * torch.randn(150, 2, 2, 64, device="cuda")).half()
    g = torch.full((150, 2, 2), -0.1, device="cuda")
    for scale in (1e4, -1e4, 0.0, -0.25):
        near(decay_attention(q=q, k=k, v=v, log_decay=g, scale=scale), decay_dense(*(x.double() for x in (q, k, v, g)), scale=scale)[0], torch.float16)


@pytest.mark.parametrize("dtype,K", [("fp32", 16), ("fp16", 64), ("bf16", 128), ("bf16", 200)])
def test_zero_gradient_of_a_first_token_behind_long_padding(dtype, K):
    from rfa_b200.decay_attention import decay_attention
    torch.manual_seed(K)
    T, H, first = 900, 2, (0, 127, 128, 129, 300, 512, 898, 899)
    B = len(first)
    mask = torch.arange(T, device="cuda")[None] < torch.tensor(first, device="cuda")[:, None]
    mask[4, 400:700] = True                                 # a gap behind the first token
    mask[2, 200] = mask[2, 256] = True
    q, k, v = make(T, B, (H, H, H), (K, K, K), TYPES[dtype], False)
    g = (-0.1 * torch.rand(T, B, H, device="cuda")).to(TYPES[dtype]).requires_grad_()
    out = decay_attention(q=q, k=k, v=v, log_decay=g, key_padding_mask=mask)
    gg, = torch.autograd.grad(out, g, torch.randn_like(out))
    for b, n in enumerate(first):
        assert not gg[:n + 1, b].any() and gg[n + 1:, b][~mask[b, n + 1:]].any(-1).all(), b


def test_decay_backward_on_states_of_its_own_has_the_same_bits():
    """Behind a forward that returned no state, what it kept and what the backward computes for itself are the same."""
    from rfa_b200 import ops
    torch.manual_seed(23)
    for dt, K, D, T in ((torch.float16, 64, 64, 400), (torch.bfloat16, 128, 128, 400), (torch.bfloat16, 64, 128, 5000)):
        q, k, v = make(T, 2, (2, 2, 2), (K, K, D), dt, False)
        g, go = (-0.1 * torch.rand(T, 2, 2, device="cuda")).to(dt), torch.randn_like(v)
        kept = ops.decay_attention_fwd(q, k, v, g, save=True)[2]
        assert kept is not None
        for a, b in zip(ops.decay_attention_bwd(q, k, v, g, None, None, None, go, kept=kept)[:4], ops.decay_attention_bwd(q, k, v, g, None, None, None, go)[:4]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,K", [("fp32", 24), ("fp16", 64), ("bf16", 128), ("fp16", 33), ("bf16", 200)])
def test_decay_reach_of_what_is_not_finite(dtype, K):
    """A token that is not finite reaches all outputs behind it, in its row and head, and none 128 places and more in front."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    torch.manual_seed(K)
    T, dt, at = 500, TYPES[dtype], 300
    q, k, v = make(T, 2, (2, 2, 2), (K, K, K), dt, False)
    g = -0.01 * torch.rand(T, 2, 2, device="cuda")
    clean = decay_attention(q=q, k=k, v=v, log_decay=g)
    for i, value in ((0, math.nan), (1, math.nan), (1, math.inf), (2, -math.inf)):
        x = [y.clone() for y in (q, k, v)]
        x[i][at, 1, 1, 2] = value
        for out in (decay_attention(q=x[0], k=x[1], v=x[2], log_decay=g), incremental_decay_attention(q=x[0], k=x[1], v=x[2], log_decay=g)[0]):
            near(out[:, 0], clean[:, 0].double(), dt)
            near(out[:, 1, 0], clean[:, 1, 0].double(), dt)
            near(out[:at - 127, 1, 1], clean[:at - 127, 1, 1].double(), dt)
            behind = out[at:at + 1, 1, 1] if i == 0 else out[at:, 1, 1]
            assert not torch.isfinite(behind).all(-1).any()
            if i == 0:
                near(out[at + 1:, 1, 1], clean[at + 1:, 1, 1].double(), dt)


@pytest.mark.parametrize("dtype,K,D", [("fp32", 64, 64), ("fp32", 24, 40), ("fp32", 130, 72), ("bf16", 200, 64), ("fp16", 64, 64), ("bf16", 128, 128), ("bf16", 64, 128), ("fp16", 33, 90)])
@pytest.mark.parametrize("rate", [0.01, 1.0, 3.0, 10.0])
def test_gradient_of_decays_of_any_strength(dtype, K, D, rate):
    """Of the gradient itself and not of what cancels in it: pairs of tokens that a decay is not between leave nothing.  Sums over 700 tokens of terms of any sign, each with the rounding
    of its weight and of two products: 12 roundings of the norm over the heads."""
    from rfa_b200.decay_attention import decay_attention, incremental_decay_attention
    torch.manual_seed(K)
    T, H, dt = 700, 8, TYPES[dtype]
    q, k, v = make(T, 2, (H, H, H), (K, K, D), dt, False)
    s, go = torch.randn(2, H, K, D, device="cuda"), torch.randn_like(v)
    gs = torch.randn_like(s)
    mask = some_mask("any", 2, T)
    mask[0] = False
    for g in (torch.full((H,), -rate, device="cuda"), -rate * (0.5 + 0.5 * torch.rand(T, 2, H, device="cuda"))):
        x = g.clone().requires_grad_()
        got, = torch.autograd.grad(decay_attention(q=q, k=k, v=v, log_decay=x, key_padding_mask=mask), x, go)
        near(got, grads(lambda g: decay_dense(q.double(), k.double(), v.double(), g, mask=mask)[0], (g,), [go])[1][0], dt, 12.0)
        got, = torch.autograd.grad(incremental_decay_attention(q=q, k=k, v=v, log_decay=x, s=s, key_padding_mask=mask), x, (go, gs))
        near(got, grads(lambda g: decay_dense(q.double(), k.double(), v.double(), g, s.double(), mask), (g,), [go, gs])[1][0], dt, 12.0)
