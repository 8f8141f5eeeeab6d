"""Decaying and windowed attention at the limits of numbers: tokens that are not finite, scores and decays beyond usual ranges, zeros behind long padding, and what is refused.

Tolerances are those of test_gpu_attention.py."""
import math

import pytest
import torch
from test_gpu_attention import TYPES, make, near, places, some_mask

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
