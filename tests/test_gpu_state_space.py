"""The state-space operators on the GPU against their oracle in 64 bits.

Tolerances.  A result in a 16-bit type is off by its own rounding, half a step of that type relative to the value, and by what
fp32 sums lose: a bound that scales with ``size``, the same sum over the magnitudes of its terms (the oracle's ``absolute``).
  convolution  W + 1 terms, the sigmoid 5e-7 relative (ex2 2^-22, two roundings, a reciprocal): 2^-19 size; its weight gradients, chains
               of 32 tokens, four warps and the parts: 2^-17 size
  scan         a state is a product of at most T decays, each off by 2^-22 (ex2) + 2^-24 (the product) and by its argument's roundings (three, and
               softplus 2^-22: times |delta a| exp(delta a) <= 0.37 each), times a term of three roundings, summed T times:
               (8 T + 16) 2^-24 size; outputs sum N states; gradients are products of two such, summed over T tokens, B rows and
               the channels: (20 T + 64 + B + D + 2 N) 2^-24 size
  norm         mean and variance of C / groups terms in chains of at most 32 and a tree, rsqrt 2 ulp, the sigmoid: 2^-18 size with the
               condition of the subtraction of the mean; weight gradients are sums of `rows` terms: (2^-18 + rows 2^-24) size
The smallest normal number is added where a type has subnormal results."""
import itertools

import pytest
import torch

from oracle import state_space_oracle as O
from rfa_b200 import SelectiveStateSpace, ops
from rfa_b200 import state_space as ss

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def near(got, want, size, unit, what):
    """|got - want| <= half a step of got's type + unit * size, element by element; the same places finite."""
    info = torch.finfo(got.dtype)
    got, want, size = got.detach().double().cpu(), want.double().cpu(), size.double().cpu()
    assert got.shape == want.shape, what
    rounding = info.eps / 2 if info.bits < 32 else 0.0
    bad = (got - want).abs() > rounding * want.abs() + unit * size + info.tiny
    bad |= ~got.isfinite()
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / (size + 1e-30)).max()):.2e} of size"


def padding(B, T, kind, gen):
    if kind is None:
        return None
    m = torch.zeros(B, T, dtype=torch.bool)
    for b in range(B):
        n = int(torch.randint(0, T + 1, (1,), generator=gen))
        if kind == "right":
            m[b, n:] = True
        elif kind == "left":
            m[b, :T - n] = True
        else:
            m[b] = torch.rand(T, generator=gen) < 0.5
    m[0] = kind == "right"                                        # a row that is all padding, or none of it
    return m


def poison(t, mask):
    """Values that must not be read in padded places."""
    if mask is not None:
        t[mask.t()] = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(t.dtype).min])[
            torch.randint(0, 4, t[mask.t()].shape, generator=torch.Generator().manual_seed(7))].to(t.dtype)
    return t


def clean(t, mask):
    return t if mask is None else torch.where(mask.t().view(*mask.t().shape, *[1] * (t.dim() - 2)), 0.0, t)


def strided(t, kind, dev):
    """The same values on the device: contiguous, batch first, a slice of wider rows, at an odd address."""
    if kind == "batch first":
        return t.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
    if kind == "slice":
        wide = torch.full((*t.shape[:-1], 2 * t.shape[-1] + 8), float("nan"), dtype=t.dtype, device=dev)
        wide[..., 8:8 + t.shape[-1]] = t.to(dev)
        return wide[..., 8:8 + t.shape[-1]]
    if kind == "odd":
        flat = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device=dev)
        flat[1:] = t.flatten().to(dev)
        return flat[1:].view(t.shape)
    return t.to(dev)


def leaves(*ts):
    return [None if t is None else t.detach().requires_grad_() for t in ts]


# --------------------------------------------------------------------------- convolution
CONV = list(itertools.product([(1, 1, 1), (1, 3, 8), (2, 2, 5), (3, 3, 40), (17, 2, 264), (33, 3, 64), (129, 3, 136), (300, 2, 1000)], [4, 2, 3]))
CONV += [((67, 3, 24), w) for w in (1, 5, 6, 7, 8)]


@pytest.mark.parametrize("shape,width", CONV)
@pytest.mark.parametrize("dtype,pad,state,layout,silu", [(F16, None, False, None, True), (BF16, "right", True, "slice", True),
                                                         (F32, "left", True, "odd", True), (F16, "mixed", True, "batch first", False)])
def test_convolution(dev, shape, width, dtype, pad, state, layout, silu):
    T, B, D = shape
    gen = torch.Generator().manual_seed(T * 100 + D + width)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    mask = padding(B, T, pad, gen)
    x, g, w, bias = poison(draw(T, B, D), mask), poison(draw(T, B, D), mask), draw(D, width), draw(D) if state else None
    s, gs = (draw(B, width - 1, D), draw(B, width - 1, D)) if state else (None, None)
    args = [None if t is None else t.double() for t in (clean(x, mask), w, bias, s)]
    more = [None if t is None else t.double() for t in (clean(g, mask), gs)]
    want, size = (O.conv(*args, mask, silu, *more, absolute=a) for a in (False, True))

    xd, wd, bd, sd = leaves(strided(x, layout, dev), *(None if t is None else t.to(dev) for t in (w, bias, s)))
    md = None if mask is None else mask.to(dev)
    act = "silu" if silu else None
    if state:
        y, out = ss.incremental_causal_conv(x=xd, weight=wd, bias=bd, state=sd, activation=act, key_padding_mask=md)
        assert torch.equal(out.cpu().double(), want["state"]) and out.dtype == dtype
        ins = [t for t in (xd, wd, bd, sd) if t.numel()]
        grads = torch.autograd.grad([y, out], ins, [strided(g, layout, dev), gs.to(dev)], allow_unused=True)
        names = [n for n, t in zip(("gx", "gweight", "gbias", "gstate"), (xd, wd, bd, sd)) if t.numel()]
        with torch.no_grad():                                     # the state updated in place gives the same bits
            kept = s.to(dev)
            y2, out2 = ss.incremental_causal_conv(x=xd, weight=wd, bias=bd, state=kept, activation=act, key_padding_mask=md)
            assert out2 is kept and torch.equal(out2, out) and torch.equal(y2, y)
    else:
        y = ss.causal_conv(x=xd, weight=wd, bias=bd, activation=act, key_padding_mask=md)
        grads, names = torch.autograd.grad(y, [xd, wd], strided(g, layout, dev)), ("gx", "gweight")
    near(y, want["y"], size["y"], 2.0 ** -19, "y")
    for n, t in zip(names, grads):
        assert t.dtype == dtype
        near(t, want[n], size[n], 2.0 ** (-17 if n in ("gweight", "gbias") else -19), n)


def test_convolution_of_one_long_row_of_padding(dev):
    """The window in front of a run lies thousands of padded tokens back."""
    T, D = 9000, 8
    x, w = torch.randn(T, 1, D, device=dev), torch.randn(D, 4, device=dev)
    mask = torch.ones(1, T, dtype=torch.bool, device=dev)
    there = [0, 1, 2, 5, 8000, 8990, 8999]
    mask[0, there] = False
    y, state = ss.incremental_causal_conv(x=x, weight=w, key_padding_mask=mask)
    assert torch.equal(y[there], ss.causal_conv(x=x[there], weight=w))
    assert torch.equal(state[0], x[there[-3:], 0]) and int(y.ne(0).any(-1).sum()) == len(there)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", range(1, 9))
def test_convolution_parameters_anywhere_in_a_flat_buffer(dev, width, dtype):
    """Weights and biases are taken at any element's address, forward, backward and one token, with the bits of aligned ones."""
    T, B, D = 37, 2, 136
    gen = torch.Generator().manual_seed(width)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(dev)
    x, g, w, b, s = draw(T, B, D).requires_grad_(), draw(T, B, D), draw(D, width), draw(D), draw(B, width - 1, D)
    flat = lambda t, at: torch.cat([t.new_zeros(at), t.flatten()])[at:].view(t.shape).detach().requires_grad_()
    want = None
    for at in (0, 1, 2, 3, 4, 6, 8):
        wd, bd = flat(w, at), flat(b, at)
        assert wd.is_contiguous() and wd.data_ptr() % 16 == at * wd.element_size() % 16
        y = ss.causal_conv(x=x, weight=wd, bias=bd)
        got = [y, *torch.autograd.grad(y, [x, wd, bd], g)]
        with torch.no_grad():
            one, held = ss.incremental_causal_conv(x=x[:1], weight=wd, bias=bd, state=s.clone())
        got += [one, held]
        want = want or got
        assert all(torch.equal(a, c) for a, c in zip(got, want)), at


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("width", [2, 3, 4, 8])
def test_a_kept_window_is_updated_in_place_token_by_token(dev, width, dtype):
    """Every CTA reads the window that it writes: the same bits as from one buffer into another, some tokens padded."""
    B, D = 37, 1028
    gen = torch.Generator().manual_seed(width)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(dev)
    x, w, b, s = draw(9, B, D), draw(D, width), draw(D), draw(B, width - 1, D)
    mask = (torch.rand(9, B, 1, generator=gen) < 0.3).to(dev)
    held, apart = s.clone(), s
    for t in range(9):
        y, same = ss.incremental_causal_conv(x=x[t:t + 1], weight=w, bias=b, state=held, key_padding_mask=mask[t])
        want, apart = ops.causal_conv_fwd(x[t:t + 1], w, b, apart, mask[t], True, True)
        assert same is held and torch.equal(y, want) and torch.equal(held, apart)


# --------------------------------------------------------------------------- selective scan
SCAN = [(1, 1, 1, 1, 1), (1, 3, 8, 16, 1), (2, 2, 6, 3, 2), (15, 2, 64, 16, 1), (16, 3, 40, 4, 1), (17, 1, 72, 8, 1), (33, 2, 130, 12, 1), (48, 1, 136, 17, 2),
        (65, 2, 36, 32, 4), (80, 2, 24, 33, 1), (70, 1, 16, 64, 1), (150, 3, 264, 16, 1), (531, 1, 48, 16, 2), (700, 1, 20, 64, 1)]


def scan_inputs(shape, dtype, gen, layout=None, dev="cpu"):
    T, B, D, N, G = shape
    draw = lambda *s: torch.randn(*s, generator=gen)
    step = torch.exp(torch.rand(D, generator=gen) * 4.6 - 6.9)
    ins = dict(x=draw(T, B, D).to(dtype), dt=(0.5 * draw(T, B, D)).to(dtype),
               a=-(torch.arange(1, N + 1).float() * torch.exp(0.1 * draw(D, N))), b=draw(T, B, G, N).to(dtype), c=draw(T, B, G, N).to(dtype), d=draw(D),
               dt_bias=step + torch.log(-torch.expm1(-step)), s=draw(B, D, N))
    return ins, draw(T, B, D).to(dtype), draw(B, D, N)


def scan_check(dev, shape, dtype, pad, layout, softplus=True, optional=True, state=True):
    T, B, D, N, G = shape
    gen = torch.Generator().manual_seed(T * 1000 + D + N)
    ins, g, gs = scan_inputs(shape, dtype, gen)
    if not softplus:
        ins["dt"] = ins["dt"].abs() / 8
        ins["dt_bias"] = ins["dt_bias"].abs() / 64
    if not optional:
        ins["d"] = ins["dt_bias"] = None
    if not state:
        ins["s"] = gs = None
    mask = padding(B, T, pad, gen)
    for n in ("x", "dt", "b", "c"):
        poison(ins[n], mask)
    poison(g, mask)
    seq = ("x", "dt", "b", "c")
    args = [None if t is None else (clean(t, mask) if n in seq else t).double() for n, t in ins.items()]
    more = [clean(g, mask).double(), None if gs is None else gs.double()]
    want, size = (O.scan(*args, mask, softplus, *more, absolute=a) for a in (False, True))

    on = {n: None if t is None else strided(t, layout, dev) if n in seq else t.to(dev) for n, t in ins.items()}
    on = dict(zip(on, leaves(*on.values())))
    md = None if mask is None else mask.to(dev)
    names = dict(x="gx", dt="gdt", a="ga", b="gb", c="gc", d="gd", dt_bias="gbias", s="gs")
    diff = [n for n in names if on[n] is not None]
    if state:
        y, out = ss.incremental_selective_scan(**on, dt_softplus=softplus, key_padding_mask=md)
        grads = torch.autograd.grad([y, out], [on[n] for n in diff], [strided(g, layout, dev), gs.to(dev)])
        with torch.no_grad():
            kept = ins["s"].to(dev)
            y2, out2 = ss.incremental_selective_scan(**{**on, "s": kept}, dt_softplus=softplus, key_padding_mask=md)
            assert out2 is kept
        for got in (out, out2):
            near(got, want["s"], size["s"], (8 * T + 16) * 2.0 ** -24, "s")
        near(y2, want["y"], size["y"], (8 * T + 16 + 2 * N) * 2.0 ** -24, "y in place")
    else:
        rest = {n: t for n, t in on.items() if n != "s"}
        y = ss.selective_scan(**rest, dt_softplus=softplus, key_padding_mask=md)
        grads = torch.autograd.grad(y, [on[n] for n in diff], strided(g, layout, dev))
    near(y, want["y"], size["y"], (8 * T + 16 + 2 * N) * 2.0 ** -24, "y")
    for n, t in zip(diff, grads):
        assert t.dtype == on[n].dtype
        near(t, want[names[n]], size[names[n]], (20 * T + 64 + B + D + 2 * N) * 2.0 ** -24, names[n])


@pytest.mark.parametrize("shape", SCAN)
@pytest.mark.parametrize("dtype,pad,layout", [(F16, None, None), (BF16, "right", "slice"), (F32, "left", "odd"), (F32, "mixed", "batch first")])
def test_scan(dev, shape, dtype, pad, layout):
    scan_check(dev, shape, dtype, pad, layout)


@pytest.mark.parametrize("shape", [(531, 1, 48, 8, 1), (400, 2, 130, 4, 2), (197, 1, 16, 1, 1), (641, 1, 24, 6, 3), (531, 1, 48, 32, 1), (400, 2, 30, 24, 2),
                                   (325, 1, 20, 17, 1)])
@pytest.mark.parametrize("dtype,pad,layout", [(F16, None, None), (BF16, "right", "slice"), (F32, "mixed", "odd"), (F32, "left", "batch first")])
def test_scan_in_segments(dev, shape, dtype, pad, layout):
    """Few rows: several segments with a ragged last tile, for up to 8 states (backward tiles of 8 tokens) and for 17 to 32."""
    scan_check(dev, shape, dtype, pad, layout)


@pytest.mark.parametrize("softplus,optional,state", [(False, True, True), (True, False, True), (True, True, False), (False, False, False)])
@pytest.mark.parametrize("shape", [(1, 2, 24, 16, 1), (40, 2, 24, 16, 1)])
def test_scan_without_its_optional_parts(dev, shape, softplus, optional, state):
    scan_check(dev, shape, F32, None, None, softplus, optional, state)
    scan_check(dev, shape, BF16, "mixed", "slice", softplus, optional, state)


@pytest.mark.parametrize("N", [4, 16, 24])
def test_scan_of_states_that_grow(dev, N):
    """exp(delta a) is e at every token, 1000 of them: a state that is zero until the last 20, and a gradient until the first 20, stays
    finite, although growth over a whole segment does not; so does one that begins at 1e-36."""
    T, B, D = 1000, 1, 10
    gen = torch.Generator().manual_seed(N)
    draw = lambda *s: torch.randn(*s, generator=gen)
    ins = dict(x=draw(T, B, D), dt=torch.ones(T, B, D), a=torch.ones(D, N), b=draw(T, B, 1, N), c=draw(T, B, 1, N), d=draw(D), dt_bias=torch.zeros(D),
               s=torch.zeros(B, D, N))
    ins["x"][:980] = 0
    g, gs = draw(T, B, D), torch.zeros(B, D, N)
    g[20:] = 0
    want, size = (O.scan(*[t.double() for t in ins.values()], None, False, g.double(), gs.double(), absolute=a) for a in (False, True))
    on = dict(zip(ins, leaves(*[t.to(dev) for t in ins.values()])))
    y, s = ss.incremental_selective_scan(**on, dt_softplus=False)
    names = ("gx", "gdt", "ga", "gb", "gc", "gd", "gbias", "gs")
    got = dict(zip(names, torch.autograd.grad([y, s], list(on.values()), [g.to(dev), gs.to(dev)])), y=y, s=s)
    for n, t in got.items():
        # growth by up to 20 tokens in front of what is compared: their roundings, relative, as in a chain that decays
        near(t, want[n], size[n], (20 * T + 64 + B + D + 2 * N) * 2.0 ** -24, n)
    # 1e-36 e^160: two segments, the growth over the first of which (e^89.6) overflows by itself
    cut = {n: t[:200] if n in ("x", "dt", "b", "c") else t for n, t in ins.items()}
    cut.update(x=torch.zeros(200, B, D), dt=torch.full((200, B, D), 0.8), s=torch.full((B, D, N), 1e-36), d=torch.zeros(D))
    want, size = (O.scan(*[t.double() for t in cut.values()], None, False, absolute=a) for a in (False, True))
    y, s = ss.incremental_selective_scan(**{n: t.to(dev) for n, t in cut.items()}, dt_softplus=False)
    for n, t in dict(y=y, s=s).items():
        near(t, want[n], size[n], (20 * 200 + 16 + 2 * N) * 2.0 ** -24, n)


@pytest.mark.parametrize("N", [3, 16, 40])
def test_a_token_whose_growth_overflows_leaves_inf(dev, N):
    """exp(88.5) is the last power that is finite; exp(100), of every state, is inf of the state's sign, and zero stays what is added."""
    x, bc = torch.ones(1, 2, 6, device=dev), torch.zeros(1, 2, 1, N, device=dev)
    s = torch.ones(2, 6, N, device=dev)
    s[1] = -1
    for power, want in ((88.5, float(torch.tensor(88.5, dtype=torch.float64).exp())), (100.0, float("inf")), (1e30, float("inf"))):
        _, held = ss.incremental_selective_scan(x=x, dt=x * power, a=torch.ones(6, N, device=dev), b=bc, c=bc, s=s.clone(), dt_softplus=False)
        # 88.5 log2(e) = 127.7 is rounded by 2^-18 (2.6e-6 of the power), log2(e) by 1.3e-8 (1.2e-6), the power by 2^-22: below 5e-6
        assert torch.allclose(held, s * want, rtol=5e-6, atol=0)


@pytest.mark.parametrize("cut", [1, 16, 100, 299])
def test_scan_in_two_calls(dev, cut):
    """A prompt in two calls is the prompt in one, whichever way either is cut into segments."""
    gen = torch.Generator().manual_seed(cut)
    ins, _, _ = scan_inputs((300, 2, 72, 16, 1), F32, gen)
    on = {n: t.to(dev) for n, t in ins.items() if n != "s"}
    y, s = ss.incremental_selective_scan(**on)
    part = lambda lo, hi: {n: t[lo:hi] if n in ("x", "dt", "b", "c") else t for n, t in on.items()}
    y1, held = ss.incremental_selective_scan(**part(0, cut))
    y2, same = ss.incremental_selective_scan(**part(cut, 300), s=held)
    assert same is held
    for a, b in ((torch.cat([y1, y2]), y), (held, s)):
        assert (a - b).norm() <= 1e-6 * b.norm()


def test_scan_with_more_rows_than_the_gpu_takes_side_by_side(dev):
    """128 CTAs: the forward in one segment, the backward in two, whose summaries join."""
    scan_check(dev, (230, 2, 4096, 16, 1), F32, "right", None)


def test_scan_keeps_fp32_over_long_sequences(dev):
    """Random errors of a chain of n steps grow as sqrt(n) half steps of 2^-24: a state's memory is at most 1000 tokens here (steps of 0.001), sums
    over tokens are chains of T / 16 tiles.  With the special function unit's 2^-22, whose sign does not change, 2^-19 of the norm in
    all; sums that keep fp32's precision are well below it, a chain of 4096 roundings to 16 bits is 2^-6."""
    T, B, D, N = 4096, 1, 40, 16
    gen = torch.Generator().manual_seed(9)
    ins, g, gs = scan_inputs((T, B, D, N, 1), F32, gen)
    want = O.scan(*[t.double() for t in ins.values()], None, True, g.double(), gs.double())
    on = dict(zip(ins, leaves(*[t.to(dev) for t in ins.values()])))
    y, s = ss.incremental_selective_scan(**on)
    got = dict(zip(("gx", "gdt", "ga", "gb", "gc", "gd", "gbias", "gs"), torch.autograd.grad([y, s], list(on.values()), [g.to(dev), gs.to(dev)])), y=y, s=s)
    for n, t in got.items():
        assert (t.detach().cpu().double() - want[n]).norm() <= 2.0 ** -19 * want[n].norm(), n


@pytest.mark.parametrize("steps", ["constant", "varied"])
@pytest.mark.parametrize("N", [8, 16, 32])
def test_scan_keeps_fp32_token_by_token(dev, N, steps):
    """4096 calls of one token each, the state carried through them, for states that remember 1000 tokens.

    Varied steps: each token's roundings are others, so that they add up as in one call over the tokens (2^-19 of the norm, above); so
    does not what has one sign.  Of the slowest state, the error along the state itself: the polynomial near 1 is off by 2.3e-7 |r|,
    |r| <= 0.002, 1000 times, the step size by 5e-7 both in the decays and in what is added: 1.5e-6 < 2^-19 (an error of -5e-9 a decay, as
    the special function unit's there, would be 5e-6).
    Constant steps: a decay just below 1 is rounded the same way every time, by up to 2^-25, so that what came k tokens ago is off by
    k 2^-25 of itself.  That is 1000 2^-25 of what the tokens brought, but k = T = 4096 for the initial state, and exp(-4.1) of its 1 is as
    much as the tokens' sqrt(0.001 / 2): up to T 2^-25 = 2^-13 of the norm."""
    T, B, D = 4096, 2, 40
    gen = torch.Generator().manual_seed(N)
    ins, _, _ = scan_inputs((T, B, D, N, 1), F32, gen)
    if steps == "constant":
        ins["dt"].zero_()
    ins["dt_bias"] = torch.full((D,), -6.9073)                    # softplus of it is 0.001
    want = O.scan(*[t.double() for t in ins.values()], None, True)
    on = {n: t.to(dev) for n, t in ins.items()}
    held, ys = on["s"], []
    for t in range(T):
        y, held = ss.incremental_selective_scan(**{**on, **{n: on[n][t:t + 1] for n in ("x", "dt", "b", "c")}, "s": held})
        ys.append(y)
    bound = 2.0 ** (-13 if steps == "constant" else -19)
    for n, got in dict(y=torch.cat(ys), s=held).items():
        off = float((got.cpu().double() - want[n]).norm() / want[n].norm())
        assert off <= bound, (n, off)
    slow, true = held[..., 0].cpu().double(), want["s"][..., 0]
    along = float(((slow - true) * true).sum() / true.square().sum())
    assert abs(along) <= bound, along


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_scan_keeps_non_finite_values_where_they_belong(dev, value):
    """One token of one channel's x: its channel from that token on, its group's b and c gradients; nothing else."""
    ins, _, _ = scan_inputs((40, 2, 72, 16, 1), F32, torch.Generator().manual_seed(0))
    on = {n: t.to(dev) for n, t in ins.items() if n != "s"}
    clean_y = ss.selective_scan(**on)
    on["x"][20, 1, 5] = value
    y = ss.selective_scan(**on)
    hit = torch.zeros_like(y, dtype=torch.bool)
    hit[20:, 1, 5] = True
    assert not y[20:, 1, 5].isfinite().any() and torch.equal(y[~hit], clean_y[~hit])


# --------------------------------------------------------------------------- group norm
NORM = [((1,), 1, 1), ((3, 2), 4, 2), ((5,), 7, 1), ((2, 3), 24, 3), ((1, 9), 64, 1), ((33,), 200, 5), ((130, 3), 1024, 16), ((7,), 300, 100), ((40,), 1000, 1),
        ((5, 2), 2048, 1), ((3,), 5000, 1), ((2,), 12000, 1), ((3,), 16384, 1), ((2,), 16383, 1), ((1500,), 40, 1), ((2,), 4096, 1), ((257,), 513, 3)]


@pytest.mark.parametrize("lead,C,groups", NORM)
@pytest.mark.parametrize("dtype,gated,weights,layout,silu", [(F16, True, True, None, True), (BF16, True, True, "slice", True), (F32, False, True, "odd", True),
                                                             (F32, True, False, "slice", False), (F16, False, False, None, False)])
def test_norm(dev, lead, C, groups, dtype, gated, weights, layout, silu):
    gen = torch.Generator().manual_seed(C + groups)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    x, g, w, bias, gate = 2 * draw(*lead, C) + 1, draw(*lead, C), draw(C) if weights else None, draw(C) if weights else None, draw(*lead, C) if gated else None
    x.view(-1, C)[0] = 3.0                                        # a row without variance
    args = [None if t is None else t.double() for t in (w, bias, gate)]
    want, size = (O.norm(x.double(), groups, *args, silu, 1e-5, g.double(), absolute=a) for a in (False, True))
    put = lambda t: None if t is None else strided(t, layout, dev)
    xd, wd, bd, zd = leaves(put(x), *(None if t is None else t.to(dev) for t in (w, bias)), put(gate))
    y = ss.group_norm(x=xd, num_groups=groups, weight=wd, bias=bd, gate=zd, activation="silu" if silu else None)
    near(y, want["y"], size["y"], 2.0 ** -18, "y")
    pairs = [(n, t) for n, t in zip(("gx", "gweight", "gbias", "ggate"), (xd, wd, bd, zd)) if t is not None]
    rows = x.numel() // C
    for (n, t), got in zip(pairs, torch.autograd.grad(y, [t for _, t in pairs], put(g))):
        assert got.dtype == dtype and got.shape == t.shape
        near(got, want[n], size[n], 2.0 ** -18 + (rows * 2.0 ** -24 if n in ("gweight", "gbias") else 0), n)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("gated,silu", [(True, True), (False, True), (False, False)])
@pytest.mark.parametrize("rows,C,groups", [(1, 8, 1), (5, 24, 3), (131, 64, 1), (77, 1024, 16), (3, 300, 1)])
def test_norm_without_an_eps(dev, rows, C, groups, gated, silu, dtype):
    """A CTA's rows are more than there are: what it walks beyond them has no variance, and leaves the weights' gradients alone."""
    gen = torch.Generator().manual_seed(rows)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype)
    x, g, w, bias, gate = draw(rows, C), draw(rows, C), draw(C), draw(C), draw(rows, C) if gated else None
    args = [None if t is None else t.double() for t in (w, bias, gate)]
    want, size = (O.norm(x.double(), groups, *args, silu, 0.0, g.double(), absolute=a) for a in (False, True))
    xd, wd, bd, zd = leaves(*(None if t is None else t.to(dev) for t in (x, w, bias, gate)))
    y = ss.group_norm(x=xd, num_groups=groups, weight=wd, bias=bd, gate=zd, activation="silu" if silu else None, eps=0.0)
    near(y, want["y"], size["y"], 2.0 ** -18, "y")
    pairs = [(n, t) for n, t in zip(("gx", "gweight", "gbias", "ggate"), (xd, wd, bd, zd)) if t is not None]
    for (n, t), got in zip(pairs, torch.autograd.grad(y, [t for _, t in pairs], g.to(dev))):
        near(got, want[n], size[n], 2.0 ** -18 + (rows * 2.0 ** -24 if n in ("gweight", "gbias") else 0), n)


# --------------------------------------------------------------------------- what goes for all of them
def calls(dev, dtype=F16, T=20, B=3, D=64, N=16):
    """Each operator's call on fresh inputs: (function of the tensors, tensors)."""
    gen = torch.Generator().manual_seed(1)
    draw = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(dev)
    ins, _, _ = scan_inputs((T, B, D, N, 1), dtype, gen)
    names = [n for n in ins if n != "s"]
    return {"conv": (lambda x, w, b: ss.causal_conv(x=x, weight=w, bias=b), [draw(T, B, D), draw(D, 4), draw(D)]),
            "scan": (lambda *t: ss.selective_scan(**dict(zip(names, t))), [ins[n].to(dev) for n in names]),
            "norm": (lambda x, w, b, z: ss.group_norm(x=x, num_groups=4, weight=w, bias=b, gate=z), [draw(T, B, D), draw(D), draw(D), draw(T, B, D)])}


KINDS = ["conv", "scan", "norm"]


@pytest.mark.parametrize("kind", KINDS)
def test_empty_calls(dev, kind):
    call, ts = calls(dev)[kind]
    for sizes in ((0, 3), (20, 0)):
        cut = [t[:sizes[0], :sizes[1]].detach().requires_grad_() if t.dim() >= 3 else t.detach().requires_grad_() for t in ts]
        y = call(*cut)
        assert y.shape == (*sizes, 64)
        for t, g in zip(cut, torch.autograd.grad(y, cut, torch.zeros_like(y))):
            assert g.shape == t.shape and not g.any()
    if kind == "norm":
        return
    s = torch.ones(3, 3, 64, device=dev).half() if kind == "conv" else torch.ones(3, 64, 16, device=dev)
    empty = [t[:0] if t.dim() >= 3 else t for t in ts]
    if kind == "conv":
        y, out = ss.incremental_causal_conv(x=empty[0], weight=empty[1], state=s)
    else:
        y, out = ss.incremental_selective_scan(**dict(zip(("x", "dt", "a", "b", "c"), empty)), s=s)
    assert out is s and bool((s == 1).all()) and y.shape == (0, 3, 64)


@pytest.mark.parametrize("kind", KINDS)
def test_a_backward_pass_is_the_same_twice_and_against_differences(dev, kind):
    call, ts = calls(dev, F32, T=37)[kind]
    ts = [t.requires_grad_() for t in ts]
    g = torch.randn(ts[0].shape, generator=torch.Generator().manual_seed(3)).to(dev)
    first, second = (torch.autograd.grad(call(*ts), ts, g) for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    # along a direction v: (f(t + h v) - f(t - h v)) / 2h, h = 2^-6: fp32 results off by 2^-24 sqrt(n) |terms| / h, third derivatives h^2
    for i, t in enumerate(ts):
        v = torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(dev)
        v /= v.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            up, down = (call(*[t + s * h * v if k == i else u for k, u in enumerate(ts)]).double() for s in (1, -1))
        slope, mine = float(((up - down) * g.double()).sum() / (2 * h)), float((first[i].double() * v.double()).sum())
        assert abs(slope - mine) <= 2e-3 * float(first[i].norm()) + 1e-3


@pytest.mark.parametrize("kind", KINDS)
def test_other_streams_and_repeated_graphs(dev, kind):
    """A call on a side stream, forward and backward; a captured forward replayed on new inputs beside another graph of the same sizes."""
    call, ts = calls(dev)[kind]
    ts = [t.requires_grad_() for t in ts]
    g = torch.ones_like(ts[0])
    want = [call(*ts)]
    want += torch.autograd.grad(want[0], ts, g)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [call(*ts)]
        got += torch.autograd.grad(got[0], ts, g)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        held = [[t.detach().clone() for t in ts] for _ in range(2)]
        graphs, outs = [torch.cuda.CUDAGraph() for _ in held], []
        torch.cuda.synchronize()
        for graph, tensors in zip(graphs, held):
            with torch.cuda.graph(graph):
                outs.append(call(*tensors))
        held[1][0].copy_(held[1][0].flip(0))
        for _ in range(2):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for out, tensors in zip(outs, held):
            assert torch.equal(out, call(*tensors))


def test_a_long_scan_captured_twice_has_workspaces_of_its_own(dev):
    """Segments' states go through a workspace: two graphs that run at once on two streams do not share it."""
    runs = []
    for seed in range(2):
        ins, _, _ = scan_inputs((2000, 1, 64, 16, 1), F16, torch.Generator().manual_seed(seed))
        runs.append({n: t.to(dev) for n, t in ins.items() if n != "s"})
    want = [ss.selective_scan(**r) for r in runs]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for r in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ss.selective_scan(**r))
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("kind", KINDS)
def test_expanded_inputs_and_gradients(dev, kind):
    """Inputs broadcast over the batch: read with stride 0, their gradients summed by autograd."""
    call, ts = calls(dev, F32)[kind]
    base = [t[:, :1].detach().clone().requires_grad_() if t.dim() >= 3 else t.detach().requires_grad_() for t in ts]
    wide = [t.expand(t.shape[0], 3, *t.shape[2:]) if t.dim() >= 3 else t for t in base]
    y = call(*wide)
    assert torch.equal(y[:, 0], y[:, 2])
    got = torch.autograd.grad(y.sum(), base)
    whole = [t.detach().contiguous().requires_grad_() for t in wide]
    want = torch.autograd.grad(call(*whole).sum(), whole)
    for a, b, t in zip(got, want, base):
        b = b.sum(1, keepdim=True) if t.dim() >= 3 else b
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5 * float(b.abs().max()))


@pytest.mark.parametrize("kind", KINDS)
def test_what_is_refused(dev, kind):
    call, ts = calls(dev)[kind]
    with pytest.raises(TypeError, match="one dtype"):
        call(ts[0].float(), *ts[1:])
    with pytest.raises(TypeError, match="unsupported dtype"):
        call(*[t.double() for t in ts])
    with pytest.raises(RuntimeError, match="expected all tensors on|no CPU path"):
        call(ts[0], *[t.cpu() for t in ts[1:]])
    with pytest.raises(AssertionError, match="expected"):
        call(ts[0], ts[1][1:], *ts[2:])
    t = [u.detach().requires_grad_() for u in ts]
    y = call(*t)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), t, create_graph=True)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(fw.make_dual(ts[0], torch.ones_like(ts[0])), *ts[1:])
    y = call(*t)
    with torch.no_grad():
        t[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_states_that_cannot_be_updated_in_place_are_refused(dev):
    _, (x, w, _) = calls(dev)["conv"]
    with pytest.raises(ValueError, match="contiguous"):
        ss.incremental_causal_conv(x=x, weight=w, state=torch.zeros(3, 64, 3, device=dev).half().transpose(1, 2))
    with pytest.raises(AssertionError, match="state"):
        ss.incremental_causal_conv(x=x, weight=w, state=torch.zeros(3, 4, 64, device=dev).half())
    with pytest.raises(ValueError, match="window"):
        ss.causal_conv(x=x, weight=torch.zeros(64, 9, device=dev).half())
    _, ts = calls(dev)["scan"]
    args = dict(zip(("x", "dt", "a", "b", "c"), ts))
    with pytest.raises(ValueError, match="contiguous"):
        ss.incremental_selective_scan(**args, s=torch.zeros(3, 16, 64, device=dev).transpose(1, 2))
    with pytest.raises(TypeError, match="fp32"):
        ss.incremental_selective_scan(**args, s=torch.zeros(3, 64, 16, device=dev).half())
    with pytest.raises(TypeError, match="fp32"):
        ss.selective_scan(**{**args, "a": ts[2].half()})
    with pytest.raises(ValueError, match="states per channel"):
        big = torch.zeros(20, 3, 1, 65, device=dev).half()
        ss.selective_scan(**{**args, "a": torch.zeros(64, 65, device=dev), "b": big, "c": big})
    with pytest.raises(ValueError, match="groups"):
        ss.selective_scan(**{**args, "b": ts[3].repeat(1, 1, 3, 1), "c": ts[4].repeat(1, 1, 3, 1)})
    with pytest.raises(AssertionError, match="key_padding_mask"):
        ss.selective_scan(**args, key_padding_mask=torch.zeros(20, 3, device=dev))
    with pytest.raises(ValueError, match="groups"):
        ss.group_norm(x=x, num_groups=3)


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_a_state_that_a_graph_keeps_is_not_overwritten_unnoticed(dev, kind, T):
    _, ts = calls(dev, F32, T=T)[kind]
    if kind == "conv":
        s = torch.randn(3, 3, 64, device=dev)
        call = lambda: ss.incremental_causal_conv(x=ts[0], weight=ts[1], state=s)
    else:
        s = torch.randn(3, 64, 16, device=dev)
        call = lambda: ss.incremental_selective_scan(**dict(zip(("x", "dt", "a", "b", "c"), ts)), s=s)
    ts[0].requires_grad_()
    y, new = call()
    assert new is not s
    with torch.no_grad():
        assert call()[1] is s
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_gradients_of_one_result_alone(dev, kind):
    """Of y alone and of the state alone; together they are the sum."""
    _, ts = calls(dev, F32)[kind]
    ts = [t.requires_grad_() for t in ts]
    if kind == "conv":
        y, s = ss.incremental_causal_conv(x=ts[0], weight=ts[1], bias=ts[2])
    else:
        y, s = ss.incremental_selective_scan(**dict(zip(("x", "dt", "a", "b", "c", "d", "dt_bias"), ts)))
    one, two, both = (torch.autograd.grad(sum(t.sum() for t in of), ts, retain_graph=True, allow_unused=True) for of in ((y,), (s,), (y, s)))
    for a, b, c in zip(one, two, both):
        assert (a + (0 if b is None else b) - c).norm() <= 1e-5 * c.norm()


def test_a_state_at_an_odd_address_is_updated_in_place(dev):
    _, ts = calls(dev, T=1)["scan"]
    args = dict(zip(("x", "dt", "a", "b", "c", "d", "dt_bias"), ts))
    s = torch.randn(3 * 64 * 16 + 1, device=dev)
    odd, plain = s[1:].view(3, 64, 16), s[1:].view(3, 64, 16).clone()
    y, same = ss.incremental_selective_scan(**args, s=odd)
    y2, _ = ss.incremental_selective_scan(**args, s=plain)
    assert same is odd and torch.equal(odd, plain) and torch.equal(y, y2)


# --------------------------------------------------------------------------- the layer, a run of them together
def layer(dev, dtype, **more):
    torch.manual_seed(0)
    return SelectiveStateSpace(embed_dim=96, state_dim=12, **more).to(dev).to(dtype)


def layer_oracle(m, x, mask):
    """The layer's forward from the oracle's functions, fp64 on the CPU."""
    p = {n: t.detach().double().cpu() for n, t in m.named_parameters()}
    u, gate = (x @ p["in_proj.weight"].t()).chunk(2, -1)
    u = O.conv(clean(u, mask), p["conv_weight"], p["conv_bias"], None, mask, True)["y"]
    n, g = m.state_dim, m.num_groups
    low, b, c = (u @ p["x_proj.weight"].t()).split([m.dt_rank, g * n, g * n], -1)
    y = O.scan(u, low @ p["dt_proj.weight"].t(), -torch.exp(p["a_log"]), b.unflatten(-1, (g, n)), c.unflatten(-1, (g, n)), p["d"], p["dt_bias"], None, mask,
               True)["y"]
    y = O.norm(y, m.norm_groups, p["norm_weight"], p["norm_bias"], gate, True, 1e-5)["y"]
    return y @ p["out_proj.weight"].t() + p["out_proj.bias"]


@pytest.mark.parametrize("pad", [None, "right", "left"])
@pytest.mark.parametrize("more", [{}, dict(num_groups=2, norm_groups=4, conv_width=3)])
def test_layer(dev, pad, more):
    """fp32: a dozen operators of fp32 precision and TF32-free products one after another, 1e-5 of the norm."""
    m = layer(dev, F32, **more)
    gen = torch.Generator().manual_seed(5)
    x, mask = torch.randn(45, 3, 96, generator=gen), padding(3, 45, pad, gen)
    y = m(x.to(dev), key_padding_mask=None if mask is None else mask.to(dev))
    want = layer_oracle(m, x.double(), mask)
    there = torch.ones(45, 3, dtype=torch.bool) if mask is None else ~mask.t()
    assert (y.cpu().double() - want)[there].norm() <= 1e-5 * want[there].norm()
    g = torch.randn(45, 3, 96, generator=gen).to(dev) * there[..., None].to(dev)
    xs = x.to(dev).requires_grad_()
    m(xs, key_padding_mask=None if mask is None else mask.to(dev)).backward(g)
    v = torch.randn(45, 3, 96, generator=gen).double()
    h = 2.0 ** -12                                                # differences of the oracle: its third derivative times h^2
    slope = ((layer_oracle(m, x.double() + h * v, mask) - layer_oracle(m, x.double() - h * v, mask)) * g.cpu().double()).sum() / (2 * h)
    mine = (xs.grad.cpu().double() * v).sum()
    assert abs(slope - mine) <= 1e-4 * float(xs.grad.norm()) * float(v.norm()) / 45 + 1e-4 * abs(float(slope))
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())


@pytest.mark.parametrize("dtype,tol", [(F32, 1e-5), (F16, 1e-2), (BF16, 8e-2)])
def test_layer_prompt_then_tokens(dev, dtype, tol):
    """A padded prompt and then single tokens with the kept state, a reordered batch on the way, is the whole sequence at once.  Products
    of other shapes round differently: a few steps of the type through seven roundings (2^-9, 2^-6), relative to the norm."""
    m = layer(dev, dtype).requires_grad_(False)
    gen = torch.Generator().manual_seed(2)
    T, P, B = 30, 19, 3
    x = torch.randn(T, B, 96, generator=gen).to(dtype).to(dev)
    mask = torch.zeros(B, P, dtype=torch.bool, device=dev)
    mask[0, 11:], mask[2, 1:] = True, True
    state = {}
    m(x[:P], key_padding_mask=mask, saved_state=state)
    order = torch.tensor([2, 0, 1])
    m.reorder_incremental_state(state, order)
    steps = torch.cat([m(x[t:t + 1], saved_state=state) for t in range(P, T)])
    for slot, row in enumerate(order.tolist()):
        alone = torch.cat([x[:P, row][~mask[row]], x[P:, slot]]).unsqueeze(1)
        want = m(alone)[-(T - P):, 0]
        assert (steps[:, slot] - want).float().norm() <= tol * want.float().norm()


def test_layer_under_autocast_and_with_gradients_through_its_state(dev):
    m = layer(dev, F32)
    x = torch.randn(6, 2, 96, device=dev)
    with torch.autocast("cuda", dtype=BF16):
        y = m(x)
    assert y.dtype == BF16 and (y.float() - m(x)).norm() <= 0.08 * m(x).norm()
    xs = x.clone().requires_grad_()
    state = {}
    a = m(xs[:4], saved_state=state)
    first = dict(state)
    b = m(xs[4:], saved_state=state)
    assert state["prev_s"] is not first["prev_s"] and state["prev_s"].requires_grad
    got = torch.autograd.grad(torch.cat([a, b]).sum(), xs)[0]
    want = torch.autograd.grad(m(xs).sum(), xs)[0]
    assert (got - want).norm() <= 1e-5 * want.norm()


def test_layer_trains_inside_a_graph(dev):
    """A whole step with its backward captured after warm-up on a side stream, replayed twice, gives the eager gradients."""
    m, x = layer(dev, F16), torch.randn(33, 2, 96, device=dev).half()
    params = list(m.parameters())
    want = torch.autograd.grad(m(x).float().sum(), params)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.autograd.grad(m(x).float().sum(), params)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(m(x).float().sum(), params)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert (a - b).float().norm() <= 1e-2 * b.float().norm() + 1e-6


def test_the_python_node_gives_the_native_ones_results(dev):
    """Inside a dispatch mode the calls go through Python autograd functions."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    for call, ts in calls(dev).values():
        ts = [t.requires_grad_() for t in ts]
        want = call(*ts)
        with Seen():
            got = call(*ts)
        assert torch.equal(got, want) and "Backward" in type(got.grad_fn).__name__
        for a, b in zip(torch.autograd.grad(got.sum(), ts), torch.autograd.grad(want.sum(), ts)):
            assert torch.equal(a, b)


def test_a_compiled_caller_runs(dev):
    for call, ts in calls(dev).values():
        want = call(*ts)
        assert torch.equal(torch.compile(lambda *a: call(*a) * 2, backend="eager")(*ts), want * 2)


def test_one_tensor_as_several_inputs(dev):
    """x as dt, b as c, x as its own gate: gradients add up as for separate tensors of the same values."""
    _, (x, dt, a, b, c, d, bias) = calls(dev, F32)["scan"]
    x, b = x.requires_grad_(), b.requires_grad_()
    f = lambda x1, x2, b1, b2: ss.selective_scan(x=x1, dt=x2, a=a, b=b1, c=b2, d=d, dt_bias=bias).square().sum() + \
        ss.group_norm(x=x1, num_groups=4, gate=x2).square().sum()
    got = torch.autograd.grad(f(x, x, b, b), [x, b])
    apart = [t.detach().clone().requires_grad_() for t in (x, x, b, b)]
    want = torch.autograd.grad(f(*apart), apart)
    assert torch.allclose(got[0], want[0] + want[1], rtol=1e-5, atol=1e-5) and torch.allclose(got[1], want[2] + want[3], rtol=1e-5, atol=1e-5)


def test_tensor_level_calls(dev):
    """``ops``: what is not asked for is None, and a state that is not updated in place is left alone."""
    _, (x, w, b) = calls(dev)["conv"]
    s = torch.ones(3, 3, 64, device=dev).half()
    y, out = ops.causal_conv_fwd(x, w, b, s, None, True, True)
    assert out is not s and bool((s == 1).all()) and torch.equal(out, x[-3:].transpose(0, 1))
    gx, gw, gb, gs = ops.causal_conv_bwd(x, w, b, s, None, True, y, None, False, False, False)
    assert gw is None and gb is None and gs is None and gx.shape == x.shape
    _, ts = calls(dev, T=1)["scan"]
    s = torch.ones(3, 64, 16, device=dev)
    y, out, kept = ops.selective_scan_fwd(*ts, s, return_state=True)
    assert kept is None and bool((s == 1).all()) and not torch.equal(out, s)
    with pytest.raises(ValueError, match="checkpoints"):
        ops.selective_scan_bwd(*ts, s, None, True, y, None, None, False)


def test_tensor_level_calls_refuse_gradients_of_other_shapes_and_devices(dev):
    """What autograd hands over fits by itself; a caller of ``ops`` may not: kernels would read beyond it."""
    _, (x, w, b) = calls(dev)["conv"]
    s = torch.ones(3, 3, 64, device=dev).half()
    conv = lambda g, g_state=None: ops.causal_conv_bwd(x, w, b, s, None, True, g, g_state, True, True, True)
    _, ts = calls(dev)["scan"]
    y, _, kept = ops.selective_scan_fwd(*ts, save=True)
    scan = lambda g, g_s=None, k=kept: ops.selective_scan_bwd(*ts, None, None, True, g, g_s, k, False)
    norm = lambda g: ops.group_norm_bwd(x, 4, b, b, None, True, 1e-5, g, True, True, False)
    for call in (conv, scan, norm):
        call(x)
        for g in (x[1:], x[:, :1], x[..., :32], x[0], x.flatten()):
            with pytest.raises(AssertionError, match="g is"):
                call(g)
        with pytest.raises(RuntimeError, match="expected all tensors on"):
            call(x.cpu())
    with pytest.raises(AssertionError, match="g_state is"):
        conv(x, s[:, 1:])
    with pytest.raises(RuntimeError, match="expected all tensors on"):
        conv(x, s.cpu())
    state = torch.zeros(3, 64, 16, device=dev)
    scan(x, state)
    with pytest.raises(AssertionError, match="g_s is"):
        scan(x, state[..., 1:])
    with pytest.raises(RuntimeError, match="expected all tensors on"):
        scan(x, state.cpu())
    for wrong in (None, kept[:-4], torch.cat([kept, kept])[::2], kept[:0]):
        with pytest.raises(ValueError, match="checkpoints"):
            scan(x, None, wrong)
    with pytest.raises(RuntimeError, match="expected all tensors on"):
        scan(x, None, kept.cpu())


def test_layer_decodes_inside_a_graph(dev):
    """One token's call with the kept state, captured once and replayed for every token, is the eager loop: the state is updated where it is."""
    m = layer(dev, F16).requires_grad_(False)
    x = torch.randn(12, 3, 96, generator=torch.Generator().manual_seed(4)).half().to(dev)
    eager, kept = {}, {}
    m(x[:5], saved_state=eager)
    m(x[:5], saved_state=kept)
    want = [m(x[t:t + 1], saved_state=eager) for t in range(5, 12)]
    one = x[5:6].clone()
    begin = {k: v.clone() for k, v in kept.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        m(one, saved_state=kept)                                  # warm-up
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = m(one, saved_state=kept)
    for k, v in begin.items():
        kept[k].copy_(v)
    for t, y in zip(range(5, 12), want):
        one.copy_(x[t:t + 1])
        graph.replay()
        # the matrix products may take another algorithm on another stream: a few steps of fp16 through seven roundings
        assert (out - y).float().norm() <= 1e-2 * y.float().norm()
    for k in begin:
        assert (kept[k] - eager[k]).float().norm() <= 1e-2 * eager[k].float().norm()


def test_a_state_in_place_of_several_tokens_inside_a_graph(dev):
    """The incremental forms over a few tokens, captured: each replay goes on from the state that the one before it left, with the eager bits."""
    _, (x, w, b) = calls(dev)["conv"]
    _, ts = calls(dev)["scan"]
    args = dict(zip(("x", "dt", "a", "b", "c", "d", "dt_bias"), ts))
    for T in (1, 20):
        xt = x[:T]
        cut = {k: v[:T] if v.dim() >= 3 else v for k, v in args.items()}
        held = torch.randn(3, 3, 64, device=dev).half(), torch.randn(3, 64, 16, device=dev)
        apart = [t.clone() for t in held]
        call = lambda s: (ss.incremental_causal_conv(x=xt, weight=w, bias=b, state=s[0]), ss.incremental_selective_scan(**cut, s=s[1]))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (y1, s1), (y2, s2) = call(held)
        assert s1 is held[0] and s2 is held[1] and all(torch.equal(a, c) for a, c in zip(held, apart))      # capture runs nothing
        for _ in range(3):
            graph.replay()
            (w1, _), (w2, _) = call(apart)
            assert all(torch.equal(a, c) for a, c in zip((y1, y2, *held), (w1, w2, *apart)))
