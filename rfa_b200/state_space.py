"""Selective state-space mixing, beside causal RFA: another causal layer whose running state has one size whatever the
sequence's length.  Functional forms and the ``SelectiveStateSpace`` layer, in the manner of ``causal_attention.py``:

* ``causal_conv``, ``incremental_causal_conv``      -> depthwise convolution over the last few tokens, with SiLU
* ``selective_scan``, ``incremental_selective_scan`` -> s_t = exp(delta_t a) s_(t-1) + delta_t b_t x_t, y_t = c_t . s_t + d x_t
* ``group_norm``                                    -> groups of a token's channels normalised, gated by silu(gate)

Activations are time-major, ``[tgt_len, bsz, channels]``, fp16, bf16 or fp32, with any strides as long as channels are
adjacent (views of a projection's output are taken as they are); sums and the scan's states are fp32.  At most 65535 sequences
and 2^24 channels a call.  The backward passes are not differentiable themselves.  No upstream counterpart.

``key_padding_mask`` ``[bsz, tgt_len]`` (1 = padding): padded tokens are skipped, wherever they stand -- every result is
what it would be without them, whatever values they hold, and their own outputs and gradients are zero.

The ``incremental_`` forms carry a state in and out, over any number of tokens.  As in ``incremental_rfa``, a state that is
passed in is UPDATED IN PLACE and returned when no gradient is being recorded; with autograd recording and an input that requires
grad the call is differentiable in all of them, returns a NEW state and leaves the one passed in alone."""
import math
from typing import Dict, Optional, Tuple

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable
from torch.nn import Parameter

from . import ops
from ._lib import native
from ._plain import plain_tensors
from .causal_attention import _underived


def _mask(mask: Optional[Tensor]) -> Optional[Tensor]:
    return None if mask is not None and mask.dim() == 0 else mask


def _silu(activation: Optional[str]) -> bool:
    if activation not in ("silu", None):
        raise ValueError(f"rfa_b200: activation is 'silu' or None, got {activation!r}")
    return activation == "silu"


# --------------------------------------------------------------------------- convolution
class _CausalConv(torch.autograd.Function):
    """(x, weight, bias or None, state or None, mask or None) -> y[, the outgoing state]."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, mask, silu, return_state):
        ctx.save_for_backward(x, weight, bias, state, mask)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        y, out = ops.causal_conv_fwd(x, weight, bias, state, mask, silu, return_state)
        return (y, out) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_state=None):
        x, weight, bias, state, mask = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = torch.zeros_like(x) if g is None else g
        gx, gw, gb, gs = ops.causal_conv_bwd(x, weight, bias, state, mask, ctx.silu, g, g_state, *need[1:4])
        return gx, gw, gb, gs, None, None, None


def causal_conv(*, x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = "silu",
                key_padding_mask: Optional[Tensor] = None) -> Tensor:
    """``y[t] = act(bias + sum_j weight[:, j] * x[t - width + 1 + j])`` per channel, zeros in front of the first token.

    x ``[tgt_len, bsz, channels]``, weight ``[channels, width]`` (width 1 to 8) and bias ``[channels]`` of x's dtype;
    activation "silu" or None."""
    silu, mask = _silu(activation), _mask(key_padding_mask)
    if plain_tensors(x, weight, bias, mask):
        return native().causal_conv_node(x, weight, bias, mask, silu)
    return _CausalConv.apply(x, weight, bias, None, mask, silu, False)


def incremental_causal_conv(*, x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, state: Optional[Tensor] = None,
                            activation: Optional[str] = "silu",
                            key_padding_mask: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``causal_conv`` that goes on from the inputs in front of its first token: state ``[bsz, width - 1, channels]`` of x's
    dtype, oldest first (None: zeros).  Returns ``(y, state)`` with the last ``width - 1`` inputs as state."""
    silu, mask = _silu(activation), _mask(key_padding_mask)
    if plain_tensors(x, weight, bias, state, mask):
        return native().incremental_causal_conv_node(x, weight, bias, state, mask, silu)
    if _underived(x, weight, bias, state):
        return ops.causal_conv_fwd(x, weight, bias, state, mask, silu, True, True)
    return _CausalConv.apply(x, weight, bias, state, mask, silu, True)


# --------------------------------------------------------------------------- selective scan
class _SelectiveScan(torch.autograd.Function):
    """(x, dt, a, b, c, d or None, dt_bias or None, s or None, mask or None) -> y[, the last state]."""

    @staticmethod
    def forward(ctx, x, dt, a, b, c, d, dt_bias, s, mask, softplus, return_state):
        y, out, kept = ops.selective_scan_fwd(x, dt, a, b, c, d, dt_bias, s, mask, softplus, return_state, False, True)
        ctx.save_for_backward(x, dt, a, b, c, d, dt_bias, s, mask, kept)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return (y, out) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_s=None):
        x, dt, a, b, c, d, dt_bias, s, mask, kept = ctx.saved_tensors
        g = torch.zeros_like(x) if g is None else g
        grads = ops.selective_scan_bwd(x, dt, a, b, c, d, dt_bias, s, mask, ctx.softplus, g, g_s, kept, ctx.needs_input_grad[7])
        return (*grads, None, None, None)


def selective_scan(*, x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None,
                   dt_bias: Optional[Tensor] = None, dt_softplus: bool = True,
                   key_padding_mask: Optional[Tensor] = None) -> Tensor:
    """Per channel, with ``num_states`` states that start at zero::

        delta[t] = softplus(dt[t] + dt_bias)                  (dt[t] + dt_bias with dt_softplus=False)
        s[t] = exp(delta[t] * a) * s[t - 1] + delta[t] * b[t] * x[t]
        y[t] = (c[t] * s[t]).sum() + d * x[t]

    x, dt ``[tgt_len, bsz, channels]``; b, c ``[tgt_len, bsz, num_groups, num_states]`` of x's dtype, shared by the
    ``channels / num_groups`` adjacent channels of a group (their gradients are sums over them); a ``[channels, num_states]``
    (finite, 1 to 64 states), d and dt_bias ``[channels]``, fp32.  ``delta * a`` is to stay below 88, where exp overflows
    (it is negative in a model, whose states decay): beyond that the results are not defined."""
    mask = _mask(key_padding_mask)
    if plain_tensors(x, dt, a, b, c, d, dt_bias, mask):
        return native().selective_scan_node(x, dt, a, b, c, d, dt_bias, mask, dt_softplus)
    return _SelectiveScan.apply(x, dt, a, b, c, d, dt_bias, None, mask, dt_softplus, False)


def incremental_selective_scan(*, x: Tensor, dt: Tensor, a: Tensor, b: Tensor, c: Tensor, d: Optional[Tensor] = None,
                               dt_bias: Optional[Tensor] = None, s: Optional[Tensor] = None, dt_softplus: bool = True,
                               key_padding_mask: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``selective_scan`` that goes on from the state s ``[bsz, channels, num_states]`` fp32 (None: zeros).  Returns
    ``(y, s)``."""
    mask = _mask(key_padding_mask)
    if plain_tensors(x, dt, a, b, c, d, dt_bias, s, mask):
        return native().incremental_selective_scan_node(x, dt, a, b, c, d, dt_bias, s, mask, dt_softplus)
    if _underived(x, dt, a, b, c, d, dt_bias, s):
        return ops.selective_scan_fwd(x, dt, a, b, c, d, dt_bias, s, mask, dt_softplus, True, True, False)[:2]
    return _SelectiveScan.apply(x, dt, a, b, c, d, dt_bias, s, mask, dt_softplus, True)


# --------------------------------------------------------------------------- group norm
class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, gate, silu, eps):
        ctx.save_for_backward(x, weight, bias, gate)
        ctx.args = num_groups, silu, eps
        return ops.group_norm_fwd(x, num_groups, weight, bias, gate, silu, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, gate = ctx.saved_tensors
        num_groups, silu, eps = ctx.args
        need = ctx.needs_input_grad
        gx, gw, gb, gg = ops.group_norm_bwd(x, num_groups, weight, bias, gate, silu, eps, g, *need[2:5])
        return gx, None, gw, gb, gg, None, None


def group_norm(*, x: Tensor, num_groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               gate: Optional[Tensor] = None, activation: Optional[str] = "silu", eps: float = 1e-5) -> Tensor:
    """Each token's channels in ``num_groups`` runs of adjacent ones, every run brought to mean 0 and variance 1 (eps added
    to the variance), times weight plus bias: n.  Returns ``n * act(gate)``, without a gate ``act(n)``.

    x and gate ``[..., channels]``, weight and bias ``[channels]``, all of one dtype, runs of at most 16384 channels;
    activation "silu" or None.  The statistics are a token's own (``torch.nn.GroupNorm`` on ``[tokens, channels]``), so that
    a causal layer stays causal and a token's result does not depend on the ones it is called with."""
    silu = _silu(activation)
    if plain_tensors(x, weight, bias, gate):
        return native().group_norm_node(x, num_groups, weight, bias, gate, silu, eps)
    return _GroupNorm.apply(x, num_groups, weight, bias, gate, silu, eps)


# --------------------------------------------------------------------------- layer
class SelectiveStateSpace(nn.Module):
    """A causal layer of the same call as ``CausalAttention``'s, without random matrices: input projection to ``inner_dim``
    channels and as many gates, short causal convolution, selective scan whose step sizes, b and c are projections of
    the convolution's output, group norm gated by silu(gate), output projection.

    a is ``-exp(a_log)``, initialised to -1 ... -state_dim; dt_bias so that the step sizes start log-uniform in
    [0.001, 0.1].  ``norm_groups`` defaults to groups of 64 channels where they divide, else one group.  What the operators
    take is asked for here: ``conv_width`` 1 to 8, ``state_dim`` 1 to 64, norm groups of at most 16384 channels."""

    def __init__(self, *, embed_dim: int, inner_dim: Optional[int] = None, state_dim: int = 16, conv_width: int = 4,
                 dt_rank: Optional[int] = None, num_groups: int = 1, norm_groups: Optional[int] = None):
        super().__init__()
        inner_dim = 2 * embed_dim if inner_dim is None else inner_dim
        dt_rank = max(1, math.ceil(embed_dim / 16)) if dt_rank is None else dt_rank
        norm_groups = (inner_dim // 64 if inner_dim % 64 == 0 else 1) if norm_groups is None else norm_groups
        assert 1 <= conv_width <= 8, "conv_width must be 1 to 8"
        assert 1 <= state_dim <= 64, "state_dim must be 1 to 64"
        assert 1 <= inner_dim <= 1 << 24, "inner_dim must be 1 to 2^24"
        assert num_groups >= 1 and inner_dim % num_groups == 0, "inner_dim must be divisible by num_groups"
        assert norm_groups >= 1 and inner_dim % norm_groups == 0, "inner_dim must be divisible by norm_groups"
        assert inner_dim // norm_groups <= 16384, "norm_groups must leave at most 16384 channels in a group"
        self.embed_dim, self.inner_dim, self.state_dim, self.conv_width = embed_dim, inner_dim, state_dim, conv_width
        self.dt_rank, self.num_groups, self.norm_groups = dt_rank, num_groups, norm_groups
        self.in_proj = nn.Linear(embed_dim, 2 * inner_dim, bias=False)
        self.conv_weight, self.conv_bias = Parameter(Tensor(inner_dim, conv_width)), Parameter(Tensor(inner_dim))
        self.x_proj = nn.Linear(inner_dim, dt_rank + 2 * num_groups * state_dim, bias=False)
        self.dt_proj = nn.Linear(dt_rank, inner_dim, bias=False)
        self.dt_bias, self.a_log, self.d = Parameter(Tensor(inner_dim)), Parameter(Tensor(inner_dim, state_dim)), Parameter(Tensor(inner_dim))
        self.norm_weight, self.norm_bias = Parameter(Tensor(inner_dim)), Parameter(Tensor(inner_dim))
        self.out_proj = nn.Linear(inner_dim, embed_dim, bias=True)
        self.reset_parameters()

    def reset_parameters(self):
        for lin in (self.in_proj, self.x_proj, self.out_proj):
            nn.init.xavier_uniform_(lin.weight, gain=1 / math.sqrt(2))
        nn.init.uniform_(self.dt_proj.weight, -self.dt_rank ** -0.5, self.dt_rank ** -0.5)
        nn.init.uniform_(self.conv_weight, -self.conv_width ** -0.5, self.conv_width ** -0.5)
        for zero in (self.conv_bias, self.norm_bias, self.out_proj.bias):
            nn.init.constant_(zero, 0.)
        for one in (self.d, self.norm_weight):
            nn.init.constant_(one, 1.)
        with torch.no_grad():
            step = torch.exp(torch.rand_like(self.dt_bias) * math.log(100.0) + math.log(1e-3))
            self.dt_bias.copy_(step + torch.log(-torch.expm1(-step)))          # softplus of it is the step
            self.a_log.copy_(torch.log(torch.arange(1, self.state_dim + 1, dtype=torch.float32)).expand_as(self.a_log))

    @staticmethod
    def reorder_incremental_state(saved_state: Dict[str, Optional[Tensor]], new_order: Tensor) -> Dict[str, Optional[Tensor]]:
        """Beam search: keep, per new batch slot i, the running state of old slot ``new_order[i]``."""
        for key in ("prev_conv", "prev_s"):
            t = saved_state.get(key)
            if t is not None:
                saved_state[key] = t.index_select(0, new_order.to(device=t.device, dtype=torch.long))
        return saved_state

    def forward(self, x: Tensor, key_padding_mask: Optional[Tensor] = None,
                saved_state: Optional[Dict[str, Optional[Tensor]]] = None) -> Tensor:
        """x ``[tgt_len, bsz, embed_dim]`` -> ``[tgt_len, bsz, embed_dim]``; key_padding_mask ``[bsz, tgt_len]``.  With
        ``saved_state`` (a dict; keys ``prev_conv``, ``prev_s`` are created on first use) the call goes on from the tokens
        of the calls before it, by one token or by a whole prompt."""
        assert x.size(-1) == self.embed_dim
        u, gate = self.in_proj(x).chunk(2, dim=-1)
        half = u.dtype
        conv = dict(weight=self.conv_weight.to(half), bias=self.conv_bias.to(half), key_padding_mask=key_padding_mask)
        if saved_state is None:
            u = causal_conv(x=u, **conv)
        else:
            u, saved_state["prev_conv"] = incremental_causal_conv(x=u, **conv, state=saved_state.get("prev_conv"))
        n, g = self.state_dim, self.num_groups
        low, b, c = self.x_proj(u).split([self.dt_rank, g * n, g * n], dim=-1)
        scan = dict(x=u, dt=self.dt_proj(low), a=-torch.exp(self.a_log.float()), b=b.unflatten(-1, (g, n)), c=c.unflatten(-1, (g, n)),
                    d=self.d.float(), dt_bias=self.dt_bias.float(), key_padding_mask=key_padding_mask)
        if saved_state is None:
            y = selective_scan(**scan)
        else:
            y, saved_state["prev_s"] = incremental_selective_scan(**scan, s=saved_state.get("prev_s"))
        y = group_norm(x=y, num_groups=self.norm_groups, weight=self.norm_weight.to(half), bias=self.norm_bias.to(half), gate=gate)
        return self.out_proj(y)
