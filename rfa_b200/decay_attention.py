"""Linear attention whose state decays, beside causal RFA: the running state S of ``incremental_rfa`` without its normaliser, faded
by a factor of its own for each head before a token is added.  Functional forms and the ``DecayAttention`` layer, in the manner
of ``causal_attention.py`` and ``state_space.py``:

* ``decay_attention``             -> out_t = scale * q_t S_t, S_t = exp(log_decay_t) S_(t-1) + k_t (x) v_t, in chunks of tokens
* ``incremental_decay_attention`` -> the same from a state and with the last one returned, over any number of tokens

Activations are time-major, ``[tgt_len, bsz, num_heads, width]``, fp16, bf16 or fp32, with any strides as long as a head's numbers are
adjacent (views of a projection's output are taken as they are); sums and states are fp32 (a state that several bf16 tokens leave is made of keys in two
parts of 8 bits and off by up to 3e-6 of its norm).  Heads of at most 256.  The backward
passes are not differentiable themselves.  No upstream counterpart.

``key_padding_mask`` ``[bsz, tgt_len]`` (1 = padding): padded tokens are skipped, wherever they stand -- every result is what it
would be without them, whatever values they hold, and their own outputs and gradients are zero.  A real token that is not finite may
reach the outputs of any token less than 128 places from it, as it reaches all behind it; gradients likewise, those of the decays anywhere in its sequence.

In fp16 and bf16 the outputs of several tokens come from 16-bit copies of the state (its own value is fp32) and of the weights, scale times q . k times the decay
between two tokens: in fp16 a state or a weight beyond 65504 gives outputs that are not finite.  A log decay below -44.36 (a factor of 2 ** -64) is taken as that
there.  Gradients pass through 16-bit products: fp16 ones below about 1e-4 lose digits, 0.3 % at 1e-5, so that a small loss wants scaling."""
from typing import Dict, Optional, Tuple

import math

import torch
import torch.nn.functional as F
from torch import Tensor, nn
from torch.autograd.function import once_differentiable
from torch.nn import Parameter

from . import ops
from ._lib import native
from ._plain import plain_tensors
from .causal_attention import _underived
from .state_space import _mask, group_norm


class _DecayAttention(torch.autograd.Function):
    """(q, k, v, log_decay, s or None, mask or None) -> out[, the last state]."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, s, mask, scale, return_state):
        out, last, kept = ops.decay_attention_fwd(q, k, v, log_decay, s, mask, scale, return_state, False, True)
        ctx.save_for_backward(q, k, v, log_decay, s, mask, kept)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_s=None):
        q, k, v, log_decay, s, mask, kept = ctx.saved_tensors
        g = torch.zeros_like(v) if g is None else g
        grads = ops.decay_attention_bwd(q, k, v, log_decay, s, mask, ctx.scale, g, g_s, kept, ctx.needs_input_grad[3], ctx.needs_input_grad[4])
        return (*grads, None, None, None)


def decay_attention(*, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: Optional[float] = None,
                    key_padding_mask: Optional[Tensor] = None) -> Tensor:
    """q, k ``[tgt_len, bsz, num_heads, key_dim]``, v ``[tgt_len, bsz, num_heads, head_dim]`` of one dtype; log_decay, of that dtype or
    fp32, ``[num_heads]`` (the same for all tokens) or ``[tgt_len, bsz, num_heads]``: at most 0 in a model, -inf forgets all that came
    before.  scale defaults to ``key_dim ** -0.5``.  Returns ``[tgt_len, bsz, num_heads, head_dim]``."""
    mask = _mask(key_padding_mask)
    if plain_tensors(q, k, v, log_decay, mask):
        return native().decay_attention_node(q, k, v, log_decay, mask, scale)
    return _DecayAttention.apply(q, k, v, log_decay, None, mask, scale, False)


def incremental_decay_attention(*, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, s: Optional[Tensor] = None,
                                scale: Optional[float] = None, key_padding_mask: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``decay_attention`` that goes on from the state s ``[bsz, num_heads, key_dim, head_dim]`` fp32 (None: zeros).  Returns ``(out,
    s)``.  As in ``incremental_rfa``, a state that is passed in is UPDATED IN PLACE and returned when no gradient is being recorded;
    with autograd recording and an input that requires grad the call is differentiable in all of them, returns a NEW state and
    leaves the one passed in alone."""
    mask = _mask(key_padding_mask)
    if plain_tensors(q, k, v, log_decay, s, mask):
        return native().incremental_decay_attention_node(q, k, v, log_decay, s, mask, scale)
    if _underived(q, k, v, log_decay, s):
        return ops.decay_attention_fwd(q, k, v, log_decay, s, mask, scale, True, True)[:2]
    return _DecayAttention.apply(q, k, v, log_decay, s, mask, scale, True)


class DecayAttention(nn.Module):
    """A causal layer of the same call as ``CausalAttention``'s, without random matrices: projections to q, k, v and a gate, attention
    with a decay, group norm of each head gated by silu(gate), output projection.

    ``decay`` "head": a factor of ``1 - 2 ** (-5 - 8 h / num_heads)`` for head h, a buffer that stays fp32 whatever type the layer gets.  "token": one for each token and head,
    ``sigmoid(x W + b) ** (1 / 16)``, learned."""

    def __init__(self, *, embed_dim: int, num_heads: int, key_dim: Optional[int] = None, head_dim: Optional[int] = None, decay: str = "token"):
        super().__init__()
        assert embed_dim % num_heads == 0 or (key_dim and head_dim), "embed_dim must be divisible by num_heads"
        assert decay in ("token", "head"), "decay is 'token' or 'head'"
        self.embed_dim, self.num_heads, self.decay = embed_dim, num_heads, decay
        self.key_dim = embed_dim // num_heads if key_dim is None else key_dim
        self.head_dim = embed_dim // num_heads if head_dim is None else head_dim
        assert 1 <= self.key_dim <= 256 and 1 <= self.head_dim <= 256, "key_dim and head_dim must be 1 to 256"
        inner = num_heads * self.head_dim
        self.in_proj = nn.Linear(embed_dim, 2 * num_heads * self.key_dim + 2 * inner, bias=False)
        self.norm_weight, self.norm_bias = Parameter(Tensor(inner)), Parameter(Tensor(inner))
        self.out_proj = nn.Linear(inner, embed_dim, bias=True)
        if decay == "token":
            self.decay_proj = nn.Linear(embed_dim, num_heads, bias=True)
        else:
            self.register_buffer("log_decay", torch.log1p(-torch.exp2(-5.0 - 8.0 * torch.arange(num_heads, dtype=torch.float32) / num_heads)))
        self.reset_parameters()

    def _apply(self, fn, *args, **kwargs):
        # The fixed decays stay in fp32 when the parameters become 16 bits: 0.4 % of a rate (bf16) would add up along a sequence.
        fixed = self._buffers.get("log_decay")
        super()._apply(fn, *args, **kwargs)
        moved = self._buffers.get("log_decay")
        if moved is not None and moved.dtype != fixed.dtype:
            self._buffers["log_decay"] = fixed.to(moved.device)
        return self

    def reset_parameters(self):
        for lin in (self.in_proj, self.out_proj):
            nn.init.xavier_uniform_(lin.weight, gain=1 / math.sqrt(2))
        nn.init.constant_(self.out_proj.bias, 0.)
        nn.init.constant_(self.norm_weight, 1.)
        nn.init.constant_(self.norm_bias, 0.)
        if self.decay == "token":
            nn.init.xavier_uniform_(self.decay_proj.weight, gain=1 / math.sqrt(2))
            nn.init.constant_(self.decay_proj.bias, 1.)

    @staticmethod
    def reorder_incremental_state(saved_state: Dict[str, Optional[Tensor]], new_order: Tensor) -> Dict[str, Optional[Tensor]]:
        """Beam search: keep, per new batch slot i, the running state of old slot ``new_order[i]``."""
        t = saved_state.get("prev_s")
        if t is not None:
            saved_state["prev_s"] = t.index_select(0, new_order.to(device=t.device, dtype=torch.long))
        return saved_state

    def forward(self, x: Tensor, key_padding_mask: Optional[Tensor] = None,
                saved_state: Optional[Dict[str, Optional[Tensor]]] = None) -> Tensor:
        """x ``[tgt_len, bsz, embed_dim]`` -> ``[tgt_len, bsz, embed_dim]``; key_padding_mask ``[bsz, tgt_len]``.  With
        ``saved_state`` (a dict; key ``prev_s`` is created on first use) the call goes on from the tokens of the calls before it,
        by one token or by a whole prompt."""
        assert x.size(-1) == self.embed_dim
        h, kd, hd = self.num_heads, self.key_dim, self.head_dim
        q, k, v, gate = self.in_proj(x).split([h * kd, h * kd, h * hd, h * hd], dim=-1)
        log_decay = F.logsigmoid(self.decay_proj(x)) / 16 if self.decay == "token" else self.log_decay.float()
        args = dict(q=q.unflatten(-1, (h, kd)), k=k.unflatten(-1, (h, kd)), v=v.unflatten(-1, (h, hd)), log_decay=log_decay,
                    key_padding_mask=key_padding_mask)
        if saved_state is None:
            y = decay_attention(**args)
        else:
            y, saved_state["prev_s"] = incremental_decay_attention(**args, s=saved_state.get("prev_s"))
        half = y.dtype
        y = group_norm(x=y.flatten(-2), num_groups=h, weight=self.norm_weight.to(half), bias=self.norm_bias.to(half), gate=gate)
        return self.out_proj(y)
