"""Softmax attention over a sliding window, beside causal RFA: exact attention to the last tokens and to a few first ones, with a cache of
one size whatever the sequence's length.  Functional forms and the ``WindowAttention`` layer, in the manner of ``causal_attention.py``:

* ``window_attention``             -> token i attends to the tokens j <= i with i - j < window or j < sinks
* ``incremental_window_attention`` -> the same behind the tokens that a cache holds, which it updates, over any number of tokens

Activations are time-major, ``[tgt_len, bsz, num_heads, head_dim]``, fp16, bf16 or fp32, with any strides as long as a head's numbers are
adjacent (views of a projection's output are taken as they are); scores, softmax and sums are fp32, in 16 bits the weights and their gradients are
rounded for the products with values, keys and queries.  The backward makes the weights again from fp32 log-sums: scores of size m cost them m 2 ** -23.  Heads of at most 256.  k and v may
have fewer heads than q: ``num_heads / num_kv_heads`` adjacent query heads share one, whose gradients are sums over them.  The
backward pass is not differentiable itself.  No upstream counterpart.

``key_padding_mask`` ``[bsz, tgt_len]`` (1 = padding): padded tokens are skipped, wherever they stand, and not counted in distances --
every result is what it would be without them, whatever values they hold, and their own outputs and gradients are zero.  A real
token that is not finite reaches the tokens that see it, and may reach the outputs and the gradients of q of tokens less than 320 from one of these.  The
gradients of k and v gather from the tokens that see a key, and may from ones as near to these; of keys less than 128 places from a first token, from any."""
from typing import Dict, Optional, Tuple

import math

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import native
from ._plain import plain_tensors
from .causal_attention import _underived
from .state_space import _mask


class _WindowAttention(torch.autograd.Function):
    """(q, k, v, window, sinks, mask or None, scale) -> out."""

    @staticmethod
    def forward(ctx, q, k, v, window, sinks, mask, scale):
        out, lse = ops.window_attention_fwd(q, k, v, window, sinks, mask, scale, True)
        ctx.save_for_backward(q, k, v, mask, out, lse)
        ctx.args = window, sinks, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, mask, out, lse = ctx.saved_tensors
        window, sinks, scale = ctx.args
        return (*ops.window_attention_bwd(q, k, v, window, sinks, mask, scale, out, lse, g), None, None, None, None)


def window_attention(*, q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int = 0, scale: Optional[float] = None,
                     key_padding_mask: Optional[Tensor] = None) -> Tensor:
    """q ``[tgt_len, bsz, num_heads, head_dim]``, k, v ``[tgt_len, bsz, num_kv_heads, head_dim]`` of one dtype; window >= 1 counts the token
    itself, the first ``sinks`` tokens stay visible to all behind them.  scale defaults to ``head_dim ** -0.5``.  Returns ``[tgt_len,
    bsz, num_heads, head_dim]``."""
    mask = _mask(key_padding_mask)
    if plain_tensors(q, k, v, mask):
        return native().window_attention_node(q, k, v, window, sinks, mask, scale)
    return _WindowAttention.apply(q, k, v, window, sinks, mask, scale)


def incremental_window_attention(*, q: Tensor, k: Tensor, v: Tensor, window: int, sinks: int = 0, prev_k: Optional[Tensor] = None,
                                 prev_v: Optional[Tensor] = None, prev_len: Optional[Tensor] = None, scale: Optional[float] = None,
                                 key_padding_mask: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """``window_attention`` that goes on from a cache: prev_k, prev_v ``[bsz, num_kv_heads, sinks + window, head_dim]`` of q's dtype and
    prev_len ``[bsz]`` int64, the number of tokens so far, all None before the first.  Token number p (from 0) is kept at slot p where
    p < sinks, else at ``sinks + (p - sinks) % window``.  Returns ``(out, prev_k, prev_v, prev_len)``; a cache that is passed in is
    UPDATED IN PLACE and returned.  For decoding: with autograd recording, inputs that require grad are refused."""
    mask = _mask(key_padding_mask)
    if not plain_tensors(q, k, v, prev_k, prev_v, prev_len, mask) and not _underived(q, k, v, prev_k, prev_v):
        raise RuntimeError("incremental_window_attention is for decoding: no gradient goes through its cache (call it under no_grad)")
    return ops.window_attention_append(q, k, v, window, sinks, prev_k, prev_v, prev_len, mask, scale)


class WindowAttention(nn.Module):
    """A causal layer of the same call as ``CausalAttention``'s, without random matrices: projections to q, k and v, attention over a
    sliding window with ``sinks`` first tokens, output projection.  It knows no positions but the window: add them to x where order
    within it matters."""

    def __init__(self, *, embed_dim: int, num_heads: int, window: int, sinks: int = 0, num_kv_heads: Optional[int] = None,
                 head_dim: Optional[int] = None):
        super().__init__()
        assert embed_dim % num_heads == 0 or head_dim, "embed_dim must be divisible by num_heads"
        assert window >= 1 and sinks >= 0, "window must be at least 1 and sinks at least 0"
        self.embed_dim, self.num_heads, self.window, self.sinks = embed_dim, num_heads, window, sinks
        self.num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        assert self.num_kv_heads >= 1 and num_heads % self.num_kv_heads == 0, "num_heads must be divisible by num_kv_heads"
        self.head_dim = embed_dim // num_heads if head_dim is None else head_dim
        assert 1 <= self.head_dim <= 256, "head_dim must be 1 to 256"
        self.in_proj = nn.Linear(embed_dim, (num_heads + 2 * self.num_kv_heads) * self.head_dim, bias=True)
        self.out_proj = nn.Linear(num_heads * self.head_dim, embed_dim, bias=True)
        self.reset_parameters()

    def reset_parameters(self):
        for lin in (self.in_proj, self.out_proj):
            nn.init.xavier_uniform_(lin.weight, gain=1 / math.sqrt(2))
            nn.init.constant_(lin.bias, 0.)

    @staticmethod
    def reorder_incremental_state(saved_state: Dict[str, Optional[Tensor]], new_order: Tensor) -> Dict[str, Optional[Tensor]]:
        """Beam search: keep, per new batch slot i, the cache of old slot ``new_order[i]``."""
        for key in ("prev_k", "prev_v", "prev_len"):
            t = saved_state.get(key)
            if t is not None:
                saved_state[key] = t.index_select(0, new_order.to(device=t.device, dtype=torch.long))
        return saved_state

    def forward(self, x: Tensor, key_padding_mask: Optional[Tensor] = None,
                saved_state: Optional[Dict[str, Optional[Tensor]]] = None) -> Tensor:
        """x ``[tgt_len, bsz, embed_dim]`` -> ``[tgt_len, bsz, embed_dim]``; key_padding_mask ``[bsz, tgt_len]``.  With ``saved_state`` (a
        dict; keys ``prev_k``, ``prev_v``, ``prev_len`` are created on first use; no gradients) the call goes on from the tokens of
        the calls before it, by one token or by a whole prompt."""
        assert x.size(-1) == self.embed_dim
        h, g, d = self.num_heads, self.num_kv_heads, self.head_dim
        q, k, v = self.in_proj(x).split([h * d, g * d, g * d], dim=-1)
        args = dict(q=q.unflatten(-1, (h, d)), k=k.unflatten(-1, (g, d)), v=v.unflatten(-1, (g, d)), window=self.window, sinks=self.sinks,
                    key_padding_mask=key_padding_mask)
        if saved_state is None:
            y = window_attention(**args)
        else:
            y, saved_state["prev_k"], saved_state["prev_v"], saved_state["prev_len"] = incremental_window_attention(
                **args, prev_k=saved_state.get("prev_k"), prev_v=saved_state.get("prev_v"), prev_len=saved_state.get("prev_len"))
        return self.out_proj(y.flatten(-2))
