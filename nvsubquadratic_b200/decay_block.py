"""A causal mixer and block around the decayed linear attention, for training and for serving.

``DecayMixerB200`` takes the place of ``HyenaB200`` in ``QKVSequenceMixerB200`` (``forward(q, k, v, cp_group)`` on
channels-last ``[B, *S, C]``, read in place as views of the projection): rotary positions on queries and keys,
``decay_attention`` with one decay for each head, and a layer norm over each head's output (its
magnitude grows with a head's memory, the norm takes that out). ``DecayBlockB200`` is the pre-norm residual block
around it. A ``DecayCache`` carries every running request from one call to the next: a prompt of any length goes through
the sequence form, a single token through the recurrent form, with the same parameters.

    block = DecayBlockB200(768, heads=12).cuda().to(torch.bfloat16)
    y = block(x)                                      # training: x [B, L, 768]
    cache = DecayCache(slots=64, heads=12, head_dim=64, device="cuda")
    with torch.no_grad():
        y = block(prompts, cache=cache, slots=slots, lengths=lengths)   # [B, L, 768], padded on the right
        y = block(token, cache=cache, slots=slots)                      # [B, 1, 768]
"""

from __future__ import annotations

import torch

from .decay_attention import decay_attention, decay_attention_step
from .layer_norm import LayerNormB200, layer_norm
from .qk_norm import qk_norm_rotary
from .rotary import rotary, rotary_turns
from .sequence_mixer import QKVSequenceMixerB200
from .state_pool import SlotCache

__all__ = ["DecayCache", "DecayMixerB200", "DecayBlockB200"]


class DecayCache(SlotCache):
    """The states of up to ``slots`` running requests: float32 ``[slots, heads, head_dim, head_dim]`` and the position of
    each one's next token. Its size does not depend on the requests' lengths.

    A slot outside ``0 .. slots - 1`` in a call marks an idle request: nothing of it is read, the mixer's output for it is zero and no
    state changes, for prompts and for single tokens alike. ``fork`` and ``compact`` copy and move requests between slots."""

    def __init__(self, slots: int, heads: int, head_dim: int, device=None):
        self.slots = slots
        # one row more than slots: what calls with idle requests gather and scatter in their place, unchanged
        self.state = torch.zeros((slots + 1, heads, head_dim, head_dim), dtype=torch.float32, device=device)
        self.position = torch.zeros(slots + 1, dtype=torch.int64, device=device)

    def reset(self, slots: torch.Tensor) -> None:
        """Forgets what the given slots held, for new requests."""
        rows = self.rows(slots, slots.numel())
        self.state.index_fill_(0, rows, 0.0)
        self.position.index_fill_(0, rows, 0)

    def tensors(self) -> list[torch.Tensor]:
        return [self.state, self.position]


class DecayMixerB200(torch.nn.Module):
    """Decayed linear attention as a mixer of ``QKVSequenceMixerB200``.

    Args:
        hidden_dim: C, split evenly over the heads.
        heads: number of heads; their decays are spread over memories of ``2 ** 4 .. 2 ** 12`` tokens.
        learn_decay: make the decays' logarithms parameters (they are a buffer by default).
        rot_dim: features of each head that rotary positions turn (all of them by default, 0: none).
        rotary_args: further arguments of ``rotary_turns`` (base, scaling, factor, original_length).
        qk_norm: divide each head of queries and keys by its root mean square and scale it by learned weights, in the pass
            that turns them (``qk_norm_rotary``).
    """

    def __init__(self, hidden_dim: int, heads: int, *, learn_decay: bool = False, rot_dim: int | None = None,
                 interleaved: bool = False, eps: float = 1e-5, rotary_args: dict | None = None, qk_norm: bool = False):
        super().__init__()
        assert hidden_dim % heads == 0, f"hidden_dim {hidden_dim} must be a multiple of heads {heads}"
        self.heads, self.head_dim, self.eps, self.interleaved = heads, hidden_dim // heads, eps, interleaved
        memory = 2.0 ** torch.linspace(4.0, 12.0, heads, dtype=torch.float64)
        log_decay = torch.log1p(-1.0 / memory).float()
        if learn_decay:
            self.log_decay = torch.nn.Parameter(log_decay)
        else:
            self.register_buffer("log_decay", log_decay)
        rot_dim = self.head_dim // 2 * 2 if rot_dim is None else rot_dim
        self.amplitude, turns = 1.0, None
        if rot_dim:
            turns, self.amplitude = rotary_turns(rot_dim, **(rotary_args or {}))
        self.register_buffer("turns", turns, persistent=False)
        self.q_norm = torch.nn.Parameter(torch.ones(self.head_dim)) if qk_norm else None
        self.k_norm = torch.nn.Parameter(torch.ones(self.head_dim)) if qk_norm else None

    def _apply(self, fn, recurse=True):
        # the decays stay float32 whatever type the rest of a model is cast to: a decay's rounding error is
        # raised to the power of the distance
        keep = self.log_decay.detach()
        grad = None if self.log_decay.grad is None else self.log_decay.grad.detach()
        super()._apply(fn, recurse)
        for t, kept in ((self.log_decay, keep), (self.log_decay.grad, grad)):
            if t is not None and t.dtype != torch.float32:
                t.data = kept.to(t.device)
        return self

    def _turn(self, q, k, positions):
        if self.q_norm is not None:
            return qk_norm_rotary(q, k, self.q_norm, self.k_norm, self.turns, positions=None if self.turns is None else positions,
                                  amplitude=self.amplitude, interleaved=self.interleaved)
        if self.turns is None:
            return q, k
        return rotary(q, k, self.turns, positions=positions, amplitude=self.amplitude, interleaved=self.interleaved)

    def forward(self, query, key, value, cp_group=None, *, cache: DecayCache | None = None,
                slots: torch.Tensor | None = None, lengths: torch.Tensor | None = None):
        if cp_group is not None and cp_group.size() > 1:
            raise NotImplementedError("DecayMixerB200 does not run context-parallel")
        shape, B = query.shape, query.shape[0]
        q, k, v = (t.flatten(1, -2).unflatten(-1, (self.heads, self.head_dim)) for t in (query, key, value))
        L = q.shape[1]
        if cache is None:
            q, k = self._turn(q, k, None)
            o = decay_attention(q, k, v, self.log_decay, lengths=lengths)
        else:
            rows = cache.rows(slots, B)
            start = cache.position[rows]
            q, k = self._turn(q, k, start[:, None] + torch.arange(L, device=start.device))
            live = None if slots is None else rows < cache.slots
            if L == 1 and lengths is None:
                owned = rows if live is None else torch.where(live, rows, -1)
                o = decay_attention_step(q[:, 0], k[:, 0], v[:, 0], self.log_decay, cache.state,
                                         slots=owned.to(torch.int32)).unsqueeze(1)
                count = torch.ones_like(start) if live is None else live.long()
            else:
                if live is not None:  # an idle request has no tokens
                    lengths = live.to(torch.int32) * L if lengths is None else lengths.masked_fill(~live, 0)
                o, state = decay_attention(q, k, v, self.log_decay, lengths=lengths, initial_state=cache.state[rows],
                                           return_state=True)
                cache.state.index_copy_(0, rows, state.detach())
                count = lengths.long().clamp(0, L) if lengths is not None else torch.full_like(start, L)
            cache.position.index_copy_(0, rows, start + count)
        return layer_norm(o, eps=self.eps).reshape(shape)


class DecayBlockB200(torch.nn.Module):
    """``x + mixer(norm(x))`` with a ``DecayMixerB200`` between its projections, on ``[B, L, C]``."""

    def __init__(self, hidden_dim: int, heads: int, *, qkv_bias: bool = False, out_proj_bias: bool = False, **mixer_args):
        super().__init__()
        self.norm = LayerNormB200(hidden_dim)
        self.mixer = QKVSequenceMixerB200(hidden_dim, DecayMixerB200(hidden_dim, heads, **mixer_args), qkv_bias,
                                          out_proj_bias)

    def forward(self, x: torch.Tensor, *, cache: DecayCache | None = None, slots: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None) -> torch.Tensor:
        return x + self.mixer(self.norm(x), cache=cache, slots=slots, lengths=lengths)
