"""A causal mixer and block around the gated linear recurrence, for training and for serving.

``GatedMixerB200`` takes the place of ``HyenaB200`` or ``DecayMixerB200`` in ``QKVSequenceMixerB200``: of the three parts of the
projection the value is what the recurrence remembers, the key says how much of the past each token keeps (the logits of its
decays), and the query gates the output, all in one pass (``gated_scan``). ``GatedBlockB200`` is the pre-norm residual block around it. A
``GatedCache`` carries running requests from one call to the next: a prompt of any length goes through the sequence form, a single
token through the recurrent form, with the same parameters; its slots are forked and compacted between tokens.

    block = GatedBlockB200(768).cuda().to(torch.bfloat16)
    y = block(x)                                      # training: x [B, L, 768]
    cache = GatedCache(slots=64, channels=768, device="cuda")
    with torch.no_grad():
        y = block(prompts, cache=cache, slots=slots, lengths=lengths)   # [B, L, 768], padded on the right
        cache.fork(source, target)                                       # one prompt answered several times
        y = block(token, cache=cache, slots=slots)                       # [B, 1, 768]
"""

from __future__ import annotations

import torch

from .gated_scan import gated_scan, gated_scan_step
from .layer_norm import LayerNormB200
from .sequence_mixer import QKVSequenceMixerB200
from .state_pool import MAX_MOVES, SlotCache, copy_slots

__all__ = ["GatedCache", "GatedMixerB200", "GatedBlockB200"]


class GatedCache(SlotCache):
    """The states of up to ``slots`` running requests: float32 ``[slots, channels]``, whatever the requests' lengths.

    A slot outside ``0 .. slots - 1`` in a call marks an idle request: nothing of it is read, the mixer's output for it is zero and no
    state changes, for prompts and for single tokens alike. ``fork`` and ``compact`` copy and move requests between slots."""

    def __init__(self, slots: int, channels: int, device=None):
        self.slots = slots
        self.state = torch.zeros((slots + 1, channels), dtype=torch.float32, device=device)

    def tensors(self) -> list[torch.Tensor]:
        return [self.state]

    def reset(self, slots: torch.Tensor) -> None:
        """Forgets what the given slots held, for new requests."""
        rows = self.rows(slots, slots.numel()).to(torch.int32)  # the spare row is no slot of the pool: idle requests clear nothing
        for part in rows.split(MAX_MOVES):
            copy_slots(self.pools(), torch.full_like(part, -1), part)


class GatedMixerB200(torch.nn.Module):
    """The gated linear recurrence as a mixer of ``QKVSequenceMixerB200``: ``silu(query) * h``, ``h = a h + (1 - a) value``,
    ``a = sigmoid(key)``. It has no parameters of its own."""

    def forward(self, query, key, value, cp_group=None, *, cache: GatedCache | None = None, slots: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None):
        if cp_group is not None and cp_group.size() > 1:
            raise NotImplementedError("GatedMixerB200 does not run context-parallel")
        shape, B = query.shape, query.shape[0]
        q, k, v = (t.flatten(1, -2) for t in (query, key, value))
        L = q.shape[1]
        if cache is None:
            return gated_scan(v, k, out_gate=q, lengths=lengths).reshape(shape)
        rows = cache.rows(slots, B)
        live = None if slots is None else rows < cache.slots
        if L == 1 and lengths is None:
            owned = rows if live is None else torch.where(live, rows, -1)
            y = gated_scan_step(v[:, 0], k[:, 0], cache.state, out_gate=q[:, 0], slots=owned.to(torch.int32))
        else:
            if live is not None:  # an idle request has no tokens
                lengths = live.to(torch.int32) * L if lengths is None else lengths.masked_fill(~live, 0)
            y, state = gated_scan(v, k, out_gate=q, lengths=lengths, initial_state=cache.state[rows], return_state=True)
            cache.state.index_copy_(0, rows, state.detach())
        return y.reshape(shape)


class GatedBlockB200(torch.nn.Module):
    """``x + mixer(norm(x))`` with a ``GatedMixerB200`` between its projections, on ``[B, L, C]``.

    The projection has a bias; that of the decays' logits starts as memories of ``2 ** 4 .. 2 ** 12`` tokens spread over the channels."""

    def __init__(self, hidden_dim: int, *, out_proj_bias: bool = False):
        super().__init__()
        self.norm = LayerNormB200(hidden_dim)
        self.mixer = QKVSequenceMixerB200(hidden_dim, GatedMixerB200(), True, out_proj_bias)
        memory = 2.0 ** torch.linspace(4.0, 12.0, hidden_dim, dtype=torch.float64)
        with torch.no_grad():
            bias = self.mixer.qkv_proj.bias
            bias.zero_()
            bias[hidden_dim:2 * hidden_dim] = torch.log(memory - 1).to(bias.dtype)

    def forward(self, x: torch.Tensor, *, cache: GatedCache | None = None, slots: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None) -> torch.Tensor:
        return x + self.mixer(self.norm(x), cache=cache, slots=slots, lengths=lengths)
