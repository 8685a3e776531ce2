"""Slots of pools of states: what serving does with running requests between tokens.

A pool is a tensor ``[slots, ...]`` with one row for each slot (``decay_attention_step``'s and ``gated_scan_step``'s states, the
positions beside them, those of other layers). ``copy_slots`` copies rows to other rows all at once: requests are forked, reordered
in place, cleared. ``compact_slots`` moves running requests into the lowest slots. The computation runs in ``libhyfft.so``
(``hyfft_pool_copy`` / ``hyfft_pool_compact``) on the caller's stream, with no CPU fallback and no wait for the device. The reference
has no counterpart.
"""

from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import _lib

__all__ = ["copy_slots", "compact_slots", "SlotCache"]

MAX_POOLS = 16
MAX_MOVES = 12800


def _pools(pools: torch.Tensor | Sequence[torch.Tensor]):
    """(pools as a list, their number of slots)."""
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    assert 1 <= len(pools) <= MAX_POOLS, f"1 to {MAX_POOLS} pools in a call; got {len(pools)}"
    for t in pools:
        assert t.ndim >= 1 and t.shape[0] == pools[0].shape[0], (
            f"the pools must have the same slots; got {[tuple(t.shape) for t in pools]}")
        assert t.is_contiguous(), "the pools must be contiguous"
    if _lib.autograd_sees(*pools):
        raise NotImplementedError("slots are copied without a gradient: call it under torch.no_grad()")
    return pools, pools[0].shape[0]


def _table(pools):
    """The pools that have bytes, as the library takes them."""
    rows = [(t.data_ptr(), t.numel() // t.shape[0] * t.element_size()) for t in pools if t.numel()]
    return (_lib.Pool * max(len(rows), 1))(*[_lib.Pool(*r) for r in rows]), len(rows)


def _workspaces(slots: int, moves: int) -> tuple[int, int]:
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.check(_lib.load().hyfft_pool_workspace_size(slots, moves, ctypes.byref(a), ctypes.byref(b)), "hyfft_pool_workspace_size")
    return a.value, b.value


def copy_slots(pools: torch.Tensor | Sequence[torch.Tensor], source: torch.Tensor, target: torch.Tensor) -> None:
    """``pool[target[i]] = pool[source[i]]`` for every i at once, in place, for one pool or several of the same slots.

    Args:
        pools: contiguous tensors ``[slots, ...]`` of any types, at most 16, that do not overlap.
        source, target: int32 ``[n]``, n <= 12800. Every source is read as it was before the call, also where it is another
            move's target. A source outside ``0 .. slots - 1`` means zeros; a move whose target is outside is not made; of
            several moves into one slot the last is made.
    """
    pools, slots = _pools(pools)
    for name, t in (("source", source), ("target", target)):
        assert t.ndim == 1, f"{name} must be [n]; got {tuple(t.shape)}"
        assert t.dtype == torch.int32, f"{name} must be int32; got {t.dtype}"
    assert source.shape == target.shape, f"source and target must agree; got {tuple(source.shape)} and {tuple(target.shape)}"
    dev = _lib.require_cuda(*pools, source, target)
    source, target = source.contiguous(), target.contiguous()
    n = source.numel()
    table, count = _table(pools)
    if not (n and slots and count):
        return
    ws = _lib.workspace(_workspaces(slots, n)[0], dev)
    rc = _lib.load().hyfft_pool_copy(table, count, slots, source.data_ptr(), target.data_ptr(), n, ws.data_ptr(), ws.numel(),
                                     _lib.stream_ptr(dev))
    _lib.check(rc, "hyfft_pool_copy")


def compact_slots(pools: torch.Tensor | Sequence[torch.Tensor], live: torch.Tensor) -> torch.Tensor:
    """Moves the running requests in the highest slots into the lowest free ones, in order and in place, so that they take slots
    ``0 .. (their number) - 1``. Rows that are left behind stay as they were.

    Args:
        pools: as for ``copy_slots``.
        live: bool ``[slots]``, which slots hold running requests.

    Returns int32 ``[slots]``: the new slot of each slot's request, -1 where there is none.
    """
    pools, slots = _pools(pools)
    assert tuple(live.shape) == (slots,), f"live must be [{slots}]; got {tuple(live.shape)}"
    assert live.dtype == torch.bool, f"live must be bool; got {live.dtype}"
    dev = _lib.require_cuda(*pools, live)
    live = live.contiguous()
    moved = torch.empty(slots, dtype=torch.int32, device=dev)
    if not slots:
        return moved
    table, count = _table(pools)
    if not count:  # rows of no bytes: the numbers alone, beside rows that nobody reads
        pools = [torch.empty(slots, dtype=torch.uint8, device=dev)]  # kept until the call has been made
        table, count = _table(pools)
    ws = _lib.workspace(_workspaces(slots, 0)[1], dev)
    rc = _lib.load().hyfft_pool_compact(table, count, slots, live.data_ptr(), moved.data_ptr(), ws.data_ptr(), ws.numel(),
                                        _lib.stream_ptr(dev))
    _lib.check(rc, "hyfft_pool_compact")
    return moved


class SlotCache:
    """What caches of running requests share: ``slots`` rows of some tensors (``tensors()``), and one row more that calls with idle
    requests gather and scatter in their place. A slot outside ``0 .. slots - 1`` marks an idle request."""

    slots: int

    def tensors(self) -> list[torch.Tensor]:
        raise NotImplementedError

    def pools(self) -> list[torch.Tensor]:
        """The rows of the slots, without the spare one."""
        return [t[:self.slots] for t in self.tensors()]

    def fork(self, source: torch.Tensor, target: torch.Tensor) -> None:
        """Slots ``target`` go on from where slots ``source`` are, all at once (see ``copy_slots``); int32 lists."""
        copy_slots(self.pools(), source, target)

    def compact(self, live: torch.Tensor) -> torch.Tensor:
        """Moves the requests of the slots in ``live`` (bool ``[slots]``) into the lowest ones; returns where each is now (see
        ``compact_slots``)."""
        return compact_slots(self.pools(), live)

    def rows(self, slots: torch.Tensor | None, batch: int) -> torch.Tensor:
        """Rows for ``batch`` requests; idle ones (slots outside 0 .. slots - 1) get the spare row."""
        device = self.tensors()[0].device
        if slots is None:
            assert batch <= self.slots, f"{batch} requests need as many slots; the cache has {self.slots}"
            return torch.arange(batch, device=device)
        assert tuple(slots.shape) == (batch,), f"slots must be [{batch}]; got {tuple(slots.shape)}"
        slots = slots.long()
        return torch.where((slots >= 0) & (slots < self.slots), slots, self.slots)
