"""Sequences packed one behind the other along one axis of rows, without padding between them.

:class:`SequencePack` is what the packed operators take: for every row the sequence it belongs to.  A training step makes
one per batch (:func:`pack_sequences`) and hands it to every layer.
"""

from __future__ import annotations

from typing import Optional

import torch


class SequencePack:
    """``spans``: int32 ``[rows, 2]``, first row and end of the sequence a row belongs to (0, 0 outside every sequence);
    ``positions``: int64 ``[rows]``, a row's position inside its sequence (0 outside).  ``plan``: what the attention kernels
    read on GPU (positions, spans and the order they take the rows in, one buffer).  ``longest``: length of the longest
    sequence, ``None`` where the offsets were on the GPU."""

    __slots__ = ("rows", "device", "plan", "longest", "_host")

    def __init__(self, rows: int, plan: Optional[torch.Tensor] = None, host=None, longest: Optional[int] = None):
        self.rows, self.plan, self._host, self.longest = rows, plan, host, longest
        self.device = plan.device if host is None else host[0].device

    @property
    def spans(self) -> torch.Tensor:
        return self._host[0] if self._host is not None else self.plan[self.rows:2 * self.rows].view(torch.int32).view(-1, 2)

    @property
    def positions(self) -> torch.Tensor:
        return self._host[1] if self._host is not None else self.plan[:self.rows]


def _check_on_host(offsets: torch.Tensor, rows: int) -> None:
    if offsets[0] < 0 or bool((offsets[1:] < offsets[:-1]).any()):
        raise ValueError("sequence offsets must start at 0 or later and never fall")
    if offsets[-1] > rows:
        raise ValueError(f"the sequences end at row {int(offsets[-1])}, beyond the {rows} rows there are")


def pack_sequences(offsets, rows: int, device: Optional[torch.device] = None) -> SequencePack:
    """The pack of sequences ``[offsets[i], offsets[i + 1])`` over ``rows`` rows.

    ``offsets``: ``[sequences + 1]`` int32 / int64 tensor, or a list.  Sequences may be empty; rows in front of the first
    and behind the last belong to none.  Offsets on the host are checked and sent to ``device``; offsets on the GPU are not
    read back (no synchronisation): they must not fall, and what reaches beyond ``rows`` is cut off."""
    if not isinstance(offsets, torch.Tensor):
        offsets = torch.tensor(offsets)
    if offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError("sequence offsets are a one-dimensional int32 or int64 tensor of at least one element")
    rows = int(rows)
    if not 0 <= rows < 1 << 30:
        raise ValueError(f"a pack holds 0 to 2^30 - 1 rows, got {rows}")
    longest = None
    if not offsets.is_cuda:
        _check_on_host(offsets, rows)
        longest = int((offsets[1:] - offsets[:-1]).max()) if offsets.numel() > 1 else 0
        if device is not None:
            offsets = offsets.to(device)
    elif device is not None and torch.device(device) not in (offsets.device, torch.device(offsets.device.type)):
        raise ValueError(f"sequence offsets on {offsets.device}, pack wanted on {device}")
    if offsets.is_cuda:
        from . import hip_packed

        return SequencePack(rows, hip_packed.pack_plan(offsets, rows), longest=longest)
    offsets = offsets.to(torch.int64)
    row = torch.arange(rows)
    at = torch.searchsorted(offsets, row, right=True) - 1  # the last sequence that starts at or before the row
    inside = (at >= 0) & (at < offsets.numel() - 1)
    at = at.clamp(0, max(offsets.numel() - 2, 0))
    ends = offsets[1:] if offsets.numel() > 1 else offsets
    spans = torch.stack([offsets[at], ends[at]], 1) * inside[:, None]
    return SequencePack(rows, host=(spans.to(torch.int32), torch.where(inside, row - spans[:, 0], 0)), longest=longest)
