"""Ring-buffer KV cache with the public surface of the reference's ``KVCache``
(inference/kv_cache.py:4-68): storage ``k, v [L, B, H, W, D]``, the token at
position ``p`` lives in slot ``p % W``, ``view`` returns the live rows in
chronological order, ``write`` stages the row of position ``t`` and ``advance``
moves on by one position.

``ring(layer)`` is an addition for the HIP decode kernel: it hands out the layer's
storage as it lies (slot order) so that a decode step reads the ring in place,
writes the new row itself, and no chronological copy is ever made.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import TYPE_CHECKING, Dict, List, Optional, Tuple

import torch
from torch import Tensor

if TYPE_CHECKING:
    from .ops import DraftTree


@dataclass
class RingContext:
    """Handle to one layer of a ``KVCache`` for the in-place decode path.

    ``k``/``v`` are the layer's ``[B, H, W, D]`` storage (views, not copies) and
    ``t`` the number of positions written so far; the row for position ``t``
    goes to slot ``t % W``.
    """
    cache: "KVCache"
    layer: int
    k: Tensor
    v: Tensor
    t: int
    W: int
    # one int32 on the GPU in which a step whose position lives in device memory reports what the
    # host cannot check beforehand (a position past the rotary tables); None = not wanted
    status: Optional[Tensor] = None

    def mark_written(self) -> None:
        self.cache._staged[self.layer] = True


class KVCache:
    """``t`` positions have been committed; a layer whose row for position ``t`` has been written
    but not yet committed is *staged* (``advance`` commits all layers at once)."""

    def __init__(self, L, B, H, W, D, device, dtype):
        self.L, self.B, self.H, self.W, self.D = L, B, H, W, D
        self.device, self.dtype = device, dtype
        self.k = torch.zeros((L, B, H, W, D), device=device, dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.t = 0
        self._staged = [False] * L

    def reset_history(self):
        # The reference allocates fresh zero tensors here (kv_cache.py:19-23); the storage is
        # reused instead so that a long-lived cache never reallocates.
        for store in (self.k, self.v):
            store.zero_()
        self.t = 0
        self._staged = [False] * self.L

    # -- reading -----------------------------------------------------------------------------
    def _live_rows(self, layer) -> Tuple[int, int]:
        """(first position, number of rows) that ``view`` shows: the newest ``min(written, W)``."""
        written = self.t + (1 if self._staged[layer] else 0)
        rows = min(written, self.W)
        return written - rows, rows

    def view(self, layer) -> Tuple[Tensor, Tensor]:
        """The live rows of a layer, oldest first, as ``[B, n, H, D]`` (``n = 0`` for an empty
        cache).  A run of slots that does not wrap is returned as a view; a run that wraps is
        the tail of the ring followed by its head (a copy)."""
        first, rows = self._live_rows(layer)
        lo = first % self.W if rows else 0
        hi = lo + rows
        out = []
        for store in (self.k[layer], self.v[layer]):          # [B, H, W, D]
            if hi <= self.W:
                run = store[:, :, lo:hi]
            else:
                run = torch.cat((store[:, :, lo:], store[:, :, :hi - self.W]), dim=2)
            out.append(run.transpose(1, 2))
        return out[0], out[1]

    def ring(self, layer) -> RingContext:
        """In-place handle for the decode kernel (no copy)."""
        return RingContext(self, layer, self.k[layer], self.v[layer], self.t, self.W)

    # -- writing -----------------------------------------------------------------------------
    def write(self, layer, k_new, v_new):
        """Stages the row of position ``t`` in slot ``t % W``.  A row may come as ``[B, 1, H, D]``
        or ``[B, H, 1, D]``; as in the reference, a size-1 second dim marks the former."""
        slot = self.t % self.W
        for store, row in ((self.k, k_new), (self.v, v_new)):
            if row.size(1) == 1:
                row = row.transpose(1, 2)
            store[layer, :, :, slot] = row[:, :, 0]
        self._staged[layer] = True

    def advance(self):
        """Commits the staged rows of all layers: position ``t`` is done."""
        self.t += 1
        self._staged = [False] * self.L

    def _prompt_runs(self, pos):
        """A prompt of ``pos`` tokens leaves room for the token that follows: only its last
        ``min(pos, W - 1)`` positions are kept.  Position p goes to slot ``p % W``, so the kept
        positions land in at most two runs of consecutive slots; returns ``(source, slots)``
        slice pairs (plain slice copies run several times faster than an indexed scatter)."""
        kept = min(pos, max(self.W - 1, 0))
        runs = []
        first = pos - kept
        while kept > 0:
            slot = first % self.W
            n = min(kept, self.W - slot)
            runs.append((slice(first, first + n), slice(slot, slot + n)))
            first, kept = first + n, kept - n
        return runs

    def bulk_write_packed(self, kv, pos):
        """Stores a prompt's keys and values from ``kv [2, L, B, H, T, D]`` and sets ``t = pos``."""
        for src, slots in self._prompt_runs(pos):
            self.k[:, :, :, slots].copy_(kv[0][:, :, :, src])
            self.v[:, :, :, slots].copy_(kv[1][:, :, :, src])
        self.t = pos
        self._staged = [False] * self.L

    def bulk_write_layer(self, layer, k, v, pos):
        """Per-layer form of ``bulk_write_packed`` for ``k, v [B, H, T, D]``; does not move ``t``."""
        for src, slots in self._prompt_runs(pos):
            self.k[layer][:, :, slots].copy_(k[:, :, src])
            self.v[layer][:, :, slots].copy_(v[:, :, src])


# ----------------------------------------------------------------------------------------------
# sequences of unequal length
# ----------------------------------------------------------------------------------------------
@dataclass
class PagedContext:
    """Handle to one layer of a ``PagedKVCache`` for one call: ``k_pages``/``v_pages`` ``[pages, H, page_size, D]`` (views), the
    cache's ``page_table``, the ``positions`` of the call's tokens and, for a prompt, the sequences (``rows``) that they belong to;
    for a step the sequences' lengths with the new token (``lens``); for a step over trees of drafted tokens the ``tree``, whose positions and rows those of the call
    are, how many ``nodes`` of it there are, and the lengths of the contexts (``lens``)."""
    k_pages: Tensor
    v_pages: Tensor
    page_table: Tensor
    positions: Tensor
    lens: Optional[Tensor]
    rows: Optional[Tensor]
    status: Optional[Tensor]
    window: Optional[int]
    tree: Optional["DraftTree"] = None
    nodes: Optional[Tensor] = None


class PagedKVCache:
    """A key-value cache for sequences of unequal length that come and go (the reference's cache has one position for the whole
    batch, inference/kv_cache.py:4-68).

    Storage is a pool of ``pages`` pages, ``k, v [L, pages, H, page_size, D]`` (bf16 or fp16); each of the ``sequences`` slots owns the pages
    that its row of ``page_table`` names, for up to ``max_len`` positions.  A step runs all slots at once; free ones are
    skipped.  With ``window``, pages that no step can see any more go back to the pool as a sequence crosses into another page; a prompt takes
    pages for all of its positions, which its own attention sees, so a pool has to hold the longest prompts whole.

    A step may run a tree of drafted tokens per sequence instead of one token: ``begin_draft`` makes room behind each context, ``accept`` keeps the nodes of the accepted
    path (``core.draft_step``).  ``fork`` gives a sequence's positions to others that go on from there: they share its full pages, which nobody writes again.

    The host knows every length, so that ``admit`` and ``begin_step`` raise where the pool is empty; the device has the table, the next token's
    ``positions`` (-1 for a free slot) and the ``lens`` with it, at fixed addresses, for steps recorded in a HIP graph.  Changes go to the
    device on the current stream: admissions, releases and steps of one cache belong on the same one.
    """

    def __init__(self, L, sequences, H, D, pages, device, dtype, page_size: int = 64, max_len: int = 65536, window: Optional[int] = None):
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"a paged cache holds bfloat16 or float16, got {dtype}")
        if page_size <= 0 or page_size % 16 != 0:
            raise ValueError(f"page_size must be a multiple of 16, got {page_size}")
        if min(L, sequences, H, D, pages, max_len) <= 0 or (window is not None and window <= 0):
            raise ValueError("a paged cache needs positive sizes")
        self.L, self.sequences, self.H, self.D, self.pages, self.page_size = L, sequences, H, D, pages, page_size
        self.max_len, self.window, self.device, self.dtype = max_len, window, device, dtype
        self.k = torch.empty((L, pages, H, page_size, D), device=device, dtype=dtype)
        self.v = torch.empty_like(self.k)
        width = -(-max_len // page_size)
        self.page_table = torch.full((sequences, width), -1, device=device, dtype=torch.int32)
        self.positions = torch.full((sequences,), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(sequences, device=device, dtype=torch.int32)
        self.status = torch.zeros(1, device=device, dtype=torch.int32)      # raised by the kernels, see check()
        self._live = torch.zeros(sequences, device=device, dtype=torch.int32)
        self._free = list(range(pages - 1, -1, -1))
        self._length: List[Optional[int]] = [None] * sequences               # None: a free slot
        self._owned: List[Dict[int, int]] = [{} for _ in range(sequences)]    # entry of the table -> page
        self._users: List[int] = [0] * pages                                 # slots that own each page
        self._reach: List[int] = [0] * sequences                             # entries that each slot has taken so far
        self._drafted: Optional[List[int]] = None                            # nodes of each slot's tree that accept() has not had yet
        self._changes: Dict[int, int] = {}                                   # flat entry -> page, not on the device yet

    # -- what there is -----------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, slot: int) -> Optional[int]:
        """Positions of a sequence, ``None`` for a free slot."""
        return self._length[slot]

    @property
    def longest(self) -> int:
        """Positions of the longest sequence, 0 where there is none."""
        return max((n for n in self._length if n is not None), default=0)

    def check(self) -> None:
        """Raises what the kernels reported since the last time (a page that is none, say).  Synchronises."""
        from . import ops
        try:
            ops.raise_for_status(self.status)
        except RuntimeError:
            self.status.zero_()
            raise

    # -- slots and pages -----------------------------------------------------------------------
    def _take(self, wanted: Dict[int, range], left: Dict[int, List[int]]) -> None:
        """Gives every slot the entries that it wants and takes those that it has left behind, or raises and changes nothing."""
        dropped: Dict[int, int] = {}
        for slot, entries in left.items():
            for entry in entries:
                page = self._owned[slot][entry]
                dropped[page] = dropped.get(page, 0) + 1
        count, back = sum(len(e) for e in wanted.values()), sum(n == self._users[page] for page, n in dropped.items())
        if count > len(self._free) + back:
            raise RuntimeError(f"the paged cache is full: {count} pages wanted, {len(self._free) + back} of {self.pages} free")
        for slot, entries in left.items():
            for entry in entries:
                self._set(slot, entry, -1)
        for slot, entries in wanted.items():
            for entry in entries:
                self._set(slot, entry, self._free.pop())
            self._reach[slot] = entries.stop

    def _set(self, slot: int, entry: int, page: int) -> None:
        if page < 0:
            old = self._owned[slot].pop(entry)
            self._users[old] -= 1
            if self._users[old] == 0:
                self._free.append(old)
        else:
            self._owned[slot][entry] = page
            self._users[page] += 1
        self._changes[slot * self.page_table.shape[1] + entry] = page

    def _upload(self) -> None:
        """The table's changes, in one copy that the host does not wait for."""
        if not self._changes:
            return
        both = torch.tensor([list(self._changes.keys()), list(self._changes.values())], dtype=torch.int64, pin_memory=self.page_table.is_cuda)
        both = both.to(self.page_table.device, non_blocking=True)
        self.page_table.view(-1).scatter_(0, both[0], both[1].to(torch.int32))
        self._changes.clear()

    def admit(self, lengths: List[int]) -> List[int]:
        """Free slots for new sequences of these many positions each, with pages for them: the slots, in order.  The positions are
        to be filled (``ops.paged_append``, ``core.admit``) before the next step."""
        if not lengths:
            return []
        slots = [s for s, n in enumerate(self._length) if n is None][:len(lengths)]
        if len(slots) < len(lengths):
            raise RuntimeError(f"the paged cache has {len(slots)} free slots for {len(lengths)} sequences")
        for n in lengths:
            if not 0 < n <= self.max_len:
                raise ValueError(f"a sequence must have 1 to {self.max_len} positions, got {n}")
        self._take({s: range(-(-n // self.page_size)) for s, n in zip(slots, lengths)}, {})
        self._upload()
        self._open(slots, lengths)
        return slots

    def _open(self, slots: List[int], lengths: List[int]) -> None:
        for s, n in zip(slots, lengths):
            self._length[s] = n
        at = torch.tensor(slots, device=self.page_table.device)
        self.positions[at] = torch.tensor(lengths, dtype=torch.int32, device=self.page_table.device)
        self.lens[at] = self.positions[at] + 1
        self._live[at] = 1

    def fork(self, slot: int, count: int = 1) -> List[int]:
        """Free slots for ``count`` sequences that begin with the positions of the one in ``slot``: the slots, in order.  Full pages are shared from then on; of the last
        one, where it is not full, each gets a copy."""
        from . import ops
        n = self._length[slot]
        if n is None:
            raise ValueError(f"slot {slot} has no sequence")
        if count <= 0:
            raise ValueError(f"a sequence forks into one more or several, not {count}")
        if self._drafted is not None:
            raise RuntimeError("accept() has not had the last draft's path yet")
        slots = [s for s, m in enumerate(self._length) if m is None][:count]
        if len(slots) < count:
            raise RuntimeError(f"the paged cache has {len(slots)} free slots for {count} sequences")
        full, rest = divmod(n, self.page_size)
        self._take({s: range(full, full + (rest > 0)) for s in slots}, {})
        try:
            for s in slots:
                for entry, page in self._owned[slot].items():
                    if entry < full:
                        self._set(s, entry, page)
            self._upload()
            if rest:
                copied = torch.zeros((3, self.sequences), dtype=torch.int32)
                copied[2] = slot
                copied[0, slots], copied[1, slots] = full * self.page_size, rest
                starts, counts, sources = copied.to(self.page_table.device)
                ops.paged_move(self.k, self.v, self.page_table, starts, counts, rows=self.page_size, sources=sources, status=self.status)
        except BaseException:
            for s in slots:
                for entry in list(self._owned[s]):
                    self._set(s, entry, -1)
                self._reach[s] = 0
            self._upload()
            raise
        self._open(slots, [n] * count)
        return slots

    def release(self, slot: int) -> None:
        """Ends a sequence: its pages go back, later steps skip the slot."""
        if self._length[slot] is None:
            raise ValueError(f"slot {slot} has no sequence")
        for entry in list(self._owned[slot]):
            self._set(slot, entry, -1)
        self._length[slot], self._reach[slot] = None, 0
        if self._drafted is not None:
            self._drafted[slot] = 0
        self._upload()
        self.positions[slot], self.lens[slot], self._live[slot] = -1, 0, 0

    def begin_step(self) -> None:
        """Makes room for one more position of every sequence, from the pages that a window has left behind and the pool."""
        if self._drafted is None:
            size, most = self.page_size, self.max_len
            for slot, n in enumerate(self._length):
                if n is not None and (n >= self._reach[slot] * size or n >= most):
                    break
            else:
                return      # (as in most steps)
        self._make_room([1] * self.sequences)

    def begin_draft(self, nodes: List[int]) -> None:
        """Makes room for a tree of ``nodes[slot]`` drafted tokens behind every sequence (free slots have none), as ``begin_step`` for one token.  ``accept`` ends
        the draft."""
        if len(nodes) != self.sequences or min(nodes) < 0:
            raise ValueError(f"a draft needs how many nodes each of the {self.sequences} slots has, got {nodes}")
        self._make_room(nodes)
        self._drafted = [0 if n is None else m for n, m in zip(self._length, nodes)]

    def _make_room(self, more: List[int]) -> None:
        if self._drafted is not None:
            raise RuntimeError("accept() has not had the last draft's path yet")
        wanted, left = {}, {}
        for slot, (n, m) in enumerate(zip(self._length, more)):
            if n is None or m == 0:
                continue
            if n + m > self.max_len:
                raise RuntimeError(f"the sequence in slot {slot} has reached {n} of {self.max_len} positions, {m} more are wanted")
            if n + m > self._reach[slot] * self.page_size:
                wanted[slot] = range(self._reach[slot], (n + m - 1) // self.page_size + 1)
                if self.window is not None:
                    left[slot] = [e for e in self._owned[slot] if (e + 1) * self.page_size <= n + 1 - self.window]
        if wanted:
            self._take(wanted, left)
            self._upload()

    def accept(self, path: Tensor, counts: Tensor) -> List[int]:
        """Ends a draft: the first ``counts[slot]`` nodes of ``path[slot]`` (``ops.verify_drafts``; [sequences, M] and [sequences], int32, on the device) become the next positions of each
        sequence, in all layers; the other nodes are forgotten.  Returns the counts, for which the host waits (0 for
        free slots, whatever theirs say).  (A row of ``path`` that does not rise leaves its positions as
        they were and is reported by ``check``.)"""
        from . import ops
        if self._drafted is None:
            raise RuntimeError("there is no draft: begin_draft() comes first")
        if path.dim() != 2 or path.shape[0] != self.sequences or counts.shape != (self.sequences,):
            raise ValueError(f"path and counts must be [{self.sequences}, M] and [{self.sequences}], got {tuple(path.shape)} and {tuple(counts.shape)}")
        taken = [0 if n is None else c for c, n in zip(counts.tolist(), self._length)]
        for slot, (n, m) in enumerate(zip(taken, self._drafted)):
            if not 0 <= n <= min(m, path.shape[1]):
                raise ValueError(f"{n} of the {min(m, path.shape[1])} nodes of slot {slot} cannot be accepted")
        ops.paged_move(self.k, self.v, self.page_table, self.positions, counts, index=path, status=self.status)
        counts = counts * self._live
        self.positions.add_(counts)
        self.lens.add_(counts)
        self._length = [None if n is None else n + more for n, more in zip(self._length, taken)]
        self._drafted = None
        return taken

    def forget_draft(self) -> None:
        """Ends a draft of which nothing is accepted."""
        self._drafted = None

    def advance(self, on_device: bool = True) -> None:
        """Every sequence has one position more.  ``on_device=False``: the device has counted already (a recorded step)."""
        if on_device:
            self.count_on_device()
        self._length = [None if n is None else n + 1 for n in self._length]

    def count_on_device(self) -> None:
        self.positions.add_(self._live)
        self.lens.add_(self._live)

    # -- handles --------------------------------------------------------------------------------
    def context(self, layer: int, positions: Optional[Tensor] = None, rows: Optional[Tensor] = None, tree: Optional["DraftTree"] = None,
                nodes: Optional[Tensor] = None) -> PagedContext:
        """The layer for a step of all slots, for a prompt's tokens at ``positions`` of sequences ``rows``, or for a step over a ``tree`` (``ops.draft_tree``)."""
        if tree is not None:
            return PagedContext(self.k[layer], self.v[layer], self.page_table, tree.positions, self.positions, tree.rows, self.status, self.window, tree, nodes)
        if positions is None:
            return PagedContext(self.k[layer], self.v[layer], self.page_table, self.positions, self.lens, None, self.status, self.window)
        return PagedContext(self.k[layer], self.v[layer], self.page_table, positions, None, rows, self.status, self.window)
