"""Page accounting of the paged K/V caches (``pa_pages_*`` in the C ABI).

The reference builds its block tables in test code (``tests/correctness.py:26-36``).
A serving loop takes pages as rows grow, gives them back as rows end or their
tokens leave a sliding window, shares them between continuations of one prompt
and, now and then, moves the live ones together. ``PagePool`` does this on the
device: counts, free bits, block tables and lengths are tensors that its calls
change in place, asynchronously on the current stream, without a host round
trip, so that they can stand in a captured graph beside the attention they serve.

One pool's calls must be ordered (one stream, or events between streams): they
share its state and scratch.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _native
from .torch_kernel import window_args

Caches = Union[torch.Tensor, Sequence[torch.Tensor]]


def int32_vector(who: str, x: torch.Tensor) -> torch.Tensor:
    """``x`` as the contiguous int32 that the calls take. int64 values beyond int32
    become its ends, which no table holds, instead of small numbers."""
    if x.dtype == torch.int64:
        x = x.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    elif x.dtype != torch.int32:
        raise ValueError(f"{who}: lengths and rows must be int32 or int64 tensors")
    return x.contiguous()


class PagePool:
    """The pages that the caches of one or more layers share: page ``i`` is
    ``cache[i]`` of every ``[num_blocks, block_size, Hkv, D]`` cache given.

    * ``refs``: int32 ``[num_blocks]``, users of each page, 0 for a free one,
    * ``free_words``: int32 bit mask of the free pages,
    * ``state``: both in one buffer (a snapshot is ``state.clone()``),
    * ``status``: a device word that the calls OR ``PA_STATUS_*`` bits into.

    All pages start out free.
    """

    def __init__(self, k_caches: Caches, v_caches: Caches):
        ks = [k_caches] if isinstance(k_caches, torch.Tensor) else list(k_caches)
        vs = [v_caches] if isinstance(v_caches, torch.Tensor) else list(v_caches)
        if not ks or not vs:
            raise ValueError("PagePool: at least one layer's caches are needed")
        if ks[0].dim() != 4:
            raise ValueError("PagePool: caches must be [num_blocks, block_size, Hkv, D]")
        self.device = ks[0].device
        if self.device.type != "cuda":
            raise ValueError("PagePool: the pool's caches must be CUDA tensors")
        self.num_blocks, self.block_size = ks[0].shape[:2]
        self._pool = _native.ext().PagePool(ks, vs, self.num_blocks, self.block_size, self.device)
        self.state = self._pool.state
        self.refs = self._pool.refs
        self.free_words = self._pool.free_words
        self.status = self._pool.status

    def adopt(self, block_table: torch.Tensor, seq_lens: torch.Tensor) -> None:
        """Take over tables made elsewhere: the pages that ``block_table``'s rows use
        (entries ``j < ceil(seq_lens / block_size)`` that are not -1) get their
        counts, all others become free. Raises (after a host read) if an entry in use
        is no page of the pool or a length exceeds the table."""
        status = int(self._pool.adopt(block_table, seq_lens).item())
        if status & _native.PA_STATUS_BAD_BLOCK:
            raise ValueError("PagePool.adopt: Block_Table names pages outside the pool")
        if status:
            raise ValueError("PagePool.adopt: seq_lens exceeds the Block_Table capacity")

    def resize(self, block_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, *,
               window: Optional[int] = None, num_sinks: int = 0) -> None:
        """Rows go from ``seq_lens`` to ``new_lens`` tokens (int32 ``[rows]``; negative:
        the row is left alone; 0 frees it), in place in ``block_table`` and ``seq_lens``.

        Pages behind the new length are released, and with a ``window`` those that
        hold no token visible to the next queries (positions ``min(old, new)`` and
        later) nor one of the first ``num_sinks``; their entries become -1. Growing
        rows then take the pages they miss, lowest first, in row order, each row all
        of them or none (``PA_STATUS_NO_PAGES``: its length stays, as does that of later
        rows that need pages). A partly filled last page that a growing row shares is
        replaced by a copy of its used slots."""
        win, sinks = window_args("PagePool.resize", window, num_sinks)
        if new_lens.dtype != torch.int32 or not new_lens.is_contiguous():
            new_lens = int32_vector("PagePool.resize", new_lens)
        self._pool.resize(block_table, seq_lens, new_lens, win, sinks)

    def fork(self, block_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor,
             children: torch.Tensor) -> None:
        """Row ``children[i]`` (empty: length 0) continues row ``parents[i]``: full pages
        are shared, the used slots of the partly filled last page are copied to a new
        page in every layer. A negative index skips the pair. ``PA_STATUS_BAD_ROW``: a
        row outside the table, a child that is not empty, or named before;
        ``PA_STATUS_NO_PAGES``: no page for the copy, the child stays empty."""
        parents, children = (x if x.dtype == torch.int32 and x.is_contiguous()
                             else int32_vector("PagePool.fork", x) for x in (parents, children))
        self._pool.fork(block_table, seq_lens, parents, children)

    def compact(self, block_table: torch.Tensor) -> torch.Tensor:
        """Moves the live pages into the front of the pool in every layer and rewrites
        ``block_table`` (which must hold every row that uses the pool). Returns their
        number, an int32 ``[1]`` on the device: pages from there on are free."""
        return self._pool.compact(block_table)

    def read_status(self) -> int:
        """Host read of the status word (synchronises the device)."""
        return int(self.status.item())
