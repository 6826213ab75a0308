"""
Which sequences of a batch share leading pages.

``RadixCache`` gives sequences with a common prompt prefix the same physical
blocks for it, so their block tables start alike. ``SharedPrefix`` names such
families for ``B200PagedBackend.plan_shared`` / ``attend_shared``, which read a
family's shared pages once instead of once per sequence.
"""

from __future__ import annotations

from typing import Sequence

__all__ = ["SharedPrefix"]


class SharedPrefix:
    """Consecutive families of a batch: family ``g`` is the next
    ``group_sizes[g]`` sequences, which share their first ``prefix_pages[g]``
    pages (0: none). The shared pages must lie before every member's new tokens:
    ``prefix_pages[g] * page_size <= kv_len - query_len``."""

    def __init__(self, group_sizes: Sequence[int], prefix_pages: Sequence[int]):
        self.group_sizes = [int(x) for x in group_sizes]
        self.prefix_pages = [int(x) for x in prefix_pages]
        if not self.group_sizes:
            raise ValueError("SharedPrefix needs at least one group")
        if len(self.group_sizes) != len(self.prefix_pages):
            raise ValueError(f"{len(self.group_sizes)} groups but {len(self.prefix_pages)} prefix lengths")
        if min(self.group_sizes) < 1:
            raise ValueError("every group must hold at least one sequence")
        if min(self.prefix_pages) < 0:
            raise ValueError("prefix_pages must be >= 0")

    @property
    def n_seqs(self) -> int:
        return sum(self.group_sizes)

    @classmethod
    def from_tables(cls, block_tables: Sequence[Sequence[int]], kv_lens: Sequence[int], query_lens: Sequence[int],
                    page_size: int) -> "SharedPrefix":
        """Families among consecutive sequences, from their block tables: a
        sequence joins the family before it when that keeps at least as many
        page reads saved ((members - 1) x shared pages)."""
        n = len(block_tables)
        if n == 0 or len(kv_lens) != n or len(query_lens) != n:
            raise ValueError(f"{n} block tables, {len(kv_lens)} kv lengths and {len(query_lens)} query lengths")
        sizes: list[int] = []
        shared: list[int] = []
        first: Sequence[int] = ()
        for table, kv, q in zip(block_tables, kv_lens, query_lens):
            own = max(0, (int(kv) - int(q)) // page_size)  # whole pages before the new tokens
            if sizes:
                most = min(own, shared[-1])
                p = 0
                while p < most and table[p] == first[p]:
                    p += 1
                if p and sizes[-1] * p >= (sizes[-1] - 1) * shared[-1]:
                    sizes[-1] += 1
                    shared[-1] = p
                    continue
            sizes.append(1)
            shared.append(own)
            first = table
        return cls(sizes, [p if s > 1 else 0 for s, p in zip(sizes, shared)])

    def __repr__(self) -> str:
        return f"SharedPrefix(group_sizes={self.group_sizes}, prefix_pages={self.prefix_pages})"
