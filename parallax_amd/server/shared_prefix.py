"""Which rows of a decode batch share leading pages of the cache, and whether attention
that reads such pages once for all of them pays.

Requests whose prompts begin alike hold the same pages at the head of their block tables
(radix_cache.py hands them out). ops.shared_prefix_attention_decode() takes what is found
here: a group per row and a length per group.
"""

from __future__ import annotations

from typing import List, Sequence, Tuple

import numpy as np

from .kv_cache import KVCacheSpec

# Bytes of keys and values a layer that must be saved before the shared form is taken. It
# plans on the device and joins its parts in a second launch, some 10 us a layer where the
# plain form starts with 6, and the plain form also rotates and stores in its launch. In
# replayed graphs, us, without that, for rows of up to 1,000 tokens of their own behind
# the prefix, bf16: 32 query heads over 8 of 128, 16 rows over 1,024 tokens (63 MB saved)
# 18.6 shared, 17.5 plain; over 2,048 (126 MB) 19.0, 20.8; 64 rows over 1,024 (264 MB)
# 30.2, 35.9; over 2,048 (528 MB) 31.7, 47.1; 256 over 8,000 (8.4 GB) 99.6, 425. 64 over 8
# of 64, 64 rows over 2,048 (264 MB) 23.3, 29.3; 14 over 2 of 64, 256 over 2,048 (267 MB)
# 22.6, 28.0. Whole decode steps, four layers of 8B's sizes, ms: 64 requests behind 1,024
# shared tokens (264 MB) 1.006 shared, 0.996 plain; 2,048 (528 MB) 1.008, 1.061; 128 behind
# 4,000 (2 GB) 1.497, 1.850; 256 behind 8,000 (8.4 GB) 2.460, 3.984.
# With fused_head_norms the plain form does not store in its launch, and the shared one
# passes it sooner, by the first figures from some 128 MB on; one limit serves both.
LEAST_BYTES = 384 << 20
MAX_GROUPS = 32    # as many as a graph's buffers hold; those that save most are kept
MAX_ROWS = 4096    # the kernel's own limit


def find_shared_prefixes(tables: Sequence, seq_lens: Sequence[int],
                         block_size: int, max_groups: int = MAX_GROUPS,
                         ) -> Tuple[List[int], List[int]]:
    """(the group of every row, -1: none; the tokens that each group's rows share).

    A group of n rows over t tokens saves t * (n - 1) tokens' reads, and what is returned
    saves the most. Rows that share a page share all pages before it, so the rows form a
    tree of common heads. A row joins one of the nodes above it, best the deepest that is
    a group, so that best[v][k], what the rows below v save if the k-th of the nodes
    above it is the next group up (0: none), follows from the nodes below: a row left to
    that group counts in full there, and a group takes off the one read of its own.
    Only whole pages that lie within every row's length count."""
    rows = len(tables)
    whole = [min(len(t), n // block_size) for t, n in zip(tables, seq_lens)]
    if rows < 2:
        return [-1] * rows, []
    pages = np.full((rows, max(whole) + 1), -1, dtype=np.int64)
    for i, (t, w) in enumerate(zip(tables, whole)):
        pages[i, :w] = t[:w]
        pages[i, w] = -2 - i     # a head that ends is followed by no one else's page
    # of every node, each behind the one above it: the pages shared, the rows and the
    # nodes right below, the nodes above
    depth_of, rows_of, below, above = [], [], [], []
    todo = [(np.arange(rows), 0, [])]
    while todo:
        members, depth, path = todo.pop()
        same = pages[members, depth:] == pages[members[0], depth:]
        # the first column in which a row differs from the first one
        depth += int(np.where(same.all(1), same.shape[1], same.argmin(1)).min())
        here = len(depth_of)
        depth_of.append(depth)
        rows_of.append([])
        below.append([])
        above.append(path)
        if path:
            below[path[-1]].append(here)
        heads = pages[members, depth]
        for head in np.unique(heads):
            part = members[heads == head]
            if len(part) > 1:
                todo.append((part, depth + 1, path + [here]))
            else:
                rows_of[here].append(int(part[0]))
    best, opens = [None] * len(below), [None] * len(below)
    for v in range(len(below) - 1, -1, -1):
        depth = depth_of[v]
        saved = len(rows_of[v]) * np.array([0] + [depth_of[u] for u in above[v]] + [depth])
        for u in below[v]:
            saved += best[u]
        opens[v] = saved[-1] - depth > saved[:-1]
        best[v] = np.maximum(saved[-1] - depth, saved[:-1])
    joins, members_of = [0] * len(below), {}
    for v in range(len(below)):
        k = joins[v]
        if opens[v][k]:
            k = len(above[v]) + 1
        for u in below[v]:
            joins[u] = k
        if k and rows_of[v]:
            members_of.setdefault((above[v] + [v])[k - 1], []).extend(rows_of[v])
    groups = sorted(members_of.items(), key=lambda g: -depth_of[g[0]] * (len(g[1]) - 1))
    group_of = [-1] * rows
    for g, (_, members) in enumerate(groups[:max_groups]):
        for row in members:
            group_of[row] = g
    return group_of, [depth_of[v] * block_size for v, _ in groups[:max_groups]]


class SharedPrefixes:
    """find_shared_prefixes() of the batch at hand, and nothing where too little would be
    saved: found again when the rows change, and kept for the last BATCHES batches, which
    a pipeline's stages go through in turn."""

    BATCHES = 8

    def __init__(self, spec: KVCacheSpec, least_bytes: int = LEAST_BYTES):
        token = 2 * spec.num_kv_heads * spec.head_dim * spec.dtype.itemsize
        self.least_tokens = -(-least_bytes // token)
        self.block_size = spec.block_size
        # of each batch its tables, the same as arrays (which take long to convert) and
        # what was found; the latest first
        self._batches: List[tuple] = []

    def find(self, tables, seq_lens):
        """(groups, lengths) as above, or None. A table only grows while its request
        lives, so the same tables share the same pages; held, none is taken for another."""
        for i, batch in enumerate(self._batches):
            if len(batch[0]) == len(tables) and all(
                    a is b for a, b in zip(batch[0], tables)):
                if i:
                    self._batches.insert(0, self._batches.pop(i))
                return batch[2]
        known = {id(t): p for kept, pages, _ in reversed(self._batches)
                 for t, p in zip(kept, pages)}
        pages = [self._extended(known.get(id(t)), t) for t in tables]
        found = self._worthwhile(pages, seq_lens) if len(tables) <= MAX_ROWS else None
        self._batches = [(list(tables), pages, found)] + self._batches[:self.BATCHES - 1]
        return found

    def _worthwhile(self, pages, seq_lens):
        groups, lens = find_shared_prefixes(pages, seq_lens, self.block_size)
        rows = [0] * len(lens)
        for g in groups:
            if g >= 0:
                rows[g] += 1
        saved = sum(t * (n - 1) for t, n in zip(lens, rows))
        return (groups, lens) if saved >= max(1, self.least_tokens) else None

    @staticmethod
    def _extended(pages, table) -> np.ndarray:
        """A table as an array, from that of an earlier step if there is one."""
        if pages is None:
            return np.array(table, dtype=np.int64)
        if len(pages) < len(table):
            return np.concatenate([pages, np.array(table[len(pages):], dtype=np.int64)])
        return pages
