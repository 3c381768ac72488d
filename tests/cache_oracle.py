"""Pages, their tables and plain forms of what reads and writes them.  CPU only."""
from __future__ import annotations

import itertools

import torch

from sequence_oracle import attend64


def ints(values):
    return torch.tensor(values, dtype=torch.int32)


def offsets_of(lengths):
    return ints([0, *itertools.accumulate(lengths)])


def tables(lk, page, prefix=0, spare=3, seed=0):
    """(table, number of pages): the samples' pages in no order, the first
    ``prefix`` of them shared, ``spare`` others free.  Entries beyond a sample's
    length name no page that there is."""
    need = [max(0, -(-n // page) - prefix) for n in lk]
    total = prefix + sum(need) + spare
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lk), prefix + max([*need, 1])), -7, dtype=torch.int32)
    at = prefix
    for b, n in enumerate(need):
        table[b, :prefix] = ints(ids[:prefix])
        table[b, prefix:prefix + n] = ints(ids[at:at + n])
        table[b, prefix + n:] = (1 << 30) if b % 2 else -7
        at += n
    return table, total


def gather(pages, table, b, n):
    """Rows 0 to n of sample b."""
    j = torch.arange(n)
    return pages[table[b].long()[j // pages.shape[1]], j % pages.shape[1]]


def scatter(pages, table, b, rows, first):
    """Writes rows at positions first, first + 1, ... of sample b."""
    j = torch.arange(first, first + len(rows))
    pages[table[b].long()[j // pages.shape[1]], j % pages.shape[1]] = rows


def attend_pages64(q, k_pages, v_pages, table, lq, lk, window, sinks, scale=None):
    """The result and the bound on its error, from attend64's over gathered rows."""
    k = torch.cat([gather(k_pages, table, b, n) for b, n in enumerate(lk)])
    v = torch.cat([gather(v_pages, table, b, n) for b, n in enumerate(lk)])
    return attend64(q, k, v, lq, lk, window, sinks, scale)
