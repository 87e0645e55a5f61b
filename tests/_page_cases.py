"""Pools, tables and caches for the page operators' tests."""

from __future__ import annotations

import numpy as np
import torch


def make_pool(rows=8, width=6, pages=64, bs=16, fill=4, seed=0, empty=2, share=0.3):
    """(tables, lengths, refs): rows of up to ``fill`` pages, some pages held by
    several rows (a common beginning); the last ``empty`` rows are empty and
    entries that no row uses hold numbers outside the pool."""
    rng = np.random.default_rng(seed)
    names = rng.permutation(pages)
    tables = rng.integers(-5, pages + 5, (rows, width)).astype(np.int32)
    tables[rng.random((rows, width)) < 0.5] = 2**30
    lengths, refs, n = np.zeros(rows, np.int32), np.zeros(pages, np.int32), 0
    for r in range(rows - empty):
        k = int(rng.integers(0, fill + 1))
        first = []
        if r and rng.random() < share:
            other = int(rng.integers(0, r))
            first = list(tables[other, : min(-(-int(lengths[other]) // bs), k)])
        own = list(names[n : n + k - len(first)])
        if len(own) < k - len(first):
            break
        n += len(own)
        row = first + own
        tables[r, : len(row)] = row
        refs[row] += 1
        lengths[r] = 0 if not row else (len(row) - 1) * bs + int(rng.integers(1, bs + 1))
    return tables, lengths, refs


def make_caches(pages, shapes, seed=0):
    """Tensors [pages, *shape]; a shape's first entry names its dtype."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for dt, *shape in shapes:
        x = torch.randint(0, 256, (pages, int(np.prod(shape)) * torch.empty(0, dtype=dt).element_size()), generator=gen,
                          dtype=torch.uint8)
        out.append(x.view(dt).view(pages, *shape))
    return out
