"""The page operators one entry at a time on numpy arrays (test
infrastructure): every rule is evaluated on the state before the call."""

from __future__ import annotations

import numpy as np


def _up(n, bs):
    return -(-n // bs)


def copy(caches, src, dst):
    nb = caches[0].shape[0]
    old = [c.copy() for c in caches]
    real = [0 <= s < nb and 0 <= d < nb for s, d in zip(src, dst)]
    status = []
    for i, (s, d) in enumerate(zip(src, dst)):
        ok = real[i]
        if ok and s != d:
            for j in range(len(src)):
                if j != i and real[j] and src[j] != dst[j] and (src[j] == d or (j > i and dst[j] == d)):
                    ok = False
        status.append(int(ok))
        if ok:
            for c, o in zip(caches, old):
                c[d] = o[s]
    return status


def fork(tables, lengths, refs, parents, children, bs):
    rows, width = tables.shape
    was = lengths.copy()
    status, seen = [], set()
    for p, c in zip(parents, children):
        ok = 0 <= p < rows and 0 <= c < rows and c not in seen and p not in list(children)
        ok = ok and was[c] == 0 and 0 <= was[p] <= width * bs
        seen.add(c)
        status.append(int(ok))
        if ok:
            n = _up(was[p], bs)
            tables[c, :n] = tables[p, :n]
            for page in tables[p, :n]:
                if 0 <= page < len(refs):
                    refs[page] += 1
            lengths[c] = was[p]
    return status


def free(tables, lengths, refs, seqs, bs, new_lengths=None):
    rows, width = tables.shape
    status, seen = [], set()
    for i, s in enumerate(seqs):
        keep = 0 if new_lengths is None else new_lengths[i]
        ok = 0 <= s < rows and s not in seen and 0 <= keep <= lengths[s]
        seen.add(s)
        status.append(int(ok))
        if ok:
            for j in range(_up(keep, bs), min(_up(lengths[s], bs), width)):
                page = tables[s, j]
                if 0 <= page < len(refs):
                    refs[page] = max(refs[page] - 1, 0)
            lengths[s] = keep
    return status


def extend(caches, tables, lengths, refs, seqs, new_lengths, bs):
    rows, width = tables.shape
    free_pages = [int(p) for p in np.flatnonzero(refs <= 0)]
    was, held = lengths.copy(), refs.copy()
    listed, shared_before, given, short = set(), {}, 0, False
    status, copies = [], []
    for s, want in zip(seqs, new_lengths):
        ok = 0 <= s < rows and s not in listed and 0 <= was[s] <= want <= width * bs
        listed.add(s)
        if not ok:
            status.append(0)
            continue
        n = was[s]
        need, part = _up(want, bs) - _up(n, bs), -1
        if want > n and n % bs and 0 <= tables[s, n // bs] < len(refs) and held[tables[s, n // bs]] > 1:
            page = int(tables[s, n // bs])
            if shared_before.get(page, 0) < held[page] - 1:
                part, need = page, need + 1
            shared_before[page] = shared_before.get(page, 0) + 1
        start, given = given, given + need
        short = short or given > len(free_pages)
        status.append(int(not short))
        if short:
            continue
        got = free_pages[start:given]
        first = n // bs if part >= 0 else _up(n, bs)
        tables[s, first : first + need] = got
        refs[got] = 1
        if part >= 0:
            refs[part] -= 1
            copies.append((part, got[0]))
        lengths[s] = want
    for a, b in copies:
        for c in caches:
            c[b] = c[a]
    return status


def compact(caches, tables, lengths, refs, bs):
    """(tables, refs, map, live); the caches change in place."""
    nb = len(refs)
    held = refs > 0
    live = int(held.sum())
    high = [p for p in range(live, nb) if held[p]]
    holes = [p for p in range(live) if not held[p]]
    where = np.where(held, np.arange(nb), -1).astype(np.int32)
    new_refs = np.where(np.arange(nb) < live, np.maximum(refs, 0), 0).astype(np.int32)
    for a, b in zip(high, holes):
        where[a] = b
        new_refs[b] = refs[a]
        for c in caches:
            c[b] = c[a]
    out = tables.copy()
    for r, n in enumerate(lengths):
        for j in range(min(_up(max(n, 0), bs), tables.shape[1])):
            if 0 <= tables[r, j] < nb:
                out[r, j] = where[tables[r, j]]
    return out, new_refs, where, live
