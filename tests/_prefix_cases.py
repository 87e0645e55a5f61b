"""Batches with shared prefixes, for the CPU and GPU tests."""

from __future__ import annotations

import math

import numpy as np
import torch

FP8 = torch.float8_e4m3fn


def make_prefix_case(groups, loose=(), *, ql=1, heads=8, kv_heads=2, page=16, head=128, per_token=False,
                     dtype=torch.bfloat16, trans=True, seed=0, spare_pages=3, poison=True, extra_cols=0):
    """groups: [(prefix length, [context length of each sequence])]; loose:
    context lengths of the sequences behind them.  A group's full prefix pages
    are the same pages in every row; the page that a prefix ends in is each
    row's own, with other bytes behind the context (``poison``: NaN there and
    in the pages that no sequence holds)."""
    rng = np.random.default_rng(seed)
    first_own = []  # first page of a row that is the row's alone
    gen = torch.Generator().manual_seed(seed)
    ctx, indptr, prefix, rows, copies, n = [], [0], [], [], [], 0
    for p, lens in list(groups) + ([(0, list(loose))] if loose else []):
        full, part = divmod(p, page)
        shared = list(range(n, n + full))
        n += full
        for j, c in enumerate(lens):
            more = max(-(-max(c, p if j == 0 else c) // page), full) - full
            rows.append(shared + list(range(n, n + more)))
            first_own.append(full)
            if part and j and c > full * page:
                copies.append((rows[len(rows) - 1 - j][full], n))
            n += more
            ctx.append(c)
        if not (loose and p == 0 and lens == list(loose)):
            prefix.append(p)
            indptr.append(len(ctx))
    nb = n + spare_pages
    names = rng.permutation(nb)
    width = max([len(r) for r in rows] + [1]) + extra_cols
    tables = np.zeros((len(rows), width), np.int32)
    for b, r in enumerate(rows):
        tables[b, : len(r)] = names[r]
    shape = (nb, kv_heads, page, head)
    kf, vf = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)
    if per_token:
        ks, vs = (x.abs().amax(-1, keepdim=True) / 448 for x in (kf, vf))
    else:
        ks, vs = (x.abs().amax().reshape(1) / 448 for x in (kf, vf))
    k, v = ((x / s).to(FP8).view(torch.uint8) for x, s in ((kf, ks), (vf, vs)))
    for a, c in copies:
        for t in (k, v) + ((ks, vs) if per_token else ()):
            t[names[c]] = t[names[a]]
    if poison:  # the last page of a row behind its tokens, and unheld pages
        for b, r in enumerate(rows):
            held = max(ctx[b], next((p for g, p in enumerate(prefix) if indptr[g] == b), 0))
            if held % page and held // page >= first_own[b]:  # (a shared page's tokens are other rows' too)
                k[names[r[held // page]], :, held % page:] = 0x7F
                v[names[r[held // page]], :, held % page:] = 0xFF
                if per_token:
                    ks[names[r[held // page]], :, held % page:] = float("nan")
                    vs[names[r[held // page]], :, held % page:] = float("nan")
        k[names[n:]], v[names[n:]] = 0x7F, 0xFF
    kc = k.view(nb, kv_heads, page, head // 16, 16).permute(0, 1, 3, 2, 4).contiguous().view(FP8)
    if trans:
        vc = v.view(nb, kv_heads, page // 16, 16, head).permute(0, 1, 2, 4, 3).contiguous().view(FP8)
    else:
        vc = v.transpose(2, 3).contiguous().view(FP8)
    q = torch.randn(len(ctx) * ql, heads, head, generator=gen).to(dtype)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32)
    return {"query": q, "key_cache": kc, "value_cache": vc, "key_scale": ks.contiguous(), "value_scale": vs.contiguous(),
            "block_tables": i32(tables), "context_lengths": i32(ctx), "prefix_indptr": i32(indptr),
            "prefix_lengths": i32(prefix), "softmax_scale": 1.0 / math.sqrt(head)}
