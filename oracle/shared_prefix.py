"""Decode attention over a paged fp8 cache in float64, with what its error
bounds need (test infrastructure).

Every sequence is computed by itself over all of its tokens, each key and
value gathered through ``pages_of(b, t)``: a group's shared tokens come from
the table row of its first sequence, as the operator's definition says.
"""

from __future__ import annotations

import torch

FP8 = torch.float8_e4m3fn


def _rows(cache, pages, offsets, values: bool):
    """[tokens, Hkv, D] float64 fp8 values at (page, offset in page)."""
    u8 = cache.view(torch.uint8)
    if not values:
        x = u8[pages, :, :, offsets]  # [n, H, D/16, 16]
    elif cache.dim() == 5:
        x = u8[pages, :, offsets // 16, :, offsets % 16]  # [n, H, D]
    else:
        x = u8[pages, :, :, offsets]  # [n, H, D]
    return x.reshape(x.shape[0], x.shape[1], -1).view(FP8).double()


def decode(query, key_cache, value_cache, tables, lengths, indptr, prefix, scale, key_scale, value_scale):
    """(out, a, dx): float64 output [B*ql, Hq, D]; a = sum_t p_t |v_t| of each
    output; dx [B*ql, Hq, 1] = scale * max_t sum_d |q_d k_td|, the size whose
    float32 rounding moves a logit."""
    b_n = len(lengths)
    ql = query.shape[0] // max(b_n, 1)
    h, bs, d = key_cache.shape[1], key_cache.shape[3], query.shape[-1]
    gqa = query.shape[1] // h
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    a, dx = torch.zeros_like(out), torch.zeros(*query.shape[:2], 1, dtype=torch.float64, device=query.device)
    first, shared = list(range(b_n)), [0] * b_n
    for g, p in enumerate(prefix):
        for b in range(indptr[g], indptr[g + 1]):
            first[b], shared[b] = indptr[g], p
    for b in range(b_n):
        n = int(lengths[b])
        if n <= 0:
            continue
        t = torch.arange(n, device=query.device)
        row = torch.where(t < shared[b], tables[first[b]].long()[t // bs], tables[b].long()[t // bs])
        off = t % bs
        k, v = _rows(key_cache, row, off, False), _rows(value_cache, row, off, True)
        if key_scale.dim() > 1:
            k, v = k * key_scale[row, :, off].double(), v * value_scale[row, :, off].double()
        else:
            k, v = k * key_scale.double(), v * value_scale.double()
        for i in range(ql):
            see = n - ql + i + 1
            if see <= 0:
                continue
            r = b * ql + i
            q = query[r].double().view(h, gqa, d)
            kk, vv = k[:see].permute(1, 2, 0).contiguous(), v[:see].transpose(0, 1).contiguous()
            w = torch.softmax(torch.matmul(q, kk) * scale, dim=-1)
            out[r] = torch.matmul(w, vv).reshape(h * gqa, d)
            a[r] = torch.matmul(w, vv.abs()).reshape(h * gqa, d)
            dx[r] = (torch.matmul(q.abs(), kk.abs()).amax(-1) * abs(scale)).reshape(h * gqa, 1)
    return out, a, dx
