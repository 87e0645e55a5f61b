"""The page operators, the cache writer and the shared-prefix decode together,
as a server that samples several answers to one prompt runs them: the prompt
is written once, forked, every answer grows by itself, some end, the cache is
compacted and the rest go on."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from flydsl_amd import (build_fused_rope_cache_module, compact_cache_pages, extend_cache_pages, fork_cache_pages,
                        free_cache_pages, pa_decode_ps_launch, pa_decode_shared_prefix)
from tests.test_gpu_shared_prefix import check

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FP8 = torch.float8_e4m3fn


class Server:
    HQ, H, D, LAYERS, ROWS, WIDTH = 16, 2, 128, 2, 8, 24

    def __init__(self, bs, pages, seed=0):
        self.bs = bs
        self.gen = torch.Generator().manual_seed(seed)
        z = lambda *s: torch.full(s, 0x7F, dtype=torch.uint8, device=DEV).view(FP8)  # NaN until written
        self.keys = [z(pages, self.H, self.D // 16, bs, 16) for _ in range(self.LAYERS)]
        self.values = [z(pages, self.H, bs // 16, self.D, 16) for _ in range(self.LAYERS)]
        self.tables = torch.zeros(self.ROWS, self.WIDTH, dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(self.ROWS, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        ang = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(self.D // 2) / (self.D // 2))
        self.cos, self.sin = ang.cos().bfloat16().to(DEV), ang.sin().bfloat16().to(DEV)
        self.scale = torch.tensor([0.02], device=DEV)
        self.write = build_fused_rope_cache_module(head_dim=self.D, num_q_heads=self.HQ, num_kv_heads=self.H,
                                                   block_size=bs, flash_layout=False, apply_scale=True)
        self.mirror = {r: [None] * self.LAYERS for r in range(self.ROWS)}  # bytes that every row must read

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    def grow(self, rows, n):
        """n more tokens in each row, in every layer; the rotated queries."""
        old = self.lengths[self.ints(rows).long()].tolist()
        st = extend_cache_pages(self.keys + self.values, self.tables, self.lengths, self.refs, self.ints(rows),
                                self.ints([o + n for o in old]), self.bs)
        assert st.tolist() == [1] * len(rows)
        pos = torch.cat([torch.arange(o, o + n, device=DEV) for o in old])
        row = self.ints([r for r in rows for _ in range(n)]).long()
        slots = (self.tables[row, pos // self.bs] * self.bs + pos % self.bs).int()
        qs, t = [], len(rows) * n
        for layer in range(self.LAYERS):
            q, k, v = (torch.randn(t, h, self.D, generator=self.gen).bfloat16().to(DEV)
                       for h in (self.HQ, self.H, self.H))
            q_out, k_out = torch.empty_like(q), torch.empty_like(k)
            self.write(q, k, v, pos.int(), self.cos, self.sin, slots, self.keys[layer], self.values[layer], q_out,
                       k_out, t, self.scale, self.scale)
            qs.append(q_out)
            for i, r in enumerate(rows):  # the bytes as the writer left them, kept outside the cache
                self.remember(r, layer, old[i], n)
        return qs

    def tokens(self, row, layer, t0, n):
        t = torch.arange(t0, t0 + n, device=DEV)
        p, o = self.tables[row].long()[t // self.bs], t % self.bs
        k = self.keys[layer].view(torch.uint8)[p, :, :, o].flatten(1)
        v = self.values[layer].view(torch.uint8)[p, :, o // 16, :, o % 16].flatten(1)
        return torch.cat([k, v], 1)

    def remember(self, row, layer, t0, n):
        new = self.tokens(row, layer, t0, n).clone()
        had = self.mirror[row][layer]
        self.mirror[row][layer] = new if had is None or t0 == 0 else torch.cat([had[:t0], new])

    def unchanged(self, rows):
        for r in rows:
            n = int(self.lengths[r])
            for layer in range(self.LAYERS):
                assert torch.equal(self.tokens(r, layer, 0, n), self.mirror[r][layer][:n]), (r, layer)

    def decode(self, layer, q, rows, prefix):
        """Rows r0 .. of one group (the table rows of the batch in their order)."""
        idx = self.ints(rows).long()
        d = {"query": q, "key_cache": self.keys[layer], "value_cache": self.values[layer],
             "context_lengths": self.lengths[idx].contiguous(), "block_tables": self.tables[idx].contiguous(),
             "prefix_indptr": self.ints([0, len(rows)]), "prefix_lengths": self.ints([prefix]),
             "softmax_scale": 1 / math.sqrt(self.D), "key_scale": self.scale, "value_scale": self.scale}
        out = torch.empty_like(q)
        pa_decode_shared_prefix(out, *[d[k] for k in (
            "query", "key_cache", "value_cache", "context_lengths", "block_tables", "prefix_indptr", "prefix_lengths",
            "softmax_scale", "key_scale", "value_scale")])
        return d, out


@pytest.mark.parametrize("bs,prompt", [(16, 77), (16, 96), (64, 130)])
def test_answers_to_one_prompt(bs, prompt):
    s = Server(bs, pages=60, seed=bs + prompt)
    s.grow([0], prompt)
    kids = [1, 2, 3, 4, 5]
    st = fork_cache_pages(s.tables, s.lengths, s.refs, s.ints([0] * 5), s.ints(kids), bs)
    assert st.tolist() == [1] * 5
    for r in kids:
        s.mirror[r] = list(s.mirror[0])
    free_cache_pages(s.tables, s.lengths, s.refs, s.ints([0]), bs)
    for step in range(20):
        qs = s.grow(kids, 1)
        s.unchanged(kids)
        for layer, q in enumerate(qs):
            d, out = s.decode(layer, q, kids, prompt)
            if step % 6 == 0:
                check(d, out)
            other = torch.empty_like(out)
            pa_decode_ps_launch(other, q, s.keys[layer], s.values[layer], d["context_lengths"], None, None,
                                d["softmax_scale"], s.scale, s.scale, block_tables=d["block_tables"])
            assert torch.allclose(out.float(), other.float(), atol=2e-2, rtol=2e-2)
        if step == 8:  # an answer ends, another is taken back by a few tokens
            free_cache_pages(s.tables, s.lengths, s.refs, s.ints([2]), bs)
            kids.remove(2)
            free_cache_pages(s.tables, s.lengths, s.refs, s.ints([4]), bs, new_lengths=s.ints([prompt + 3]))
        if step == 12:  # compaction moves pages and changes nothing else
            before = [s.decode(layer, q, kids, prompt)[1]
                      for layer, q in enumerate(qs)]
            tables, refs, _, live = compact_cache_pages(s.keys + s.values, s.tables, s.lengths, s.refs, bs)
            s.tables, s.refs = tables, refs
            assert int(live) == int((refs > 0).sum()) and not refs[int(live):].any()
            s.unchanged(kids)
            for layer, q in enumerate(qs):
                assert torch.equal(s.decode(layer, q, kids, prompt)[1], before[layer])
    held = set(np.concatenate([s.tables[r, : -(-int(s.lengths[r]) // bs)].cpu().numpy() for r in kids]).tolist())
    assert held == set(torch.nonzero(s.refs).flatten().tolist())
    free_cache_pages(s.tables, s.lengths, s.refs, s.ints(kids), bs)
    assert not s.refs.any() and not s.lengths.any()
